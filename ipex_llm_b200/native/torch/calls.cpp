// Calls of the CUDA library's training kernels with tensors, where a call from Python would take longer than the kernels: lists of
// hundreds of tensors, and the backward passes (a node of the autograd graph in C++ needs no interpreter on autograd's thread).
// The kernels' addresses come from the library that ctypes has loaded (`bind`), so that there is one of them in a process.
//
// Where an argument is not as it should be, or a list holds anything out of the ordinary (another type, device or order of memory, a
// tensor twice), the functions here answer so and do nothing; their callers in Python name what is wrong, or put it right.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <tuple>
#include <unordered_map>
#include <vector>

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

namespace {

// ------------------------------------------------------------------------------------------------ the library's entries
using AdamwStep = int (*)(const int64_t*, const int64_t*, const int64_t*, int64_t, void*, void*, uint8_t*, uint8_t*, void*, int, int64_t*,
                          int, void*, const float*, double, double, const float*, double, double, double, double, uint32_t, int, int,
                          void*);
using GradNorm = int (*)(const int64_t*, const int64_t*, int64_t, double*, float*, int, void*);
using Size = int64_t (*)(int64_t);
using RowSize = int64_t (*)(int64_t, int, int);
using PolicyLoss = int (*)(const void*, int64_t, int64_t, int64_t, const int64_t*, const float*, const float*, const float*, int64_t,
                           int64_t, int64_t, float*, float*, float*, uint8_t*, void*, void*, int64_t, int, int64_t, double, double, double,
                           float, int, int*, void*);
using PolicyGrad = int (*)(const void*, int64_t, int64_t, int64_t, const int64_t*, const void*, const float*, int64_t, int64_t, int64_t,
                           void*, int64_t, int, float, int, void*);
using PreferenceLoss = int (*)(const void*, int64_t, int64_t, int64_t, const int64_t*, const float*, float*, float*, void*, void*, int,
                               int64_t, int, int64_t, int, int, double, double, double, float, int, int*, void*);
using PreferenceGrad = int (*)(const void*, int64_t, int64_t, int64_t, const int64_t*, const void*, const float*, int64_t, const float*,
                               void*, int, int64_t, int, float, int, void*);

struct Entries {
  AdamwStep adamw_step = nullptr;
  GradNorm grad_norm = nullptr;
  Size grad_norm_sums = nullptr, keep_bytes = nullptr;
  RowSize work_bytes = nullptr;
  PolicyLoss policy_loss = nullptr;
  PolicyGrad policy_grad = nullptr;
  PreferenceLoss preference_loss = nullptr;
  PreferenceGrad preference_grad = nullptr;
} entries;

void bind(const std::unordered_map<std::string, uint64_t>& at) {
  auto take = [&](auto& f, const char* name) {
    const auto i = at.find(name);
    if (i != at.end()) f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(i->second);
  };
  take(entries.adamw_step, "ipex_adamw_step");
  take(entries.grad_norm, "ipex_grad_norm");
  take(entries.grad_norm_sums, "ipex_grad_norm_sums");
  take(entries.keep_bytes, "ipex_preference_keep_bytes");
  take(entries.work_bytes, "ipex_preference_work_bytes");
  take(entries.policy_loss, "ipex_policy_loss");
  take(entries.policy_grad, "ipex_policy_grad");
  take(entries.preference_loss, "ipex_preference_loss");
  take(entries.preference_grad, "ipex_preference_grad");
}

int type_code(at::ScalarType t) { return t == at::kHalf ? 0 : t == at::kBFloat16 ? 1 : t == at::kFloat ? 2 : -1; }

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "ipex_llm_b200 CUDA kernel '", what, "' failed: cudaError ", rc);
}

void* stream_of(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

template <typename T>
T* at_of(const std::optional<Tensor>& t) {
  return t.has_value() && t->defined() ? reinterpret_cast<T*>(t->data_ptr()) : nullptr;
}

// ------------------------------------------------------------------------------------------------ lists
// A list or tuple of tensors (or None) without copies of its references.
struct List {
  py::object held;
  PyObject** items = nullptr;
  Py_ssize_t n = -1;
  explicit List(py::handle h) {
    if (!PyList_Check(h.ptr()) && !PyTuple_Check(h.ptr())) return;
    held = py::reinterpret_borrow<py::object>(h);
    items = PySequence_Fast_ITEMS(h.ptr());
    n = PySequence_Fast_GET_SIZE(h.ptr());
  }
  bool ok() const {
    for (Py_ssize_t i = 0; i < n; ++i)
      if (items[i] != Py_None && !THPVariable_Check(items[i])) return false;
    return n > 0;
  }
  const Tensor* get(Py_ssize_t i) const { return items[i] == Py_None ? nullptr : &THPVariable_Unpack(items[i]); }
};

bool like(const Tensor& t, at::ScalarType type, const at::Device& dev) {
  return t.layout() == at::kStrided && t.scalar_type() == type && t.device() == dev;
}
bool flat(const Tensor& t, at::ScalarType type, const at::Device& dev, int64_t n, uintptr_t aligned) {
  return like(t, type, dev) && t.numel() == n && t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & (aligned - 1)) == 0;
}
bool one_of(const Tensor& t, const at::Device& dev) { return like(t, at::kFloat, dev) && t.numel() == 1; }

bool adamw_step(py::handle params_, py::handle grads_, const Tensor& m, const Tensor& v, const Tensor& step,
                const std::optional<Tensor>& m_scale, const std::optional<Tensor>& v_scale, const std::optional<Tensor>& rest,
                const std::optional<Tensor>& norm, double max_norm, double lr, const std::optional<Tensor>& lr_at, double b1, double b2,
                double eps, double decay, uint32_t seed) {
  const List params(params_), grads(grads_);
  if (params.n != grads.n || !params.ok() || !grads.ok() || params.get(0) == nullptr) return false;
  const int64_t n = params.n;
  const at::ScalarType type = params.get(0)->scalar_type();
  const at::Device dev = params.get(0)->device();
  if (!dev.is_cuda() || type_code(type) < 0) return false;
  std::vector<int64_t> at(4 * n);
  int64_t *p_at = at.data(), *g_at = p_at + n, *sizes = g_at + n, *sorted = sizes + n;
  int64_t total = 0, used = 0;
  for (int64_t i = 0; i < n; ++i) {
    const Tensor *p = params.get(i), *g = grads.get(i);
    if (p == nullptr || !like(*p, type, dev)) return false;
    const bool plain = p->is_contiguous();
    if (!plain && !p->is_non_overlapping_and_dense()) return false;
    sizes[i] = p->numel();
    total += (sizes[i] + 255) / 256 * 256;
    p_at[i] = reinterpret_cast<int64_t>(p->data_ptr());
    g_at[i] = 0;
    if (g == nullptr) continue;
    if (!like(*g, type, dev) || g->sizes() != p->sizes() || !((plain && g->is_contiguous()) || g->strides() == p->strides())) return false;
    g_at[i] = reinterpret_cast<int64_t>(g->data_ptr());
    if (sizes[i] > 0) sorted[used++] = p_at[i];
  }
  std::sort(sorted, sorted + used);
  if (std::adjacent_find(sorted, sorted + used) != sorted + used) return false;
  const bool small = m.scalar_type() == at::kFloat8_e4m3fn;
  if (!flat(m, small ? at::kFloat8_e4m3fn : at::kFloat, dev, total, 16) || !flat(v, small ? at::kFloat8_e5m2 : at::kFloat, dev, total, 16) ||
      !like(step, at::kLong, dev) || (step.numel() != 1 && step.numel() != n) || !step.is_contiguous())
    return false;
  if (small && (!m_scale || !v_scale || !flat(*m_scale, at::kByte, dev, total / 256, 1) || !flat(*v_scale, at::kByte, dev, total / 256, 1)))
    return false;
  int kind = 0;
  if (rest) {
    kind = rest->scalar_type() == at::kShort ? 1 : 2;
    if (type == at::kFloat || (kind == 1 && type != at::kBFloat16) || !flat(*rest, kind == 1 ? at::kShort : at::kFloat, dev, total, 16))
      return false;
  }
  if ((norm && !one_of(*norm, dev)) || (lr_at && !one_of(*lr_at, dev))) return false;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const Tensor factors = at::empty({8 * step.numel()}, at::TensorOptions().dtype(at::kFloat).device(dev));
  check(entries.adamw_step(p_at, g_at, sizes, n, m.data_ptr(), v.data_ptr(), at_of<uint8_t>(m_scale), at_of<uint8_t>(v_scale),
                           at_of<void>(rest), kind, step.data_ptr<int64_t>(), (int)step.numel(), factors.data_ptr(),
                           at_of<const float>(norm), max_norm, lr, at_of<const float>(lr_at), b1, b2, eps, decay, seed, type_code(type),
                           small, stream_of(dev)),
        "adamw_step");
  for (int64_t i = 0; i < n; ++i)
    if (g_at[i] != 0 && !params.get(i)->is_inference()) params.get(i)->unsafeGetTensorImpl()->bump_version();
  return true;
}

std::optional<Tensor> grad_norm(py::handle grads_) {
  const List grads(grads_);
  if (!grads.ok()) return std::nullopt;
  std::vector<int64_t> at, sizes;
  at.reserve(grads.n);
  sizes.reserve(grads.n);
  const Tensor* first = nullptr;
  for (Py_ssize_t i = 0; i < grads.n; ++i) {
    const Tensor* g = grads.get(i);
    if (g == nullptr) continue;
    if (first == nullptr) first = g;
    if (!like(*g, first->scalar_type(), first->device()) || !(g->is_contiguous() || g->is_non_overlapping_and_dense())) return std::nullopt;
    at.push_back(reinterpret_cast<int64_t>(g->data_ptr()));
    sizes.push_back(g->numel());
  }
  if (first == nullptr || !first->is_cuda() || type_code(first->scalar_type()) < 0) return std::nullopt;
  const at::Device dev = first->device();
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const at::TensorOptions opt = at::TensorOptions().device(dev);
  const Tensor sums = at::empty({entries.grad_norm_sums((int64_t)at.size())}, opt.dtype(at::kDouble));
  Tensor norm = at::empty({}, opt.dtype(at::kFloat));
  check(entries.grad_norm(at.data(), sizes.data(), (int64_t)at.size(), sums.data_ptr<double>(), norm.data_ptr<float>(),
                          type_code(first->scalar_type()), stream_of(dev)),
        "grad_norm");
  return norm;
}

// ------------------------------------------------------------------------------------------------ losses with a gradient
// Logits with unit stride along the vocabulary, and where their rows lie.
struct Rows {
  Tensor x;
  int64_t s0, s1, n1;
  explicit Rows(const Tensor& logits) : x(logits) {
    if (x.dim() > 3) x = x.reshape({-1, x.size(-2), x.size(-1)});
    if (x.stride(-1) != 1 && x.size(-1) > 1) x = x.contiguous();
    if (x.dim() == 3) s0 = x.stride(0), s1 = x.stride(1), n1 = x.size(1);
    else s0 = 0, s1 = x.dim() == 2 ? x.stride(0) : 0, n1 = x.dim() == 2 ? x.size(0) : 1;
  }
};

// Numbers for each row, broadcast to the targets' shape: strides over all but the last dimension, and along it.
struct PerRow {
  Tensor t;
  int64_t s0, s1, inner;
  PerRow(const Tensor& given, at::IntArrayRef shape) : t(given.expand(shape)) {
    if (t.dim() != 2) t = shape.empty() ? t.reshape({1, 1}) : t.reshape({-1, shape.back()});
    s0 = t.stride(0), s1 = t.stride(1), inner = t.size(1);
  }
};

Tensor bytes(int64_t n, const at::Device& dev) { return at::empty({n}, at::TensorOptions().dtype(at::kByte).device(dev)); }

// A gradient that has no gradient: differentiating it again raises instead of giving nothing.
Tensor once(Tensor dx, const variable_list& from) {
  if (!at::GradMode::is_enabled()) return dx;
  bool any = false;
  for (const auto& t : from) any = any || (t.defined() && t.requires_grad());
  if (!any) return dx;
  auto node = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", 1);
  return (*node)({dx.detach().requires_grad_()})[0];
}

struct Preference : torch::autograd::Function<Preference> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, const std::optional<Tensor>& reference,
                               double beta, int64_t form, double smooth, double margin, bool average, double temperature,
                               int64_t ignore, int64_t err) {
    const at::Device dev = logits.device();
    const c10::cuda::OptionalCUDAGuard guard(dev);
    const Rows r(logits);
    const int64_t n = logits.size(0), tokens = logits.size(1);
    const int type = type_code(logits.scalar_type());
    const at::TensorOptions opt = at::TensorOptions().dtype(at::kFloat).device(dev);
    Tensor loss = at::empty({n / 2}, opt), logprob = at::empty({n}, opt);
    const Tensor keep = bytes(entries.keep_bytes(n * tokens), dev), work = bytes(entries.work_bytes(n * tokens, (int)logits.size(2), type), dev);
    check(entries.preference_loss(r.x.data_ptr(), r.s0, r.s1, r.n1, targets.data_ptr<int64_t>(), at_of<const float>(reference),
                                  loss.data_ptr<float>(), logprob.data_ptr<float>(), keep.data_ptr(), work.data_ptr(), (int)(n / 2), tokens,
                                  (int)logits.size(2), ignore, (int)form, average, beta, smooth, margin, (float)temperature,
                                  type_code(logits.scalar_type()), reinterpret_cast<int*>(err), stream_of(dev)),
          "preference_loss");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, targets, keep});
    ctx->saved_data["temperature"] = temperature;
    return {loss, logprob};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(11);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &targets = saved[1], &keep = saved[2];
    Tensor dx;
    {
      const at::AutoGradMode off(false);
      const at::Device dev = logits.device();
      const c10::cuda::OptionalCUDAGuard guard(dev);
      const Rows r(logits);
      const Tensor g = grads[0].defined() ? grads[0].to(at::kFloat) : Tensor();
      const Tensor g_seq = grads[1].defined() ? grads[1].to(at::kFloat).contiguous() : Tensor();
      dx = at::empty(logits.sizes(), logits.options());
      check(entries.preference_grad(r.x.data_ptr(), r.s0, r.s1, r.n1, targets.data_ptr<int64_t>(), keep.data_ptr(), at_of<const float>(g),
                                    g.defined() ? g.stride(0) : 0, at_of<const float>(g_seq), dx.data_ptr(), (int)(logits.size(0) / 2),
                                    logits.size(1), (int)logits.size(2), (float)ctx->saved_data["temperature"].toDouble(),
                                    type_code(logits.scalar_type()), stream_of(dev)),
            "preference_grad");
    }
    out[0] = once(dx, {logits, grads[0], grads[1]});
    return out;
  }
};

struct Policy : torch::autograd::Function<Policy> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, const Tensor& advantages,
                               const std::optional<Tensor>& old, const std::optional<Tensor>& ref, double lo, double hi, double weight,
                               double temperature, int64_t ignore, int64_t err) {
    const at::Device dev = logits.device();
    const c10::cuda::OptionalCUDAGuard guard(dev);
    const Rows r(logits);
    const int64_t rows = targets.numel();
    const at::TensorOptions opt = at::TensorOptions().dtype(at::kFloat).device(dev);
    Tensor loss = at::empty(targets.sizes(), opt), logprob = at::empty(targets.sizes(), opt), kl = at::empty(targets.sizes(), opt);
    Tensor clipped = at::empty(targets.sizes(), opt.dtype(at::kBool));
    const Tensor keep = bytes(entries.keep_bytes(rows), dev);
    if (rows > 0) {
      const Tensor work = bytes(entries.work_bytes(rows, (int)logits.size(-1), type_code(logits.scalar_type())), dev);
      const PerRow a(advantages, targets.sizes());
      check(entries.policy_loss(r.x.data_ptr(), r.s0, r.s1, r.n1, targets.data_ptr<int64_t>(), at_of<const float>(old),
                                at_of<const float>(ref), a.t.data_ptr<float>(), a.s0, a.s1, a.inner, loss.data_ptr<float>(),
                                logprob.data_ptr<float>(), kl.data_ptr<float>(), reinterpret_cast<uint8_t*>(clipped.data_ptr()),
                                keep.data_ptr(), work.data_ptr(), rows, (int)logits.size(-1), ignore, lo, hi, weight, (float)temperature,
                                type_code(logits.scalar_type()), reinterpret_cast<int*>(err), stream_of(dev)),
            "policy_loss");
    }
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({logprob, kl, clipped});
    ctx->save_for_backward({logits, targets, keep});
    ctx->saved_data["temperature"] = temperature;
    return {loss, logprob, kl, clipped};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(11);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &targets = saved[1], &keep = saved[2];
    Tensor dx;
    {
      const at::AutoGradMode off(false);
      const at::Device dev = logits.device();
      const c10::cuda::OptionalCUDAGuard guard(dev);
      dx = at::empty(logits.sizes(), logits.options());
      if (targets.numel() > 0) {
        const Rows r(logits);
        const PerRow g(grads[0].to(at::kFloat), targets.sizes());
        check(entries.policy_grad(r.x.data_ptr(), r.s0, r.s1, r.n1, targets.data_ptr<int64_t>(), keep.data_ptr(), g.t.data_ptr<float>(),
                                  g.s0, g.s1, g.inner, dx.data_ptr(), targets.numel(), (int)logits.size(-1),
                                  (float)ctx->saved_data["temperature"].toDouble(), type_code(logits.scalar_type()), stream_of(dev)),
              "policy_grad");
      }
    }
    out[0] = once(dx, {logits, grads[0]});
    return out;
  }
};

// Whether arguments are as the documentation asks for; else the caller finds out what is wrong with them.
bool logits_fit(const Tensor& x, double temperature) {
  return x.is_cuda() && x.layout() == at::kStrided && type_code(x.scalar_type()) >= 0 && x.dim() >= 1 && x.size(-1) >= 1 &&
         x.size(-1) <= (int64_t)1 << 30 && x.numel() / x.size(-1) <= (int64_t)1 << 27 && temperature >= 1e-6 && temperature <= 1e6;
}
bool targets_fit(const Tensor& t, at::IntArrayRef shape, const Tensor& x) {
  return t.device() == x.device() && t.layout() == at::kStrided && at::isIntegralType(t.scalar_type(), false) &&
         t.sizes() == shape;
}
bool numbers_fit(const std::optional<Tensor>& t, at::IntArrayRef shape, const Tensor& x) {
  return !t || (t->device() == x.device() && t->layout() == at::kStrided && t->is_floating_point() && t->sizes() == shape);
}
Tensor whole(const Tensor& t) { return t.scalar_type() == at::kLong && t.is_contiguous() ? t : t.to(at::kLong).contiguous(); }
Tensor single(const Tensor& t) {      // a constant, in 32 bits
  const Tensor d = t.requires_grad() ? t.detach() : t;
  return d.scalar_type() == at::kFloat ? d : d.to(at::kFloat);
}
std::optional<Tensor> single(const std::optional<Tensor>& t) {
  return t ? std::optional<Tensor>(single(*t).contiguous()) : std::nullopt;
}

std::optional<std::tuple<Tensor, Tensor>> preference(const Tensor& logits, const Tensor& targets, const std::optional<Tensor>& reference,
                                                     double beta, int64_t form, double smooth, double margin, bool average,
                                                     double temperature, int64_t ignore, int64_t err) {
  if (!logits_fit(logits, temperature) || logits.dim() != 3 || logits.size(0) < 2 || logits.size(0) % 2 || logits.size(1) < 1 ||
      !targets_fit(targets, logits.sizes().slice(0, 2), logits) || !numbers_fit(reference, logits.sizes().slice(0, 1), logits) || form < 0 ||
      !(beta > 0.0 && beta < INFINITY && smooth >= 0.0 && smooth <= 1.0 && std::isfinite(margin)) ||
      (form > 0 && (smooth != 0.0 || margin != 0.0)))
    return std::nullopt;
  const auto out = Preference::apply(logits, whole(targets), single(reference), beta, form, smooth, margin, average, temperature, ignore, err);
  return std::make_tuple(out[0], out[1]);
}

std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>> policy(const Tensor& logits, const Tensor& targets, const Tensor& advantages,
                                                                 const std::optional<Tensor>& old, const std::optional<Tensor>& ref,
                                                                 double lo, double hi, double weight, double temperature, int64_t ignore,
                                                                 int64_t err) {
  if (!logits_fit(logits, temperature)) return std::nullopt;
  const at::IntArrayRef shape = logits.sizes().slice(0, logits.dim() - 1);
  if (!targets_fit(targets, shape, logits) || !numbers_fit(old, shape, logits) || !numbers_fit(ref, shape, logits) ||
      !numbers_fit(advantages, advantages.sizes(), logits) || advantages.dim() > (int64_t)shape.size() ||
      !(lo >= 0.0 && lo <= 1.0 && hi >= 0.0 && weight >= 0.0 && weight < INFINITY) || (weight != 0.0 && !ref))
    return std::nullopt;
  for (int64_t i = 1; i <= advantages.dim(); ++i)
    if (advantages.size(-i) != 1 && advantages.size(-i) != shape[shape.size() - i]) return std::nullopt;
  const auto out = Policy::apply(logits, whole(targets), single(advantages), single(old), single(ref), lo, hi, weight, temperature, ignore, err);
  return std::make_tuple(out[0], out[1], out[2], out[3]);
}

}  // namespace

PYBIND11_MODULE(libipex_calls, m) {
  m.def("bind", &bind);
  m.def("adamw_step", &adamw_step);
  m.def("grad_norm", &grad_norm);
  m.def("preference", &preference);
  m.def("policy", &policy);
}
