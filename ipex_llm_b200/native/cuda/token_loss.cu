// What stands behind an output layer: log probabilities of given tokens with their entropy and the best alternatives, and
// the divergence from a teacher's top logits, each with the gradient of the logits.  sm_100a.
//
// With y = x / T, m = max x, s = sum e^((x - m) / T), t = sum e^((x - m) / T) (x - m):
//
//   log p_j = (x_j - m) / T - ln s            H = ln s - t / (s T)
//   d log p_t / dx_j = (1[j = t] - p_j) / T   dH / dx_j = -p_j (log p_j + H) / T
//
// All of them are bound by memory: forward reads a row once, backward reads it once more and writes it once.  A row belongs
// to one CTA (many rows) or to a cluster of up to eight (few rows).  A thread takes four 16-byte requests at a time, which
// keeps 32 KB of a CTA in flight, folds their maximum into its own and rescales its sums once for all of them, so that an
// element costs one exponential (0.73 of what the special function units do at the rate of memory, for 16-bit logits).
// x - m is taken before the factor log2(e) / T: its rounding then does not grow with m, as that of one fma(x, c, -m c) would.
//
// Statistics are 32-bit, 250 to 500 elements to a thread's sum and a tree above that; exponentials by ex2.approx (2 ulp).
#include <cooperative_groups.h>

#include <type_traits>

#include "common/utils.cuh"
#include "tcgen05_common.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kNT = 512;
constexpr int kWarps = kNT / 32;
constexpr int kU = 4;             // 16-byte requests of a thread in flight
constexpr int kMaxTop = 32;
constexpr int kMaxK = 1024;
constexpr int kCand = 1024;       // candidates for the best tokens of a slice before it is scanned in rounds instead
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kErrToken = 61;     // a token outside of the vocabulary

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// x - m, held above -1e25 (e^(-1e25 / T) is 0 for every temperature up to 1e6), so that its product with a sum of up to 2^30
// stays finite and 0 * (x - m) is 0 for hidden tokens (-inf, or the type's lowest value); NaN stays NaN.
__device__ __forceinline__ float below(float x, float m) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(x - m), "f"(-1.0e25f));
  return d;
}

struct Rows {
  const void* x;
  int64_t s0, s1;      // strides of the outer and the inner row index, in elements
  int64_t n1;          // rows to an outer index
  int V;
};

template <typename T>
__device__ __forceinline__ const T* row_at(const Rows& r, int64_t row) {
  return reinterpret_cast<const T*>(r.x) + row / r.n1 * r.s0 + row % r.n1 * r.s1;
}

// A row [V] of any alignment: elements in front of the first 16-byte boundary, vectors, what is left.
template <typename T>
struct Slice {
  static constexpr int VEC = 16 / sizeof(T);
  int head, nvec, tail;  // of the whole row
  int v0, v1;            // vectors of this CTA
  int h, t;              // single elements of this CTA: [0, h) and [V - t, V)
  int V;
  __device__ Slice(const T* x, int V_, int rank, int parts) : V(V_) {
    const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15) / (int)sizeof(T);
    head = off ? min(VEC - off, V) : 0;
    nvec = (V - head) / VEC;
    tail = V - head - nvec * VEC;
    v0 = (int)((int64_t)nvec * rank / parts);
    v1 = (int)((int64_t)nvec * (rank + 1) / parts);
    h = rank == 0 ? head : 0;
    t = rank == parts - 1 ? tail : 0;
  }
  __device__ bool has(int j) const {
    return (j >= head + v0 * VEC && j < head + v1 * VEC) || j < h || (j >= V - t && j < V);
  }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& w, float* f) {
  const T* p = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) f[i] = DT<T>::to_f(p[i]);
}
template <typename T>
__device__ __forceinline__ uint4 hidden() {  // a vector of -inf
  const uint32_t w = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
  return make_uint4(w, w, w, w);
}

// Larger keys come first: by value (NaN above all), then by the lower index.  No element has key 0.
__device__ __forceinline__ uint64_t order_key(float v, int idx) {
  const uint32_t b = v != v ? 0x7FFFFFFFu : __float_as_uint(v == 0.f ? 0.f : v);   // -0 and 0 are equal
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)o << 32 | (0xFFFFFFFFu - (uint32_t)idx);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

// m: maximum, s: sum of e^((x - m) / T), t: that sum weighted by x - m (ENT), or over the tokens not given (TAIL).
struct Stat {
  float m, s, t;
};
template <bool ENT>
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float c) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  const float da = below(a.m, ref), db = below(b.m, ref);   // sums of a side without tokens are 0
  const float ea = ex2(da * c), eb = ex2(db * c);
  r.s = a.s * ea + b.s * eb;
  r.t = ENT ? (a.t + a.s * da) * ea + (b.t + b.s * db) * eb : a.t * ea + b.t * eb;
  return r;
}

struct Shared {
  Stat warp[kWarps];
  Stat part;                      // this CTA's
  Stat all;                       // the row's
  uint64_t best[kNT];             // each thread's best key
  uint64_t cand[kCand];
  uint64_t top[kMaxTop];          // this CTA's best, sorted
  uint64_t thr;
  int n_cand, n_list;
  int list[kMaxTop];              // threads that may hold one of the best
};

template <typename T, bool ENT, bool TOP, bool TAIL>
__device__ void scan(const T* x, const Slice<T>& sl, float c, const uint32_t* given, const int* ids, int K, Shared& sh) {
  constexpr int VEC = Slice<T>::VEC;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Stat st = {-INFINITY, 0.f, 0.f};
  float best = -INFINITY;
  int best_at = -1;                // first vector of the batch that holds `best`; -2 - j: the single element j
  auto single = [&](int j) {
    const float v = DT<T>::to_f(x[j]);
    bool is_given = false;
    if constexpr (TAIL)
      for (int k = 0; k < K; ++k) is_given |= ids[k] == j;
    Stat one = {v, 1.f, TAIL && !is_given ? 1.f : 0.f};
    if (v == -INFINITY) one.s = one.t = 0.f;
    if (v != v) one.s = one.t = v;
    st = join<ENT>(st, one, c);
    if (TOP && (best_at == -1 || order_key(v, 0) > order_key(best, 0))) {
      best = v;
      best_at = -2 - j;
    }
  };
  if (tid < sl.h) single(tid);
  const uint4* xv = reinterpret_cast<const uint4*>(x + sl.head);
  for (int base = sl.v0 + tid; base < sl.v1; base += kNT * kU) {
    uint4 w[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) w[u] = base + u * kNT < sl.v1 ? ldg_nc_v4(xv + base + u * kNT) : hidden<T>();
    float f[kU * VEC], mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kU; ++u) unpack<T>(w[u], f + u * VEC);
#pragma unroll
    for (int i = 0; i < kU * VEC; ++i) mx = fmaxf(mx, f[i]);
    const float m = fmaxf(st.m, mx), ref = m == -INFINITY ? 0.f : m;
    const float down = below(st.m, ref), fac = ex2(down * c);
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float sv = 0.f;
      uint32_t bits = 0;
      if constexpr (TAIL) {
        const int pos = min(base + u * kNT, sl.v1 - 1) * VEC - sl.v0 * VEC;
        bits = given[pos >> 5] >> (pos & 31) & ((1u << VEC) - 1);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = ENT ? below(f[u * VEC + i], ref) : f[u * VEC + i] - ref;
        const float e = ex2(d * c);
        sv += e;
        if constexpr (ENT) t = fmaf(e, d, t);
        if constexpr (TAIL) t += bits >> i & 1 ? 0.f : e;
      }
      s += sv;
    }
    if constexpr (ENT) st.t = (st.t + st.s * down) * fac + t;
    else if constexpr (TAIL) st.t = st.t * fac + t;
    st.s = st.s * fac + s;
    st.m = m;
    if constexpr (TOP) {
      if (s != s) {
#pragma unroll
        for (int i = 0; i < kU * VEC; ++i) mx = f[i] != f[i] ? NAN : mx;
      }
      if (best_at == -1 || order_key(mx, 0) > order_key(best, 0)) {
        best = mx;
        best_at = base;
      }
    }
  }
  if (tid >= kNT - sl.t) single(sl.V - (kNT - tid));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat other = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                  __shfl_xor_sync(0xffffffffu, st.t, o)};
    st = lane & o ? join<ENT>(other, st, c) : join<ENT>(st, other, c);
  }
  if (lane == 0) sh.warp[warp] = st;
  if constexpr (TOP) {
    uint64_t key = 0;
    if (best_at <= -2) key = order_key(best, -2 - best_at);
    if (best_at >= 0) {
      for (int u = kU - 1; u >= 0; --u) {
        const int v = best_at + u * kNT;
        if (v >= sl.v1) continue;
        float f[VEC];
        unpack<T>(ldg_nc_v4(xv + v), f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const uint64_t k = order_key(f[i], sl.head + v * VEC + i);
          key = k > key ? k : key;
        }
      }
    }
    sh.best[tid] = key;
  }
  __syncthreads();
  if (tid == 0) {
    Stat a = sh.warp[0];
    for (int i = 1; i < kWarps; ++i) a = join<ENT>(a, sh.warp[i], c);
    sh.part = a;
  }
}

// The elements of thread `t`, every `step`-th of its vectors from `first` on.
template <typename T, typename F>
__device__ __forceinline__ void elements_of(const T* x, const Slice<T>& sl, int t, int first, int step, F f) {
  constexpr int VEC = Slice<T>::VEC;
  const uint4* xv = reinterpret_cast<const uint4*>(x + sl.head);
  if (first == 0 && t < sl.h) f(DT<T>::to_f(x[t]), t);
  for (int64_t v = (int64_t)sl.v0 + t + (int64_t)first * kNT; v < sl.v1; v += (int64_t)step * kNT) {
    float e[VEC];
    unpack<T>(ldg_nc_v4(xv + v), e);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f(e[i], sl.head + (int)v * VEC + i);
  }
  if (first == 0 && t >= kNT - sl.t) f(DT<T>::to_f(x[sl.V - (kNT - t)]), sl.V - (kNT - t));
}

// The `top` largest keys of a slice, sorted, into sh.top (0 behind the last element).  The top-th largest of the threads' best
// keys bounds them from below, and only the threads above that bound (top of them, keys being unique) can hold any: their
// elements are read again, by a warp each, and what passes the bound is ranked by counting.  Where more than kCand pass (a few
// threads hold nearly all large values), the slice is scanned once for each rank instead.
template <typename T>
__device__ void best_tokens(const T* x, const Slice<T>& sl, int top, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kMaxTop) sh.top[tid] = 0;
  if (tid == 0) {
    sh.thr = 0;
    sh.n_cand = sh.n_list = 0;
  }
  __syncthreads();
  const uint64_t mine = sh.best[tid];
  int rank = 0;
  if (mine != 0)
    for (int i = 0; i < kNT; ++i) rank += sh.best[i] > mine;
  if (mine != 0 && rank < top) sh.list[rank] = tid;
  const int held = __syncthreads_count(mine != 0);
  if (mine != 0 && rank == top - 1) sh.thr = mine;
  __syncthreads();
  const uint64_t thr = sh.thr;
  const int n_list = min(held, top);
  for (int i = warp; i < n_list; i += kWarps)
    elements_of<T>(x, sl, sh.list[i], lane, 32, [&](float v, int j) {
      const uint64_t k = order_key(v, j);
      if (k >= thr) {
        const int at = atomicAdd(&sh.n_cand, 1);
        if (at < kCand) sh.cand[at] = k;
      }
    });
  __syncthreads();
  const int n = sh.n_cand;
  if (n <= kCand) {
    for (int i = tid; i < n; i += kNT) {
      const uint64_t k = sh.cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += sh.cand[j] > k;
      if (r < top) sh.top[r] = k;
    }
    __syncthreads();
    return;
  }
  uint64_t under = ~0ull;
  for (int r = 0; r < top; ++r) {
    uint64_t b = 0;
    elements_of<T>(x, sl, tid, 0, 1, [&](float v, int j) {
      const uint64_t k = order_key(v, j);
      if (k < under && k > b) b = k;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t w = __shfl_xor_sync(0xffffffffu, b, o);
      b = w > b ? w : b;
    }
    if (lane == 0) sh.best[warp] = b;
    __syncthreads();
    b = sh.best[0];
    for (int i = 1; i < kWarps; ++i) b = sh.best[i] > b ? sh.best[i] : b;
    if (tid == 0) sh.top[r] = b;
    under = b;
    __syncthreads();
    if (b == 0) break;
  }
}

// The row's statistics from those of the cluster's CTAs, in every thread of the first one.
template <bool ENT>
__device__ __forceinline__ Stat row_stat(Shared& sh, int parts, float c) {
  if (parts == 1) {
    __syncthreads();
    return sh.part;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  Stat a = *cl.map_shared_rank(&sh.part, 0);
  for (int i = 1; i < parts; ++i) a = join<ENT>(a, *cl.map_shared_rank(&sh.part, i), c);
  return a;
}

struct ProbArgs {
  Rows rows;
  const int64_t* targets;
  float* logprob;
  float* entropy;      // null: not asked for
  float* stats;        // [rows, 4]: m, 1 / s, ln s, H
  float* top_logprob;  // [rows, top]
  int64_t* top_id;
  int top, parts;
  int64_t ignore;
  float temp, inv_t;
  int* err;
};

template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kNT, 2) token_logprobs_kernel(ProbArgs a) {
  __shared__ Shared sh;
  const int parts = a.parts, rank = parts == 1 ? 0 : (int)(blockIdx.x % parts);
  const int64_t row = blockIdx.x / parts;
  const T* x = row_at<T>(a.rows, row);
  const Slice<T> sl(x, a.rows.V, rank, parts);
  const float c = a.inv_t * kLog2e;
  scan<T, ENT, TOP, false>(x, sl, c, nullptr, nullptr, 0, sh);
  if constexpr (TOP) best_tokens<T>(x, sl, a.top, sh);
  const Stat st = row_stat<ENT>(sh, parts, c);
  if (rank == 0) {
    const bool none = st.m == -INFINITY && st.s == 0.f;      // a row without any token
    const float m = none ? 0.f : st.m, ln_s = none ? 0.f : log2f(st.s) * kLn2;
    const float H = !ENT || none ? 0.f : ln_s - st.t / st.s / a.temp;
    if (threadIdx.x == 0) {
      const int64_t t = a.targets[row];
      const bool ignored = t == a.ignore, bad = !ignored && (t < 0 || t >= a.rows.V);
      float lp = 0.f;
      if (bad) {
        tc5::report(a.err, kErrToken);
        lp = NAN;
      } else if (!ignored) {
        lp = none ? -INFINITY : (DT<T>::to_f(x[t]) - m) / a.temp - ln_s;
      }
      a.logprob[row] = lp;
      if (ENT) a.entropy[row] = ignored ? 0.f : bad ? NAN : H;
      float4 s4 = make_float4(m, none ? 0.f : 1.f / st.s, ln_s, H);
      if (a.stats != nullptr) reinterpret_cast<float4*>(a.stats)[row] = s4;
    }
    if constexpr (TOP) {
      // the parts' sorted lists joined: a key's rank is the number of larger ones in all of them
      uint64_t* all = sh.cand;
      const int n = parts * a.top;
      if (parts == 1) {
        for (int i = threadIdx.x; i < n; i += kNT) all[i] = sh.top[i];
      } else {
        cg::cluster_group cl = cg::this_cluster();
        for (int i = threadIdx.x; i < n; i += kNT) all[i] = cl.map_shared_rank(&sh, i / a.top)->top[i % a.top];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kNT) {
        const uint64_t k = all[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += all[j] > k;
        if (k != 0 && r < a.top) {
          const int id = key_index(k);
          a.top_id[row * a.top + r] = id;
          a.top_logprob[row * a.top + r] = none ? -INFINITY : (DT<T>::to_f(x[id]) - m) / a.temp - ln_s;
        }
      }
    }
  }
  if (parts > 1) cg::this_cluster().sync();      // shared memory stays until the first CTA has read it
}

// Elementwise over a row, VEC at a time where input and output lie alike, else one by one on the way out.
template <typename T, typename F>
__device__ __forceinline__ void map_row(const T* x, T* y, const Slice<T>& sl, F f) {
  constexpr int VEC = Slice<T>::VEC;
  const int tid = threadIdx.x;
  if (tid < sl.h) y[tid] = DT<T>::from_f(f(DT<T>::to_f(x[tid])));
  if (tid >= kNT - sl.t) {
    const int j = sl.V - (kNT - tid);
    y[j] = DT<T>::from_f(f(DT<T>::to_f(x[j])));
  }
  const uint4* xv = reinterpret_cast<const uint4*>(x + sl.head);
  const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  for (int base = sl.v0 + tid; base < sl.v1; base += kNT * 2) {
    uint4 w[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (base + u * kNT < sl.v1) w[u] = ldg_nc_v4(xv + base + u * kNT);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int v = base + u * kNT;
      if (v >= sl.v1) break;
      float e[VEC];
      unpack<T>(w[u], e);
      __align__(16) T o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = DT<T>::from_f(f(e[i]));
      T* at = y + sl.head + (int64_t)v * VEC;
      if (alike) {
        *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(o);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) at[i] = o[i];
      }
    }
  }
}

struct ProbGradArgs {
  Rows rows;
  const int64_t* targets;
  const float* stats;
  const float* g;        // of the log probability, or null
  const float* g_ent;    // of the entropy, or null
  void* dx;              // [rows, V]
  int64_t ignore;
  float inv_t;
  int parts;
};

template <typename T, bool ENT>
__global__ void __launch_bounds__(kNT) token_logprobs_grad_kernel(ProbGradArgs a) {
  const int64_t row = blockIdx.x / a.parts;
  const T* x = row_at<T>(a.rows, row);
  T* y = reinterpret_cast<T*>(a.dx) + row * a.rows.V;
  const Slice<T> sl(x, a.rows.V, (int)(blockIdx.x % a.parts), a.parts);
  const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
  const int64_t t = a.targets[row];
  const bool ignored = t == a.ignore, bad = !ignored && (t < 0 || t >= a.rows.V);
  float g = ignored || a.g == nullptr ? 0.f : a.g[row], ge = ignored || !ENT ? 0.f : a.g_ent[row];
  if (bad) g = NAN;
  if (st.y == 0.f) g = ge = 0.f;                    // no token in the row
  const float c = a.inv_t * kLog2e, scale = -st.y * a.inv_t, lp0 = st.w - st.z;
  if (g == 0.f && ge == 0.f) {                      // nothing flows into this row, whatever its logits hold
    map_row<T>(x, y, sl, [](float) { return 0.f; });
    return;
  }
  auto grad = [&](float v) {
    const float d = ENT ? below(v, st.x) : v - st.x;
    const float e = ex2(d * c) * scale;
    return ENT ? e * fmaf(ge, fmaf(d, a.inv_t, lp0), g) : e * g;
  };
  map_row<T>(x, y, sl, grad);
  __syncthreads();
  if (threadIdx.x == 0 && !bad && t >= 0 && t < a.rows.V && !ignored && sl.has((int)t))
    y[t] = DT<T>::from_f(fmaf(g, a.inv_t, grad(DT<T>::to_f(x[t]))));
}

// ------------------------------------------------------------------------------------------------ distillation
// The teacher's top tokens: q_k = softmax of the given logits / T over them, or e^(t_k / T - lse) with the teacher's own
// logsumexp; then what they leave, rest = max(0, 1 - sum q), belongs to all other tokens together (TAIL), whose sum under
// the student is taken over them alone (a bitmap of the given ones in shared memory): 1 - sum p of the given would cancel.
//   loss = T^2 (sum_k q_k (log q_k - log p_id) + rest (log rest - log left))
//   dx_j = T g (M p_j - sum_{k: id_k = j} q_k - [j not given] (rest / left) p_j)        M = sum q + rest
struct DistillArgs {
  Rows rows;
  const int64_t* ids;      // [rows, K], below 0: no token
  const float* values;     // [rows, K]
  const float* lse;        // [rows] or null
  float* loss;             // [rows]
  float* stats;            // [rows, 8]: m, 1 / s, M, rest / left, log-normaliser of q, -, -, -
  int K, parts;
  float temp, inv_t;
  int* err;
};

__device__ __forceinline__ float block_reduce(float v, bool is_max, float* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = is_max ? fmaxf(v, w) : v + w;
  }
  __syncthreads();
  if (lane == 0) buf[warp] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < kWarps; ++i) v = is_max ? fmaxf(v, buf[i]) : v + buf[i];
  return v;
}

template <typename T, bool TAIL>
__global__ void __launch_bounds__(kNT, 2) distill_kernel(DistillArgs a) {
  extern __shared__ uint32_t given[];                        // a bit for each element of this CTA's vectors
  __shared__ Shared sh;
  __shared__ int ids[kMaxK];
  __shared__ float red[kWarps];
  const int parts = a.parts, rank = parts == 1 ? 0 : (int)(blockIdx.x % parts), tid = threadIdx.x, K = a.K;
  const int64_t row = blockIdx.x / parts;
  const T* x = row_at<T>(a.rows, row);
  const Slice<T> sl(x, a.rows.V, rank, parts);
  constexpr int VEC = Slice<T>::VEC;
  const float c = a.inv_t * kLog2e;
  bool bad = false;
  for (int k = tid; k < K; k += kNT) {
    const int64_t id = a.ids[row * K + k];
    bad |= id >= a.rows.V;
    ids[k] = id < 0 || id >= a.rows.V ? -1 : (int)id;
  }
  if constexpr (TAIL) {
    for (int i = tid; i < ((sl.v1 - sl.v0) * VEC + 31) / 32; i += kNT) given[i] = 0;
  }
  bad = __syncthreads_or(bad);
  if constexpr (TAIL) {
    for (int k = tid; k < K; k += kNT) {
      const int pos = ids[k] - sl.head - sl.v0 * VEC;
      if (ids[k] >= 0 && pos >= 0 && pos < (sl.v1 - sl.v0) * VEC) atomicOr(&given[pos >> 5], 1u << (pos & 31));
    }
    __syncthreads();
  }
  scan<T, false, false, TAIL>(x, sl, c, given, ids, K, sh);
  const Stat st = row_stat<false>(sh, parts, c);
  if (rank == 0) {
    const bool none = st.m == -INFINITY && st.s == 0.f;
    const float m = none ? 0.f : st.m, ln_s = none ? 0.f : log2f(st.s) * kLn2;
    float z = 0.f;                                           // log q_k = t_k / T - z
    float top = -INFINITY, sum = 0.f;
    for (int k = tid; k < K; k += kNT)
      if (ids[k] >= 0) top = fmaxf(top, a.values[row * K + k] / a.temp);
    top = block_reduce(top, true, red);
    const bool empty = top == -INFINITY;                     // no token given
    if constexpr (TAIL) {
      z = a.lse[row];
    } else if (!empty) {
      for (int k = tid; k < K; k += kNT)
        if (ids[k] >= 0) sum += ex2((a.values[row * K + k] / a.temp - top) * kLog2e);
      sum = block_reduce(sum, false, red);
      z = top + log2f(sum) * kLn2;
    }
    float part = 0.f, mass = 0.f;
    for (int k = tid; k < K; k += kNT) {
      if (ids[k] < 0) continue;
      const float lq = a.values[row * K + k] / a.temp - z, q = ex2(lq * kLog2e);
      const float lp = (DT<T>::to_f(x[ids[k]]) - m) / a.temp - ln_s;
      if (q != 0.f) part = fmaf(q, lq - lp, part);
      mass += q;
    }
    part = block_reduce(part, false, red);
    mass = block_reduce(mass, false, red);
    if (tid == 0) {
      float rest = 0.f, ratio = 0.f;
      if constexpr (TAIL) {
        rest = fmaxf(1.f - mass, 0.f);
        const float left = none ? 0.f : st.t / st.s;
        if (rest > 0.f && left > 0.f) {
          ratio = rest / left;
          part = fmaf(rest, (log2f(rest) - log2f(left)) * kLn2, part);
        } else {
          rest = 0.f;                                        // the student has no other token: the term is left out
        }
      }
      if (empty) part = mass = rest = ratio = 0.f;
      if (bad) {
        tc5::report(a.err, kErrToken);
        part = mass = NAN;
      }
      a.loss[row] = part * (a.temp * a.temp);
      if (a.stats != nullptr) {
        float4* s4 = reinterpret_cast<float4*>(a.stats) + 2 * row;
        s4[0] = make_float4(m, none ? 0.f : 1.f / st.s, mass + rest, ratio);
        s4[1] = make_float4(z, 0.f, 0.f, 0.f);
      }
    }
  }
  if (parts > 1) cg::this_cluster().sync();
}

struct DistillGradArgs {
  Rows rows;
  const int64_t* ids;
  const float* values;
  const float* stats;
  const float* g;
  void* dx;
  int K, parts;
  float temp, inv_t;
};

template <typename T>
__global__ void __launch_bounds__(kNT) distill_grad_kernel(DistillGradArgs a) {
  __shared__ int ids[kMaxK];
  __shared__ float q[kMaxK];
  const int64_t row = blockIdx.x / a.parts;
  const int K = a.K;
  const T* x = row_at<T>(a.rows, row);
  T* y = reinterpret_cast<T*>(a.dx) + row * a.rows.V;
  const Slice<T> sl(x, a.rows.V, (int)(blockIdx.x % a.parts), a.parts);
  const float4 st = reinterpret_cast<const float4*>(a.stats)[2 * row];
  const float z = a.stats[8 * row + 4];
  const float g = a.g[row] * a.temp, c = a.inv_t * kLog2e;
  if (g == 0.f || st.z == 0.f || st.y == 0.f) {
    map_row<T>(x, y, sl, [](float) { return 0.f; });
    return;
  }
  for (int k = threadIdx.x; k < K; k += kNT) {
    const int64_t id = a.ids[row * K + k];
    const bool ok = id >= 0 && id < a.rows.V;
    ids[k] = ok ? (int)id : -1;
    q[k] = ok ? ex2((a.values[row * K + k] / a.temp - z) * kLog2e) : 0.f;
  }
  const float other = g * st.y * (st.z - st.w), own = g * st.y * st.z;
  map_row<T>(x, y, sl, [&](float v) { return ex2((v - st.x) * c) * other; });
  __syncthreads();
  // given tokens once more: the first of those with the same index writes for all of them
  for (int k = threadIdx.x; k < K; k += kNT) {
    const int id = ids[k];
    if (id < 0 || !sl.has(id)) continue;
    float sum = 0.f;
    bool first = true;
    for (int j = 0; j < K; ++j)
      if (ids[j] == id) {
        first &= j >= k;
        sum += q[j];
      }
    if (first) y[id] = DT<T>::from_f(fmaf(-g, sum, ex2((DT<T>::to_f(x[id]) - st.x) * c) * own));
  }
}

// ------------------------------------------------------------------------------------------------ host
// CTAs to a row: one where the rows alone fill the SMs, else as many (up to a portable cluster) as do, while each still has a
// batch of requests for its threads.
int parts_of(int64_t rows, int V, int elem) {
  const int64_t batch = (int64_t)kNT * 16 / elem;
  int parts = 1;
  while (parts < kMaxCluster && rows * parts < 148 && (int64_t)V > batch * parts) parts *= 2;
  return parts;
}

template <typename Args>
int launch(void (*kern)(Args), const Args& a, int64_t rows, int parts, bool cluster, size_t smem, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3(kNT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster && parts > 1 ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, kern, a);
}

bool rows_ok(const void* x, int64_t s0, int64_t s1, int64_t n1, int64_t rows, int V, int elem) {
  return x != nullptr && rows >= 1 && rows <= (1ll << 27) && n1 >= 1 && V >= 1 && V <= (1 << 30) && s0 >= 0 && s1 >= 0 &&
         (reinterpret_cast<uintptr_t>(x) % elem) == 0;
}

bool temp_ok(float t) { return t >= 1e-6f && t <= 1e6f; }

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == DT_F16) return f((__half*)nullptr);
  if (dtype == DT_BF16) return f((__nv_bfloat16*)nullptr);
  if (dtype == DT_F32) return f((float*)nullptr);
  return (int)cudaErrorInvalidValue;
}

}  // namespace

// logits: rows of V elements, row r at (r / n1) * s0 + (r % n1) * s1; targets [rows] (`ignore`: no target, all results 0);
// logprob [rows]; entropy [rows] or null; stats [rows, 4] (16-byte aligned) for the backward pass, or null; top tokens
// [rows, top] sorted, equal ones by index (top up to 32 and up to V, 0: none).  A target outside of [0, V) gives NaN and sets
// `err`.  Returns a cudaError_t.
IPEX_API int ipex_token_logprobs(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* targets, float* logprob,
                                 float* entropy, float* stats, float* top_logprob, int64_t* top_id, int64_t rows, int V, int top,
                                 int64_t ignore, float temp, int dtype, int* err, void* stream) {
  if (!rows_ok(logits, s0, s1, n1, rows, V, dtype == DT_F32 ? 4 : 2) || top < 0 || top > kMaxTop || top > V || !temp_ok(temp) ||
      targets == nullptr || logprob == nullptr || (top > 0 && (top_logprob == nullptr || top_id == nullptr)) ||
      (reinterpret_cast<uintptr_t>(stats) & 15))
    return (int)cudaErrorInvalidValue;
  ProbArgs a = {{logits, s0, s1, n1, V}, targets, logprob, entropy, stats, top_logprob, top_id, top, 0, ignore, temp, 1.f / temp, err};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto kern = entropy != nullptr ? (top ? token_logprobs_kernel<T, true, true> : token_logprobs_kernel<T, true, false>)
                                   : (top ? token_logprobs_kernel<T, false, true> : token_logprobs_kernel<T, false, false>);
    return launch<ProbArgs>(kern, a, rows, a.parts, true, 0, (cudaStream_t)stream);
  });
}

// g / g_entropy [rows]: gradients of the log probability and of the entropy (either may be null); dlogits [rows, V].
IPEX_API int ipex_token_logprobs_grad(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* targets,
                                      const float* stats, const float* g, const float* g_entropy, void* dlogits, int64_t rows,
                                      int V, int64_t ignore, float temp, int dtype, void* stream) {
  if (!rows_ok(logits, s0, s1, n1, rows, V, dtype == DT_F32 ? 4 : 2) || !temp_ok(temp) ||
      targets == nullptr || dlogits == nullptr || stats == nullptr || (reinterpret_cast<uintptr_t>(stats) & 15))
    return (int)cudaErrorInvalidValue;
  ProbGradArgs a = {{logits, s0, s1, n1, V}, targets, stats, g, g_entropy, dlogits, ignore, 1.f / temp, 0};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto kern = g_entropy != nullptr ? token_logprobs_grad_kernel<T, true> : token_logprobs_grad_kernel<T, false>;
    return launch<ProbGradArgs>(kern, a, rows, a.parts, false, 0, (cudaStream_t)stream);
  });
}

// ids / values [rows, K]: the teacher's tokens (below 0: none) and their logits, K up to 1024; lse [rows]: logsumexp of the
// teacher's logits / temp, or null; loss [rows]; stats [rows, 8] (16-byte aligned) or null.  V up to 1048576 with lse.
IPEX_API int ipex_distill(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* ids, const float* values,
                          const float* lse, float* loss, float* stats, int64_t rows, int V, int K, float temp, int dtype, int* err,
                          void* stream) {
  if (!rows_ok(logits, s0, s1, n1, rows, V, dtype == DT_F32 ? 4 : 2) || K < 1 || K > kMaxK || !temp_ok(temp) ||
      ids == nullptr || values == nullptr || loss == nullptr || (lse != nullptr && V > (1 << 20)) || (reinterpret_cast<uintptr_t>(stats) & 15))
    return (int)cudaErrorInvalidValue;
  DistillArgs a = {{logits, s0, s1, n1, V}, ids, values, lse, loss, stats, K, 0, temp, 1.f / temp, err};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    if (lse == nullptr) return launch<DistillArgs>(distill_kernel<T, false>, a, rows, a.parts, true, 0, (cudaStream_t)stream);
    const size_t smem = ((size_t)V / a.parts + 64) / 32 * 4 + 16;
    static SmemLimit limit;
    const cudaError_t e = limit((const void*)distill_kernel<T, true>, (1 << 20) / 8 + 64);
    if (e != cudaSuccess) return (int)e;
    return launch<DistillArgs>(distill_kernel<T, true>, a, rows, a.parts, true, smem, (cudaStream_t)stream);
  });
}

IPEX_API int ipex_distill_grad(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* ids, const float* values,
                               const float* stats, const float* g, void* dlogits, int64_t rows, int V, int K, float temp, int dtype,
                               void* stream) {
  if (!rows_ok(logits, s0, s1, n1, rows, V, dtype == DT_F32 ? 4 : 2) || K < 1 || K > kMaxK || !temp_ok(temp) ||
      ids == nullptr || values == nullptr || dlogits == nullptr || stats == nullptr || g == nullptr || (reinterpret_cast<uintptr_t>(stats) & 15))
    return (int)cudaErrorInvalidValue;
  DistillGradArgs a = {{logits, s0, s1, n1, V}, ids, values, stats, g, dlogits, K, 0, temp, 1.f / temp};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return launch<DistillGradArgs>(distill_grad_kernel<T>, a, rows, a.parts, false, 0, (cudaStream_t)stream);
  });
}
