// Losses of preference and policy finetuning straight from logits, with the gradient of the logits.  sm_100a.
//
// log p of a row's target, as in token_loss.cu: with c = log2(e) / T, r = rint(c max x) and s = sum 2^(c x - r),
//   log p_t = x_t / T - (r / c / T + log s)            d log p_t / dx_j = (1[j = t] - p_j) / T
//
// preferred over rejected: S = sum (or mean) of a sequence's log p, h = (S_c - R_c) - (S_r - R_r), z = b h - margin,
//   sigmoid  (1 - e) log(1 + e^-z) + e log(1 + e^z)    dh: b (e sig(z) - (1 - e) sig(-z))
//   hinge    max(0, 1 - b h)                           dh: -b where b h < 1
//   ipo      (h - 1 / 2b)^2                            dh: 2 (h - 1 / 2b)
// policy: w = e^(log p - old), d = ref - log p,
//   -min(w A, min(max(w, 1 - lo), 1 + hi) A) + k (e^d - d - 1)      d log p: -A w where w A is the smaller, + k (1 - e^d)
// (differences of equal numbers are 0, also where both policies hide a target: of -inf)
//
// Prompts and padding have no target: their logits are never read.  A first kernel (or, for few rows, each CTA of the second for itself)
// lists the rows that have one; the second reads them: batches of 32 x 4 vectors of 16 bytes, all rows' behind one another, are dealt to
// the warps in equal runs, whatever rows they belong to, so that no warp waits for another and none has more to do; a run leaves a sum,
// and what its exponents were taken from, for each row that it touches.  The third joins those of a row (up to kSlots) and does what
// comes behind them, in 64 bits.  The backward pass deals its batches the same way, from the last row to the first, then the rows
// without a target, which it only writes.
// All of it is bound by memory: 2042 rows of 128256 in bf16, 1329 of them with a target, take 71 us for the list and the sums (341 MB,
// and what the pass before has left in L2 to be written: 6.3 TB/s) and 133 us for the gradient (865 MB: 6.5 TB/s; writes alone reach
// 3.9); 2048 of 32000, 1287 of them with one, 24 and 35.
#include <cooperative_groups.h>

#include "common/logit_rows.cuh"
#include "common/utils.cuh"
#include "tcgen05_common.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kNT = 256;
constexpr int kU = 4;                       // vectors of a lane in a batch
constexpr int kBatch = 32 * kU;             // vectors of a batch
// To an SM: 64 registers for the sums, which spill 36 to 52 bytes a thread there, 80 for gradients (8 to 24 bytes).  One CTA less of
// each, without spills, is as fast within 2 %: 2048 x 32000 68 and 67 us for both passes, 4096 x 32000 118 and 119.5, 2048 x 128256 214
// and 210.
constexpr int kCtas = 4, kGradCtas = 3;
constexpr int kRun = 16;                    // batches of a warp's run, at most where a warp has many
constexpr int kSlots = 18;                  // runs that may have a part in a row, at most; one of its batches each

// What the forward pass keeps: the rows with a target, then those without, and each row's place among the former (-1: none); the
// what a listed row's exponents are taken from, and 1 / its sum; how a listed row's loss (policy) or a sequence's (preference) moves
// with its log p.
struct Keep {
  int* count;
  int* list;
  int* place;
  float2* stat;
  float* slope;
  float* share;      // of a row's log p in its sequence's
};
__host__ __device__ inline Keep keep_at(void* at, int64_t rows) {
  char* b = reinterpret_cast<char*>(at);
  const int64_t r = (rows + 3) / 4 * 4;
  Keep k;
  k.count = reinterpret_cast<int*>(b);
  k.stat = reinterpret_cast<float2*>(b + 16);
  k.list = reinterpret_cast<int*>(b + 16 + 8 * r);
  k.place = k.list + r;
  k.slope = reinterpret_cast<float*>(k.place + r);
  k.share = k.slope + r;
  return k;
}
constexpr int64_t keep_bytes(int64_t rows) { return 16 + 24 * ((rows + 3) / 4 * 4); }

// How the batches of `count` rows of `per` each are dealt to `warps`: runs of `len`.
struct Deal {
  int64_t total;
  int per, len;
  __device__ Deal(int count, int per_, int warps) : total((int64_t)count * per_), per(per_) {
    const int64_t rounds = max((int64_t)1, (total + (int64_t)warps * kRun - 1) / ((int64_t)warps * kRun));
    const int least = per / (kSlots - 2) + 1;                     // so that kSlots runs reach through a row
    const int64_t even = (total + warps * rounds - 1) / (warps * rounds);
    len = (int)max((int64_t)least, even);
  }
  __device__ int64_t runs() const { return (total + len - 1) / len; }
  __device__ int64_t run_of(int place) const { return (int64_t)place * per / len; }   // the first one with a part in a row
};

__host__ __device__ inline int slots_of(int per) { return per < kSlots ? per : kSlots; }

__host__ __device__ inline int batches_of(int V, int vec) {
  const int nvec = V / vec;
  return nvec > kBatch ? (nvec + kBatch - 1) / kBatch : 1;
}

// A row [V] of any alignment: elements in front of the first 16-byte boundary, vectors, what is left.
template <typename T>
struct Span {
  static constexpr int VEC = 16 / sizeof(T);
  int head, nvec, tail;
  __device__ Span(const void* x, int V) {
    const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15) / (int)sizeof(T);
    head = off ? min(VEC - off, V) : 0;
    nvec = (unsigned)(V - head) / VEC;
    tail = V - head - nvec * VEC;
  }
};

// ------------------------------------------------------------------------------------------------ rows with a target
// Calls put(row, place among the rows with a target so far, whether it has one) for each row, in order of the rows for each thread;
// returns how many have one.  PER rows to a thread at a time.
template <int NT, int PER, typename F>
__device__ __forceinline__ int for_rows(const int64_t* targets, int64_t rows, int64_t ignore, int* sums, F put) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int have = 0;                                       // so far
  for (int64_t at = 0; at < rows; at += NT * PER) {
    const int64_t r0 = at + threadIdx.x * PER;
    bool real[PER];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      real[i] = r0 + i < rows && targets[r0 + i] != ignore;
      mine += real[i];
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int all = lane < NT / 32 ? sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, all, o);
      if (lane >= o) all += v;
    }
    const int before = __shfl_sync(0xffffffffu, all, warp == 0 ? 0 : warp - 1);
    int place = have + (warp == 0 ? 0 : before) + upto - mine;
    have += __shfl_sync(0xffffffffu, all, 31);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (r0 + i >= rows) break;
      put(r0 + i, place, real[i]);
      place += real[i];
    }
    __syncthreads();
  }
  return have;
}
__device__ __forceinline__ void keep_row(const Keep& k, int64_t rows, int64_t row, int place, bool real) {
  k.list[real ? place : rows - 1 - (row - place)] = (int)row;
  k.place[row] = real ? place : -1;
}

constexpr int kListNT = 1024;

__global__ void __launch_bounds__(kListNT) list_rows(const int64_t* targets, int64_t rows, int64_t ignore, void* keep) {
  __shared__ int sums[kListNT / 32];
  pdl_wait();
  pdl_launch_dependents();
  const Keep k = keep_at(keep, rows);
  const int have = for_rows<kListNT, 4>(targets, rows, ignore, sums,
                                        [&](int64_t row, int place, bool real) { keep_row(k, rows, row, place, real); });
  if (threadIdx.x == 0) *k.count = have;
}

// ------------------------------------------------------------------------------------------------ sums
// A lane's part of a row: the sum of 2^(c x - r), r of a logit that none passes by more than 2^kSlack times its share.  It moves, and
// the sum with it, only when one does (with sixteen octaves, the largest terms' exponents lost a place of the result: 7e-7).
constexpr float kSlack = 4.f;
struct Part {
  Base base;
  float s;
};
__device__ __forceinline__ void add_single(Part& p, float v, float c) {
  const Base now(fmaxf(p.base.m, v), c);              // a NaN is not the maximum, and makes the sum one
  p.s = p.s * ex2(shift(p.base, now, c)) + ex2(held(now.exponent(v, c)));
  if (v != v) p.s = v;
  p.base = now;
}
// The largest element of the first `n` vectors; a number before NaN.  16-bit numbers by pairs, as they are.
template <typename T, bool WHOLE>
__device__ __forceinline__ float largest(const uint4* w, int n) {
  if constexpr (std::is_same<T, float>::value) {
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (!WHOLE && u >= n) break;
      float f[4];
      unpack<T>(w[u], f);
      mx = max3(max3(mx, f[0], f[1]), f[2], f[3]);
    }
    return mx;
  } else {
    uint32_t a = max2<T>(w[0].x, w[0].y), b = max2<T>(w[0].z, w[0].w);
#pragma unroll
    for (int u = 1; u < kU; ++u) {
      if (!WHOLE && u >= n) break;
      a = max2<T>(a, max2<T>(w[u].x, w[u].y));
      b = max2<T>(b, max2<T>(w[u].z, w[u].w));
    }
    a = max2<T>(a, b);
    const T* e = reinterpret_cast<const T*>(&a);
    return max3(-INFINITY, DT<T>::to_f(e[0]), DT<T>::to_f(e[1]));
  }
}
template <typename T, bool FAR, bool WHOLE>
__device__ __forceinline__ float sum_of(const uint4* w, int n, const Base& now, float c) {
  constexpr int VEC = 16 / sizeof(T);
  float a[2] = {0.f, 0.f};
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    if (!WHOLE && u >= n) break;
    float f[VEC], v[2] = {0.f, 0.f};
    unpack<T>(w[u], f);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      if (FAR) {
        f[i] = held(now.exponent(f[i], c));
        f[i + 1] = held(now.exponent(f[i + 1], c));
      } else {
        exponents2(f[i], f[i + 1], c, -now.to);
      }
      add2(v[0], v[1], ex2(f[i]), ex2(f[i + 1]));
    }
    add2(a[0], a[1], v[0], v[1]);
  }
  return a[0] + a[1];
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void add_vectors(Part& p, const uint4* w, int n, float c) {
  const float mx = largest<T, WHOLE>(w, n);
  if (!(fmaf(mx, c, -p.base.to) <= kSlack) || p.base.far || p.base.m == -INFINITY) {
    const Base now(fmaxf(p.base.m, mx), c);
    p.s *= ex2(shift(p.base, now, c));
    p.base = now;
  }
  p.s += p.base.far ? sum_of<T, true, false>(w, n, p.base, c) : sum_of<T, false, WHOLE>(w, n, p.base, c);
}
template <typename T>
__device__ __forceinline__ void add_batch(Part& p, const uint4* w, int n, float c) {
  if (n == kU) add_vectors<T, true>(p, w, n, c);
  else if (n > 0) add_vectors<T, false>(p, w, n, c);
}

struct SumArgs {
  Rows rows;
  int64_t n;
  const int64_t* targets;
  int64_t ignore;
  void* keep;
  float2* part;        // [places, slots_of(batches of a row)]
  float inv_t;
};

// LIST: of up to kListed rows, each CTA lists those with a target for itself, and the first one keeps the list: a launch less (2048 rows
// of 32000: 25.0 us with a launch for the list, 24.4 so, and 2 us less of host time; 48 rows of 1000: 5.5 and 4.3).
constexpr int kListed = 2048;

template <typename T, bool LIST>
__global__ void __launch_bounds__(kNT, kCtas) row_sums(SumArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ int sums[kNT / 32];
  __shared__ int own[LIST ? kListed : 1];
  const int lane = threadIdx.x & 31, warps = gridDim.x * (kNT / 32), warp = blockIdx.x * (kNT / 32) + (threadIdx.x >> 5);
  const Keep k = keep_at(a.keep, a.n);
  const float c = a.inv_t * kLog2e;
  pdl_wait();
  pdl_launch_dependents();
  int count;
  if constexpr (LIST) {
    count = for_rows<kNT, kListed / kNT>(a.targets, a.n, a.ignore, sums, [&](int64_t row, int place, bool real) {
      if (real) own[place] = (int)row;
      if (blockIdx.x == 0) keep_row(k, a.n, row, place, real);
    });
    if (blockIdx.x == 0 && threadIdx.x == 0) *k.count = count;
  } else {
    count = *k.count;
  }
  const int* list = LIST ? own : k.list;
  const Deal deal(count, batches_of(a.rows.V, VEC), warps);
  for (int64_t run = warp; run < deal.runs(); run += warps) {
    int64_t at = run * deal.len;
    const int64_t end = min(at + deal.len, deal.total);
    int place = (int)(at / deal.per), b = (int)(at - (int64_t)place * deal.per);
    for (; at < end; ++place, b = 0) {
      const T* x = row_at<T>(a.rows, list[place]);
      const Span<T> sp(x, a.rows.V);
      const int b1 = (int)min((int64_t)deal.per, b + (end - at));
      at += b1 - b;
      const uint4* xv = reinterpret_cast<const uint4*>(x + sp.head) + lane;
      // vectors of this lane, 32 apart, from `from` on
      auto count = [&](int from) { return min(kU, (sp.nvec - from - lane + 31) / 32); };
      auto load = [&](uint4* w, int b) {
        const int from = b * kBatch;
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (from + u * 32 + lane < sp.nvec) w[u] = ldg_nc_v4(xv + from + u * 32);
      };
      uint4 w[kU], v[kU];
      load(w, b);
      Part p = {Base(-INFINITY, c), 0.f};
      if (b == 0 && lane < sp.head) add_single(p, DT<T>::to_f(x[lane]), c);
      if (b1 == deal.per && lane < sp.tail) add_single(p, DT<T>::to_f(x[a.rows.V - sp.tail + lane]), c);
      while (true) {                                  // a batch is asked for while the one in front of it is added
        if (b + 1 < b1) load(v, b + 1);
        add_batch<T>(p, w, count(b * kBatch), c);
        if (++b >= b1) break;
        if (b + 1 < b1) load(w, b + 1);
        add_batch<T>(p, v, count(b * kBatch), c);
        if (++b >= b1) break;
      }
      // all taken to the largest base, then added up
      float m;
      asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(p.base.m));
      float s = p.s * ex2(shift(p.base, Base(m, c), c));
#pragma unroll
      for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) a.part[(int64_t)place * slots_of(deal.per) + (int)(run - deal.run_of(place))] = make_float2(m, s);
    }
  }
}

// ------------------------------------------------------------------------------------------------ what comes behind the sums
// A listed row's statistics from its parts, and log p of its target.
struct RowArgs {
  Rows rows;
  const int64_t* targets;
  int64_t n;
  void* keep;
  const float2* part;
  int warps, per;      // of the sums' launch
  float temp, inv_t;
  int* err;
};

template <typename T>
__device__ __forceinline__ double row_logprob(const RowArgs& a, const Keep& k, const Deal& deal, int64_t row, int place) {
  const float c = a.inv_t * kLog2e;
  const int64_t t = a.targets[row];
  const bool bad = t < 0 || t >= a.rows.V;
  const float xt = bad ? 0.f : DT<T>::to_f(row_at<T>(a.rows, row)[t]);
  const int parts = (int)(((int64_t)(place + 1) * deal.per - 1) / deal.len - deal.run_of(place)) + 1;
  const float2* at = a.part + (int64_t)place * slots_of(deal.per);
  float2 p[kSlots];
  Stat st = {-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kSlots; ++i)
    if (i < parts) p[i] = at[i];
#pragma unroll
  for (int i = 0; i < kSlots; ++i)
    if (i < parts) st.m = fmaxf(st.m, p[i].x);
  const Base to(st.m, c);
#pragma unroll
  for (int i = 0; i < kSlots; ++i)
    if (i < parts) st.s += p[i].y * ex2(shift(Base(p[i].x, c), to, c));
  const bool none = no_token(st);
  const Base base(none ? 0.f : st.m, c);
  k.stat[place] = make_float2(base.m, none ? 0.f : bad ? NAN : 1.f / st.s);
  if (bad) {
    tc5::report(a.err, kErrToken);
    return NAN;
  }
  if (none) return -INFINITY;
  const double log2_s = log2((double)st.s), lse = log_sum(base, log2_s, c, a.temp);
  if (base.far) return ((double)xt - base.m) / a.temp - lse;
  return fabsf(xt) < INFINITY ? xt / (double)a.temp - lse : (double)(xt - (float)log2_s);
}

struct PolicyArgs {
  RowArgs row;
  const float* old;       // [rows] or null: log p itself
  const float* ref;       // [rows] or null
  const float* adv;       // strides of outer and inner index
  int64_t adv0, adv1, inner;
  float* loss;
  float* logprob;
  float* kl;
  uint8_t* clipped;
  double lo, hi, weight;
};

__device__ __forceinline__ double apart(double a, double b) { return a == b ? 0.0 : a - b; }

template <typename T>
__global__ void __launch_bounds__(128) policy_rows(PolicyArgs a) {
  const Keep k = keep_at(a.row.keep, a.row.n);
  pdl_wait();
  const Deal deal(*k.count, a.row.per, a.row.warps);
  const int64_t row = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (row >= a.row.n) return;
  const int place = k.place[row];
  float loss = 0.f, kl = 0.f, slope = 0.f;
  double lp = 0.0;
  bool clipped = false;
  if (place >= 0) {
    lp = row_logprob<T>(a.row, k, deal, row, place);
    const double A = a.adv[row / a.inner * a.adv0 + row % a.inner * a.adv1];
    const double w = a.old != nullptr ? exp(apart(lp, a.old[row])) : lp == lp ? 1.0 : lp;
    const double inside = w < 1.0 - a.lo ? 1.0 - a.lo : w > 1.0 + a.hi ? 1.0 + a.hi : w;      // NaN stays
    clipped = inside * A < w * A;
    double l = -(clipped ? inside * A : w * A), g = clipped ? 0.0 : -A * w;
    if (a.ref != nullptr) {
      const double d = apart(a.ref[row], lp), e = expm1(d), est = e < INFINITY ? e - d : e;
      kl = (float)est;
      if (a.weight != 0.0) {
        l += a.weight * est;
        g -= a.weight * e;
      }
    }
    if (lp == -INFINITY) g = 0.0;                     // a hidden target: no other logit brings it back
    loss = (float)l;
    slope = (float)g;
  }
  a.loss[row] = loss;
  a.logprob[row] = (float)lp;
  a.kl[row] = kl;
  a.clipped[row] = clipped;
  k.slope[row] = slope;
}

enum { FORM_SIGMOID = 0, FORM_HINGE = 1, FORM_IPO = 2 };

struct PairArgs {
  RowArgs row;
  const float* reference;   // [2 pairs] or null
  int64_t tokens;
  int pairs, form, average;
  double beta, smooth, margin;
  float* loss;              // [pairs]
  float* logprob;           // [2 pairs]
};

constexpr int kPairNT = 256, kPairCtas = 8;

// A cluster of eight CTAs to a pair: half of them to each sequence.
template <typename T>
__global__ void __cluster_dims__(kPairCtas, 1, 1) __launch_bounds__(kPairNT) pair_losses(PairArgs a) {
  __shared__ double sums[kPairNT / 32];
  __shared__ int counts[kPairNT / 32];
  __shared__ double sum;
  __shared__ int count;
  const Keep k = keep_at(a.row.keep, a.row.n);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = blockIdx.x % kPairCtas, pair = blockIdx.x / kPairCtas;
  const int half = rank / (kPairCtas / 2), part = rank % (kPairCtas / 2);
  pdl_wait();
  const Deal deal(*k.count, a.row.per, a.row.warps);
  const int64_t r0 = ((int64_t)half * a.pairs + pair) * a.tokens;
  double s = 0.0;
  int n = 0;
  for (int64_t t = part * kPairNT + threadIdx.x; t < a.tokens; t += kPairNT * (kPairCtas / 2)) {
    const int place = k.place[r0 + t];
    if (place < 0) continue;
    s += row_logprob<T>(a.row, k, deal, r0 + t, place);
    ++n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if (lane == 0) {
    sums[warp] = s;
    counts[warp] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPairNT / 32; ++w) {
      s += sums[w];
      n += counts[w];
    }
    sum = s;
    count = n;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  double S[2] = {0.0, 0.0};
  int N[2] = {0, 0};
  if (rank == 0 && threadIdx.x == 0)
    for (int i = 0; i < kPairCtas; ++i) {
      S[i / (kPairCtas / 2)] += *cl.map_shared_rank(&sum, i);
      N[i / (kPairCtas / 2)] += *cl.map_shared_rank(&count, i);
    }
  cl.sync();
  if (rank != 0 || threadIdx.x != 0) return;
  double share[2];
  for (int h = 0; h < 2; ++h) {
    share[h] = a.average ? 1.0 / max(N[h], 1) : 1.0;
    S[h] *= share[h];
  }
  const int c = pair, r = pair + a.pairs;
  const double h = (S[0] - (a.reference == nullptr ? 0.0 : a.reference[c])) - (S[1] - (a.reference == nullptr ? 0.0 : a.reference[r]));
  double loss, d;
  if (a.form == FORM_SIGMOID) {
    const double z = a.beta * h - a.margin, e = exp(-fabs(z)), near = log1p(e), small = e / (1.0 + e), large = 1.0 / (1.0 + e);
    const double minus = near + fmax(-z, 0.0), plus = near + fmax(z, 0.0);      // log(1 + e^-z), log(1 + e^z)
    const double up = z >= 0.0 ? large : small, down = z >= 0.0 ? small : large;
    loss = (1.0 - a.smooth) * minus + (a.smooth == 0.0 ? 0.0 : a.smooth * plus);
    d = a.beta * (a.smooth * up - (1.0 - a.smooth) * down);
    if (z != z) loss = d = z;
  } else if (a.form == FORM_HINGE) {
    const double z = 1.0 - a.beta * h;
    loss = z < 0.0 ? 0.0 : z;
    d = z > 0.0 ? -a.beta : z != z ? z : 0.0;
  } else {
    const double z = h - 0.5 / a.beta;
    loss = z * z;
    d = 2.0 * z;
  }
  a.loss[c] = (float)loss;
  a.logprob[c] = (float)S[0];
  a.logprob[r] = (float)S[1];
  k.slope[c] = (float)(d * share[0]);
  k.slope[r] = (float)(-d * share[1]);
  k.share[c] = (float)share[0];
  k.share[r] = (float)share[1];
}

// ------------------------------------------------------------------------------------------------ gradient
struct GradArgs {
  Rows rows;
  const int64_t* targets;
  int64_t n;
  const void* keep;
  const float* g;           // of the loss: strides of outer and inner index; null: none
  int64_t g0, g1, inner;    // inner: of g's rows; preference: tokens of a sequence
  const float* g_seq;       // of the sequences' log p, or null
  int pairs;                // 0: policy
  void* dx;
  float inv_t;
};

__device__ __forceinline__ void times2(float& x, float& y, float a) {
  asm("{\n.reg .b64 p, q;\nmov.b64 p, {%0, %1};\nmov.b64 q, {%2, %2};\nmul.rn.f32x2 p, p, q;\nmov.b64 {%0, %1}, p;\n}\n" : "+f"(x), "+f"(y) : "f"(a));
}
// scale 2^(c x - r) of a vector's elements.
template <typename T>
__device__ __forceinline__ uint4 shares(const uint4& w, float c, float minus_r, float scale) {
  constexpr int VEC = 16 / sizeof(T);
  float f[VEC];
  unpack<T>(w, f);
  uint4 o;
  T* to = reinterpret_cast<T*>(&o);
#pragma unroll
  for (int i = 0; i < VEC; i += 2) {
    exponents2(f[i], f[i + 1], c, minus_r);
    f[i] = ex2(f[i]);
    f[i + 1] = ex2(f[i + 1]);
    times2(f[i], f[i + 1], scale);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      *reinterpret_cast<__nv_bfloat162*>(to + i) = __floats2bfloat162_rn(f[i], f[i + 1]);
    } else if constexpr (std::is_same<T, __half>::value) {
      *reinterpret_cast<__half2*>(to + i) = __floats2half2_rn(f[i], f[i + 1]);
    } else {
      to[i] = f[i];
      to[i + 1] = f[i + 1];
    }
  }
  return o;
}

template <typename T>
__global__ void __launch_bounds__(kNT, kGradCtas) row_grads(GradArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  const int lane = threadIdx.x & 31, warps = gridDim.x * (kNT / 32), warp = blockIdx.x * (kNT / 32) + (threadIdx.x >> 5);
  const Keep k = keep_at(const_cast<void*>(a.keep), a.n);
  const float c = a.inv_t * kLog2e;
  pdl_wait();
  const int V = a.rows.V, count = *k.count;
  T* dx = reinterpret_cast<T*>(a.dx);
  const Deal deal(count, batches_of(V, VEC), warps);
  for (int64_t back = warp; back < deal.runs(); back += warps) {
    const int64_t run = deal.runs() - 1 - back;
    int64_t at = run * deal.len;
    const int64_t end = min(at + deal.len, deal.total);
    int place = (int)(at / deal.per), b = (int)(at - (int64_t)place * deal.per);
    for (; at < end; ++place, b = 0) {
      const int64_t row = k.list[place];
      const T* x = row_at<T>(a.rows, row);
      T* y = dx + row * V;
      const Span<T> sp(x, V);
      const int b1 = (int)min((int64_t)deal.per, b + (end - at));
      at += b1 - b;
      const uint4* xv = reinterpret_cast<const uint4*>(x + sp.head) + lane;
      uint4* yv = reinterpret_cast<uint4*>(y + sp.head) + lane;
      auto load = [&](uint4* w, int b) {
        const int from = b * kBatch;
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (from + u * 32 + lane < sp.nvec) w[u] = ldg_nc_v4(xv + from + u * 32);
      };
      uint4 w[kU], v[kU];
      load(w, b);
      const float2 st = k.stat[place];
      const int64_t t = a.targets[row];
      float g = 0.f;
      if (a.pairs > 0) {
        const int64_t seq = row / a.inner;
        if (a.g != nullptr) g = a.g[(seq < a.pairs ? seq : seq - a.pairs) * a.g0] * k.slope[seq];
        if (a.g_seq != nullptr) g += a.g_seq[seq] * k.share[seq];
      } else {
        g = a.g[row / a.inner * a.g0 + row % a.inner * a.g1] * k.slope[row];
      }
      if (st.y == 0.f) g = 0.f;                       // no token in the row
      const Base base(st.x, c);
      const float scale = -g * st.y * a.inv_t;
      const bool nothing = g == 0.f;                  // flows into the row, whatever its logits hold
      const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0;
      auto one = [&](int j) {
        const float f = DT<T>::to_f(x[j]);
        const float e = nothing ? 0.f : ex2(base.exponent(f, c)) * scale;
        y[j] = DT<T>::from_f(j == t && !nothing ? fmaf(g, a.inv_t, e) : e);
      };
      if (b == 0 && lane < sp.head) one(lane);
      if (b1 == deal.per && lane < sp.tail) one(V - sp.tail + lane);
      const int v0 = b * kBatch, v1 = min(b1 * kBatch, sp.nvec);
      if (nothing) {
        for (int i = v0 + lane; i < v1; i += 32) {
          if (alike) {
            __stcs(yv + i - lane, make_uint4(0, 0, 0, 0));
          } else {
            for (int e = 0; e < VEC; ++e) y[sp.head + (int64_t)i * VEC + e] = DT<T>::from_f(0.f);
          }
        }
      } else if (alike && !base.far) {
        auto store = [&](const uint4* w, int b) {
          const int from = b * kBatch;
#pragma unroll
          for (int u = 0; u < kU; ++u)
            if (from + u * 32 + lane < sp.nvec) __stcs(yv + from + u * 32, shares<T>(w[u], c, -base.r, scale));     // nothing here reads them again
        };
        while (true) {                                // a batch is asked for while the one in front of it is worked on
          if (b + 1 < b1) load(v, b + 1);
          store(w, b);
          if (++b >= b1) break;
          if (b + 1 < b1) load(w, b + 1);
          store(v, b);
          if (++b >= b1) break;
        }
      } else {
        for (int i = v0 + lane; i < v1; i += 32)
          for (int e = 0; e < VEC; ++e) one(sp.head + i * VEC + e);
      }
      // the target once more, by the lane that has written it
      const int64_t at_t = t - sp.head;
      if (!nothing && at_t >= (int64_t)v0 * VEC && at_t < (int64_t)v1 * VEC && (at_t / VEC - v0) % 32 == lane) one((int)t);
    }
  }
  // rows without a target
  const int per = deal.per;
  const int64_t rest = (a.n - count) * per;
  for (int64_t at = warp; at < rest; at += warps) {
    const int64_t i = at / per;
    const int b = (int)(at - i * per);
    T* y = dx + (int64_t)k.list[count + i] * V;
    const Span<T> sp(y, V);
    const T zero = DT<T>::from_f(0.f);
    if (b == 0 && lane < sp.head) y[lane] = zero;
    if (b == per - 1 && lane < sp.tail) y[V - sp.tail + lane] = zero;
    uint4* yv = reinterpret_cast<uint4*>(y + sp.head);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int v = b * kBatch + u * 32 + lane;
      if (v < sp.nvec) __stcs(yv + v, make_uint4(0, 0, 0, 0));
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
int elem_of(int dtype) { return dtype == DT_F32 ? 4 : 2; }

// CTAs that stay, or as many as there are batches for.
int grid_of(int64_t rows, int V, int elem, int64_t most) {
  const int64_t batches = rows * batches_of(V, 16 / elem), ctas = (batches + kNT / 32 - 1) / (kNT / 32);
  return (int)(ctas < most ? ctas : most);
}

// CTAs of the backward pass: SMs do not all run at one speed, so that more are launched than stay, up to eight times as many, while
// each warp still has eight batches (2042 rows of 128256: 148 us with those that stay, 139 with four times as many, 133 with eight;
// 2048 of 32000: 35.8, 35.8 and 37.7, and 35.2 with twice as many).  The sums gain nothing (69 to 72 us): their ends cost more.
int grad_grid_of(int64_t rows, int V, int elem) {
  const int64_t stay = (int64_t)sm_count() * kGradCtas, times = rows * batches_of(V, 16 / elem) / (stay * (kNT / 32) * 8);
  return grid_of(rows, V, elem, stay * (times < 1 ? 1 : times > 8 ? 8 : times));
}

// The list and the sums; then `a` is ready for the kernel behind them.
int forward(RowArgs& a, int64_t ignore, int dtype, cudaStream_t s) {
  if (sm_count() == 0) return (int)cudaErrorInvalidDevice;
  const int grid = grid_of(a.n, a.rows.V, elem_of(dtype), (int64_t)sm_count() * kCtas);
  a.warps = grid * (kNT / 32);
  a.per = batches_of(a.rows.V, 16 / elem_of(dtype));
  const bool list = a.n <= kListed;
  if (!list) {
    const cudaError_t e = launch_kernel(list_rows, dim3(1), dim3(kListNT), 0, s, true, a.targets, a.n, ignore, a.keep);
    if (e != cudaSuccess) return (int)e;
  }
  const SumArgs sums = {a.rows, a.n, a.targets, ignore, a.keep, const_cast<float2*>(a.part), a.inv_t};
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return (int)launch_kernel(list ? row_sums<T, true> : row_sums<T, false>, dim3(grid), dim3(kNT), 0, s, true, sums);
  });
}

int backward(const GradArgs& a, int dtype, cudaStream_t s) {
  if (sm_count() == 0) return (int)cudaErrorInvalidDevice;
  return by_type(dtype, [&](auto* tag) {
    return (int)launch_kernel(row_grads<std::remove_pointer_t<decltype(tag)>>, dim3(grad_grid_of(a.n, a.rows.V, elem_of(dtype))), dim3(kNT),
                              0, s, true, a);
  });
}

bool args_ok(const void* logits, int64_t s0, int64_t s1, int64_t n1, int64_t rows, int V, float temp, int dtype, const void* targets,
             const void* keep) {
  return rows_ok(logits, s0, s1, n1, rows, V, elem_of(dtype)) && temp_ok(temp) && targets != nullptr && keep != nullptr &&
         (reinterpret_cast<uintptr_t>(keep) & 15) == 0;
}

}  // namespace

// Bytes that the forward pass keeps for the backward one, and those that it works in.
IPEX_API int64_t ipex_preference_keep_bytes(int64_t rows) { return keep_bytes(rows); }
IPEX_API int64_t ipex_preference_work_bytes(int64_t rows, int V, int dtype) {
  return rows * slots_of(batches_of(V, 16 / elem_of(dtype))) * (int64_t)sizeof(float2);
}

// logits: rows of V elements, row r at (r / n1) * s0 + (r % n1) * s1; targets [rows] (`ignore`: none, all results 0); old, ref [rows] or
// null; advantage of row r at (r / inner) * adv0 + (r % inner) * adv1; loss, logprob, kl (0 without ref), clipped [rows].  A target
// outside of [0, V) gives NaN and sets `err`.  Returns a cudaError_t.
IPEX_API int ipex_policy_loss(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* targets, const float* old,
                              const float* ref, const float* adv, int64_t adv0, int64_t adv1, int64_t inner, float* loss,
                              float* logprob, float* kl, uint8_t* clipped, void* keep, void* work, int64_t rows, int V, int64_t ignore,
                              double lo, double hi, double weight, float temp, int dtype, int* err, void* stream) {
  if (!args_ok(logits, s0, s1, n1, rows, V, temp, dtype, targets, keep) || work == nullptr || adv == nullptr || inner < 1 ||
      loss == nullptr || logprob == nullptr || clipped == nullptr || kl == nullptr)
    return (int)cudaErrorInvalidValue;
  RowArgs r = {rows_of(logits, s0, s1, n1, rows, V), targets, rows, keep, (const float2*)work, 0, 0, temp, 1.f / temp, err};
  const int rc = forward(r, ignore, dtype, (cudaStream_t)stream);
  if (rc != 0) return rc;
  const PolicyArgs a = {r, old, ref, adv, adv0, adv1, inner, loss, logprob, kl, clipped, lo, hi, weight};
  return by_type(dtype, [&](auto* tag) {
    return (int)launch_kernel(policy_rows<std::remove_pointer_t<decltype(tag)>>, dim3((unsigned)((rows + 127) / 128)), dim3(128), 0,
                              (cudaStream_t)stream, true, a);
  });
}

// g: the loss's gradient, of row r at (r / inner) * g0 + (r % inner) * g1; dlogits [rows, V].
IPEX_API int ipex_policy_grad(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* targets, const void* keep,
                              const float* g, int64_t g0, int64_t g1, int64_t inner, void* dlogits, int64_t rows, int V, float temp,
                              int dtype, void* stream) {
  if (!args_ok(logits, s0, s1, n1, rows, V, temp, dtype, targets, keep) || g == nullptr || inner < 1 || dlogits == nullptr)
    return (int)cudaErrorInvalidValue;
  const GradArgs a = {rows_of(logits, s0, s1, n1, rows, V), targets, rows, keep, g, g0, g1, inner, nullptr, 0, dlogits, 1.f / temp};
  return backward(a, dtype, (cudaStream_t)stream);
}

// 2 pairs x tokens rows, the preferred sequences first; reference [2 pairs] or null; form: 0 sigmoid, 1 hinge, 2 ipo; loss [pairs],
// logprob [2 pairs].
IPEX_API int ipex_preference_loss(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* targets,
                                  const float* reference, float* loss, float* logprob, void* keep, void* work, int pairs,
                                  int64_t tokens, int V, int64_t ignore, int form, int average, double beta, double smooth,
                                  double margin, float temp, int dtype, int* err, void* stream) {
  const int64_t rows = 2 * (int64_t)pairs * tokens;
  if (!args_ok(logits, s0, s1, n1, rows, V, temp, dtype, targets, keep) || work == nullptr || loss == nullptr || logprob == nullptr ||
      pairs < 1 || form < 0 || form > 2 || !(beta > 0.0))
    return (int)cudaErrorInvalidValue;
  RowArgs r = {rows_of(logits, s0, s1, n1, rows, V), targets, rows, keep, (const float2*)work, 0, 0, temp, 1.f / temp, err};
  const int rc = forward(r, ignore, dtype, (cudaStream_t)stream);
  if (rc != 0) return rc;
  const PairArgs a = {r, reference, tokens, pairs, form, average, beta, smooth, margin, loss, logprob};
  return by_type(dtype, [&](auto* tag) {
    return (int)launch_kernel(pair_losses<std::remove_pointer_t<decltype(tag)>>, dim3((unsigned)pairs * kPairCtas), dim3(kPairNT), 0,
                              (cudaStream_t)stream, true, a);
  });
}

// g [pairs] (every g0-th) and g_seq [2 pairs]: gradients of the losses and of the sequences' log p; either may be null.
IPEX_API int ipex_preference_grad(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* targets, const void* keep,
                                  const float* g, int64_t g0, const float* g_seq, void* dlogits, int pairs, int64_t tokens, int V,
                                  float temp, int dtype, void* stream) {
  const int64_t rows = 2 * (int64_t)pairs * tokens;
  if (!args_ok(logits, s0, s1, n1, rows, V, temp, dtype, targets, keep) || dlogits == nullptr || pairs < 1)
    return (int)cudaErrorInvalidValue;
  const GradArgs a = {rows_of(logits, s0, s1, n1, rows, V), targets, rows, keep, g, g0, 0, tokens, g_seq, pairs, dlogits, 1.f / temp};
  return backward(a, dtype, (cudaStream_t)stream);
}
