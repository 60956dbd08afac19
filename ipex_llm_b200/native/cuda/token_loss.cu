// What stands behind an output layer: log probabilities of given tokens with their entropy and the best alternatives, and
// the divergence from a teacher's top logits, each with the gradient of the logits.  sm_100a.
//
// With y = x / T, m = max x, s = sum e^((x - m) / T), t = sum e^((x - m) / T) (x - m):
//
//   log p_j = (x_j - m) / T - ln s            H = ln s - t / (s T)
//   d log p_t / dx_j = (1[j = t] - p_j) / T   dH / dx_j = -p_j (log p_j + H) / T
//
// All of them are bound by memory: forward reads a row once, backward reads it once more and writes it once.  A row belongs
// to one CTA (many rows; the CTAs stay and take the next row) or to a cluster of up to eight (few rows).  Each thread copies its
// own four 16-byte vectors at a time to shared memory, asynchronously and two batches ahead, into the next row while a row's
// parts are joined: without that, loads waited for arithmetic and arithmetic for loads (2048 rows of 32000 in bf16: 53 us).
// A thread folds the maximum of a batch into its own and rescales its sums once for all of it, so that an element costs one
// exponential (0.73 of what the special function units do at the rate of memory, for 16-bit logits).
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

__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_end_batch() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {      // until all but the newest N batches have come
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

// The vectors of a CTA's rows as a stream of batches, each thread's four to a batch, kStages batches ahead of their use.
constexpr int kStages = 2;
constexpr int kRing = kStages * kU * kNT * 16;

template <typename T>
struct Feed {
  const Rows& rows;
  uint4* ring;
  int64_t row, step, end;      // the row that is fetched, the distance to the next one, all of them
  int rank, parts;
  int at, v1, slot;            // next vector of this thread, the end of the row's, the next batch's place
  const uint4* xv;
  __device__ Feed(const Rows& r, uint4* ring_, int64_t first, int64_t step_, int64_t end_, int rank_, int parts_)
      : rows(r), ring(ring_ + threadIdx.x), row(first), step(step_), end(end_), rank(rank_), parts(parts_), slot(0) {
    open();
    for (int i = 0; i < kStages; ++i) fetch();
  }
  __device__ void open() {
    if (row >= end) return;
    const T* x = row_at<T>(rows, row);
    const Slice<T> sl(x, rows.V, rank, parts);
    xv = reinterpret_cast<const uint4*>(x + sl.head);
    at = sl.v0;
    v1 = sl.v1;
  }
  __device__ void fetch() {
    if (row < end) {
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (at + u * kNT + (int)threadIdx.x < v1) copy_async(ring + (slot * kU + u) * kNT, xv + at + u * kNT + threadIdx.x);
      at += kU * kNT;
      if (at >= v1) {
        row += step;
        open();
      }
    }
    copies_end_batch();
    slot = slot + 1 == kStages ? 0 : slot + 1;
  }
  // The oldest batch, whose first vector is `first` of a row that ends at `last`; fetches the next one into its place.
  __device__ void take(int first, int last, uint4 (&w)[kU]) {
    copies_wait<kStages - 1>();
#pragma unroll
    for (int u = 0; u < kU; ++u)
      w[u] = first + u * kNT + (int)threadIdx.x < last ? ring[(slot * kU + u) * kNT] : hidden<T>();
    fetch();
  }
};

struct Shared {
  Stat warp[kWarps];
  Stat part;                      // this CTA's
  uint64_t best[kNT];             // the threads' best keys, sorted in each warp
  uint64_t cand[kCand];
  uint64_t top[kMaxTop];          // this CTA's best, sorted
  uint64_t thr;
  int n_cand, n_list;
  int list[kNT];                  // threads that may hold one of the best
};

// A thread's best element: its value, and where it is: in the batch whose first vector of this thread is `at`, or alone at -2 - at;
// -1: it has none.
struct Best {
  float v;
  int at;
};

// A row's statistics into sh.part, TOP: this thread's best.
template <typename T, bool ENT, bool TOP, bool TAIL>
__device__ void scan(const T* x, const Slice<T>& sl, float c, Feed<T>& feed, const uint32_t* given, const int* ids, int K, Shared& sh,
                     Best& best) {
  constexpr int VEC = Slice<T>::VEC;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Stat st = {-INFINITY, 0.f, 0.f};
  best = {0.f, -1};
  auto single = [&](int j) {
    const float v = DT<T>::to_f(x[j]);
    bool is_given = false;
    if constexpr (TAIL)
      for (int k = 0; k < K; ++k) is_given |= ids[k] == j;
    Stat one = {v, 1.f, TAIL && !is_given ? 1.f : 0.f};
    if (v == -INFINITY) one.s = one.t = 0.f;
    if (v != v) one.s = one.t = v;
    st = join<ENT>(st, one, c);
    if (TOP && (best.at == -1 || order_key(v, 0) > order_key(best.v, 0))) best = {v, -2 - j};
  };
  if (tid < sl.h) single(tid);
  // as the feed does: at least one batch a row, whether it holds vectors or not
  for (int base = sl.v0; base == sl.v0 || base < sl.v1; base += kNT * kU) {
    uint4 w[kU];
    feed.take(base, sl.v1, w);
    if (base + tid >= sl.v1) continue;
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
        const int pos = (min(base + u * kNT + tid, sl.v1 - 1) - sl.v0) * VEC;
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
      if (best.at == -1 || order_key(mx, 0) > order_key(best.v, 0)) best = {mx, base + tid};
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
  __syncthreads();
  if (tid == 0) {
    Stat a = sh.warp[0];
    for (int i = 1; i < kWarps; ++i) a = join<ENT>(a, sh.warp[i], c);
    sh.part = a;
  }
}

// Keys of a warp: sorted from large to small over its lanes, and the 32 largest of two such rows of lanes.
__device__ __forceinline__ uint64_t exchange(uint64_t k, int o, bool keep_large) {
  const uint64_t w = __shfl_xor_sync(0xffffffffu, k, o);
  return (k > w) == keep_large ? k : w;
}
__device__ __forceinline__ uint64_t warp_sort(uint64_t k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o > 0; o /= 2) k = exchange(k, o, ((lane & o) == 0) == ((lane & size) == 0 || size == 32));
  return k;
}
__device__ __forceinline__ uint64_t warp_merge(uint64_t a, uint64_t b, int lane) {   // b: the other row, read backwards
  uint64_t k = a > b ? a : b;
#pragma unroll
  for (int o = 16; o > 0; o /= 2) k = exchange(k, o, (lane & o) == 0);
  return k;
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

// The 32 largest of the CTA's keys, sorted, in the lanes of the first warp.
__device__ uint64_t largest32(uint64_t k, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  k = warp_sort(k, lane);
  __syncthreads();
  sh.best[threadIdx.x] = k;
#pragma unroll
  for (int n = kWarps / 2; n > 0; n /= 2) {
    __syncthreads();
    if (warp < n) {
      k = warp_merge(k, sh.best[(warp + n) * 32 + 31 - lane], lane);
      sh.best[threadIdx.x] = k;
    }
  }
  return k;
}

// The `top` largest keys of a slice, sorted, into sh.top (0 behind the last element).  The top-th largest of the threads' best keys
// bounds them from below, and only the threads that reach it (top of them, keys being unique) can hold any: their elements are read
// again, sixteen lanes to a thread, and what reaches the bound is ranked by counting.  Values nearly always decide; where several
// threads have the bound's, these look up where they have it (the lower index comes first).  Where more than kCand elements
// reach it (a few threads hold nearly all large values), the slice is scanned once for each rank instead.
template <typename T>
__device__ void best_tokens(const T* x, const Slice<T>& sl, int top, const Best& best, Shared& sh) {
  constexpr int VEC = Slice<T>::VEC;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kMaxTop) sh.top[tid] = 0;
  if (tid == 0) sh.n_cand = sh.n_list = 0;
  uint64_t mine = best.at == -1 ? 0 : order_key(best.v, tid);
  uint64_t k = largest32(mine, sh);
  if (tid == top - 1) sh.thr = k >> 32 << 32;       // the value alone: below every key that has it
  __syncthreads();
  uint64_t thr = sh.thr;
  if (__syncthreads_count(mine != 0 && mine >= thr) > top) {
    if (mine != 0 && mine >> 32 == thr >> 32) {
      if (best.at < 0) {
        mine = order_key(best.v, -2 - best.at);
      } else {
        mine = 0;
        const uint4* xv = reinterpret_cast<const uint4*>(x + sl.head);
        for (int v = best.at; v < min(best.at + kU * kNT, sl.v1); v += kNT) {
          float f[VEC];
          unpack<T>(ldg_nc_v4(xv + v), f);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const uint64_t key = order_key(f[i], sl.head + v * VEC + i);
            mine = key > mine ? key : mine;
          }
        }
      }
    }
    k = largest32(mine, sh);
    if (tid == top - 1) sh.thr = k;
    __syncthreads();
    thr = sh.thr;
  }
  if (mine != 0 && mine >= thr) sh.list[atomicAdd(&sh.n_list, 1)] = tid;
  __syncthreads();
  const int n_list = sh.n_list;
  for (int i = tid >> 4; i < n_list; i += kNT / 16)
    elements_of<T>(x, sl, sh.list[i], tid & 15, 16, [&](float v, int j) {
      const uint64_t key = order_key(v, j);
      if (key >= thr) {
        const int at = atomicAdd(&sh.n_cand, 1);
        if (at < kCand) sh.cand[at] = key;
      }
    });
  __syncthreads();
  const int n = sh.n_cand;
  if (n <= kCand) {
    for (int i = tid; i < n; i += kNT) {
      const uint64_t key = sh.cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += sh.cand[j] > key;
      if (r < top) sh.top[r] = key;
    }
    __syncthreads();
    return;
  }
  uint64_t under = ~0ull;
  for (int r = 0; r < top; ++r) {
    uint64_t b = 0;
    elements_of<T>(x, sl, tid, 0, 1, [&](float v, int j) {
      const uint64_t key = order_key(v, j);
      if (key < under && key > b) b = key;
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
  int64_t ignore, n;   // n rows
  float temp, inv_t;
  int* err;
};

template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kNT, 2) token_logprobs_kernel(ProbArgs a) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Shared sh;
  const int parts = a.parts, rank = parts == 1 ? 0 : (int)(blockIdx.x % parts);
  const int64_t step = gridDim.x / parts;
  const float c = a.inv_t * kLog2e;
  Feed<T> feed(a.rows, reinterpret_cast<uint4*>(dynamic), blockIdx.x / parts, step, a.n, rank, parts);
  for (int64_t row = blockIdx.x / parts; row < a.n; row += step) {
    const T* x = row_at<T>(a.rows, row);
    const Slice<T> sl(x, a.rows.V, rank, parts);
    Best best;
    scan<T, ENT, TOP, false>(x, sl, c, feed, nullptr, nullptr, 0, sh, best);
    if constexpr (TOP) best_tokens<T>(x, sl, a.top, best, sh);
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
    else __syncthreads();
  }
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
  float* stats;            // [rows, 8]: m, 1 / s, M, rest / left, z, share, -, -
  int64_t n;               // rows
  int K, parts;
  float temp, inv_t;
  int* err;
};

__device__ __forceinline__ double block_reduce(double v, bool is_max, double* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double w = __shfl_xor_sync(0xffffffffu, v, o);
    v = is_max ? fmax(v, w) : v + w;
  }
  __syncthreads();
  if (lane == 0) buf[warp] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < kWarps; ++i) v = is_max ? fmax(v, buf[i]) : v + buf[i];
  return v;
}

// The teacher's part of a row is in 64 bits (some K numbers beside V): 1 - sum q cancels, and a loss near 0 is a difference.
template <typename T, bool TAIL>
__global__ void __launch_bounds__(kNT, 2) distill_kernel(DistillArgs a) {
  extern __shared__ __align__(16) uint8_t dynamic[];         // the feed's ring; TAIL: a bit for each element of this CTA's vectors
  __shared__ Shared sh;
  __shared__ int ids[kMaxK];
  __shared__ double red[kWarps];
  uint32_t* given = reinterpret_cast<uint32_t*>(dynamic + kRing);
  const int parts = a.parts, rank = parts == 1 ? 0 : (int)(blockIdx.x % parts), tid = threadIdx.x, K = a.K;
  const int64_t step = gridDim.x / parts;
  const float c = a.inv_t * kLog2e;
  constexpr int VEC = Slice<T>::VEC;
  Feed<T> feed(a.rows, reinterpret_cast<uint4*>(dynamic), blockIdx.x / parts, step, a.n, rank, parts);
  for (int64_t row = blockIdx.x / parts; row < a.n; row += step) {
    const T* x = row_at<T>(a.rows, row);
    const Slice<T> sl(x, a.rows.V, rank, parts);
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
    Best unused;
    scan<T, false, false, TAIL>(x, sl, c, feed, given, ids, K, sh, unused);
    const Stat st = row_stat<false>(sh, parts, c);
    if (rank == 0) {
      const bool none = st.m == -INFINITY && st.s == 0.f;
      const float m = none ? 0.f : st.m, ln_s = none ? 0.f : log2f(st.s) * kLn2;
      const double temp = a.temp;
      double z = TAIL ? a.lse[row] : -INFINITY, share = 1.0;   // q_k = e^(t_k / T - z) * share
      if constexpr (!TAIL) {
        for (int k = tid; k < K; k += kNT)
          if (ids[k] >= 0) z = fmax(z, a.values[row * K + k] / temp);
        z = (float)block_reduce(z, true, red);
      }
      double sum = 0.0;
      bool some = false;
      for (int k = tid; k < K; k += kNT)
        if (ids[k] >= 0) {
          const float t = a.values[row * K + k];
          some |= t != -INFINITY;
          if (TAIL || z != -INFINITY) sum += exp(t / temp - z);
        }
      sum = block_reduce(sum, false, red);
      const bool empty = !__syncthreads_or(some);              // no token given
      const double log_share = TAIL || empty ? 0.0 : -log(sum);
      if (!TAIL && !empty) share = 1.0 / sum;
      double part = 0.0;
      if (!empty)
        for (int k = tid; k < K; k += kNT) {
          if (ids[k] < 0) continue;
          const double d = a.values[row * K + k] / temp - z, q = exp(d) * share;
          const float lp = (DT<T>::to_f(x[ids[k]]) - m) / a.temp - ln_s;
          if (q != 0.0) part += q * (d + log_share - lp);
        }
      part = block_reduce(part, false, red);
      if (tid == 0) {
        double mass = sum * share, rest = 0.0;
        float ratio = 0.f;
        if constexpr (TAIL) {
          rest = fmax(1.0 - mass, 0.0);
          const float left = none ? 0.f : st.t / st.s;
          if (rest > 0.0 && left > 0.f) {
            ratio = (float)rest / left;
            part += rest * (log(rest) - (double)(log2f(left) * kLn2));
          } else {
            rest = 0.0;                                        // the student has no other token: the term is left out
          }
        }
        if (empty) {
          part = mass = rest = 0.0;
          ratio = 0.f;
        }
        if (bad) {
          tc5::report(a.err, kErrToken);
          part = mass = NAN;
        }
        a.loss[row] = (float)(part * temp * temp);
        if (a.stats != nullptr) {
          float4* s4 = reinterpret_cast<float4*>(a.stats) + 2 * row;
          s4[0] = make_float4(m, none ? 0.f : 1.f / st.s, (float)(mass + rest), ratio);
          s4[1] = make_float4((float)z, (float)share, 0.f, 0.f);
        }
      }
    }
    if (parts > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
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
  const float z = a.stats[8 * row + 4], share = a.stats[8 * row + 5];
  const float g = a.g[row] * a.temp, c = a.inv_t * kLog2e;
  if (g == 0.f || st.z == 0.f || st.y == 0.f) {
    map_row<T>(x, y, sl, [](float) { return 0.f; });
    return;
  }
  for (int k = threadIdx.x; k < K; k += kNT) {
    const int64_t id = a.ids[row * K + k];
    const bool ok = id >= 0 && id < a.rows.V;
    ids[k] = ok ? (int)id : -1;
    q[k] = ok ? ex2((float)(a.values[row * K + k] / (double)a.temp - z) * kLog2e) * share : 0.f;
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

// CTAs that stay, two to an SM, or a cluster for each row.
template <typename Args>
int launch_rows(void (*kern)(Args), const Args& a, size_t smem, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return (int)e;
  cfg.gridDim = dim3((unsigned)(a.parts > 1 || a.n < 2 * sms ? a.n * a.parts : 2 * sms));
  cfg.blockDim = dim3(kNT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.parts > 1 ? 1 : 0;
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
  ProbArgs a = {{logits, s0, s1, n1, V}, targets, logprob, entropy, stats, top_logprob, top_id, top, 0, ignore, rows, temp, 1.f / temp, err};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto kern = entropy != nullptr ? (top ? token_logprobs_kernel<T, true, true> : token_logprobs_kernel<T, true, false>)
                                   : (top ? token_logprobs_kernel<T, false, true> : token_logprobs_kernel<T, false, false>);
    static SmemLimit limit[4];
    const cudaError_t e = limit[(entropy != nullptr) * 2 + (top > 0)]((const void*)kern, kRing);
    return e != cudaSuccess ? (int)e : launch_rows<ProbArgs>(kern, a, kRing, (cudaStream_t)stream);
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
    kern<<<(unsigned)(rows * a.parts), kNT, 0, (cudaStream_t)stream>>>(a);
    return (int)cudaGetLastError();
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
  DistillArgs a = {{logits, s0, s1, n1, V}, ids, values, lse, loss, stats, rows, K, 0, temp, 1.f / temp, err};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    static SmemLimit limit[2];
    const size_t bits = lse != nullptr ? ((size_t)V / a.parts + 64) / 32 * 4 + 16 : 0;
    auto kern = lse != nullptr ? distill_kernel<T, true> : distill_kernel<T, false>;
    const cudaError_t e = limit[lse != nullptr]((const void*)kern, kRing + (lse != nullptr ? (1 << 20) / 8 + 64 : 0));
    return e != cudaSuccess ? (int)e : launch_rows<DistillArgs>(kern, a, kRing + bits, (cudaStream_t)stream);
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
    distill_grad_kernel<T><<<(unsigned)(rows * a.parts), kNT, 0, (cudaStream_t)stream>>>(a);
    return (int)cudaGetLastError();
  });
}
