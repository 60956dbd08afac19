// What stands behind an output layer: log probabilities of given tokens with their entropy and the best alternatives, and
// the divergence from a teacher's top logits, each with the gradient of the logits.  sm_100a.
//
// With c = log2(e) / T, r = rint(c max x), y = c x - r, s = sum 2^y, t = sum 2^y y (all to base 2):
//
//   log p_j = (y_j - log2 s) ln 2             H = (log2 s - t / s) ln 2
//   d log p_t / dx_j = (1[j = t] - p_j) / T   dH / dx_j = -p_j (log p_j + H) / T
//
// All of them are bound by memory: forward reads a row once, backward reads it once more and writes it once.  A row belongs
// to one CTA (many rows; the CTAs stay and take the next row) or to a cluster of up to eight (few rows).  Each thread copies its
// own four 16-byte vectors at a time to shared memory, asynchronously and two batches ahead, into the next row while a row's
// parts are joined.  Seven warps of a CTA read; an eighth does what a row has beside its sums (its target, the teacher's tokens,
// the results), on this row while the others read it and on its sums while they read the next one: in their way, those latencies
// took half of the time.  Four such CTAs to an SM: what is left of a row's latencies (the joining of its sums) hides behind the
// other CTAs' rows.  2048 rows of 32000 in bf16 took 47 us with two CTAs of sixteen warps and 38 so (the divergence 52 and 37); maxima
// by pairs of 16-bit numbers, as they are, whole batches without a test for each vector and a warp's sums joined at one base made it
// 30 us (4.4 TB/s; the divergence 32).  Nothing is at its limit then: while CTAs run, 62 % of the issue slots and 60 % of what the
// special function units do are taken, and 2048 rows are 3.46 rounds of 592 CTAs that take 4.  Backward is a plain pass of 224
// threads to a row, four vectors in flight (43 us for these rows, 6.1 TB/s).
// A thread folds the maximum of a batch into its own and rescales its sums once for all of it, so that an element costs one
// exponential (0.73 of what the special function units do at the rate of memory, for 16-bit logits).
// y is one fma: what rounding takes from r, common to a row, takes part everywhere alike and so cancels, as long as r is the same
// number everywhere (the maximum goes to the backward pass, and rescaling goes by differences of r).  r is whole, so sums are
// rescaled by powers of two, exactly: ex2.approx of other numbers is low by 5e-8 on average (measured), which a tree of partial
// sums adds up.  From |c max x| = 2^24 on (masks of -1e10, temperatures of 1e-6) r is no longer within a half of it, and what the
// fma leaves may be of any size: there y = (x - max x) c.
//
// Statistics are 32-bit: V / (224 x CTAs of a row) elements to a thread's sum (143 of 32000, 573 of 128256 with one CTA to a row)
// and a tree above that; exponentials by ex2.approx (2 ulp).
#include <cooperative_groups.h>

#include <type_traits>

#include "common/logit_rows.cuh"
#include "common/utils.cuh"
#include "tcgen05_common.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 7;         // that read rows
constexpr int kCtas = 4;          // to an SM
constexpr int kNT = 32 * kWarps;
constexpr int kU = 4;             // 16-byte requests of a thread in flight
constexpr int kMaxTop = 32;
constexpr int kMaxK = 1024;
constexpr int kCand = 1024;       // candidates for the best tokens of a slice before it is scanned in rounds instead
constexpr int kMaxCluster = 8;
constexpr int kMaxTailV = 1 << 19;
constexpr int kMaxBits = 2 * (kMaxTailV / 8 + 64);     // bytes: bits of two rows
constexpr float kNothing = 0x1p-100f;  // what the student gives to no other token: rest / left stays finite, and times a gradient

__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_end_batch() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {      // until all but the newest N batches have come
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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
    nvec = (unsigned)(V - head) / VEC;
    tail = V - head - nvec * VEC;
    const int by = __ffs(parts) - 1;                 // parts is a power of two
    v0 = (int)((int64_t)nvec * rank >> by);
    v1 = (int)((int64_t)nvec * (rank + 1) >> by);
    h = rank == 0 ? head : 0;
    t = rank == parts - 1 ? tail : 0;
  }
  __device__ bool has(int j) const {
    return (j >= head + v0 * VEC && j < head + v1 * VEC) || j < h || (j >= V - t && j < V);
  }
};

// The largest element of `n` (1 to kU) vectors that lie kNT apart.  16-bit numbers by pairs, as they are.
template <typename T, bool WHOLE>
__device__ __forceinline__ float largest_of(const uint4* w, int n) {
  if constexpr (std::is_same<T, float>::value) {
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (!WHOLE && u >= n) break;
      float f[4];
      unpack<T>(w[u * kNT], f);
      mx = max3(max3(mx, f[0], f[1]), f[2], f[3]);
    }
    return mx;
  } else {
    const uint4 v = w[0];
    uint32_t a = max2<T>(v.x, v.y), b = max2<T>(v.z, v.w);
#pragma unroll
    for (int u = 1; u < kU; ++u) {
      if (!WHOLE && u >= n) break;
      const uint4 x = w[u * kNT];
      a = max2<T>(a, max2<T>(x.x, x.y));
      b = max2<T>(b, max2<T>(x.z, x.w));
    }
    a = max2<T>(a, b);
    const T* e = reinterpret_cast<const T*>(&a);
    return max3(-INFINITY, DT<T>::to_f(e[0]), DT<T>::to_f(e[1]));
  }
}

// Larger keys come first: by value (NaN above all), then by the lower index.  No element has key 0.
__device__ __forceinline__ uint64_t order_key(float v, int idx) {
  const uint32_t b = v != v ? 0x7FFFFFFFu : __float_as_uint(v == 0.f ? 0.f : v);   // -0 and 0 are equal
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)o << 32 | (0xFFFFFFFFu - (uint32_t)idx);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

// The statistics of the first LANES lanes joined, in the first lane: all taken to the largest base, then added up.
template <bool ENT, int LANES>
__device__ __forceinline__ Stat join_lanes(const Stat& a, const Base& base, float c) {
  Stat o;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(o.m) : "f"(a.m));
  const float d = shift(base, Base(o.m, c), c), f = ex2(d);          // sums of a lane without tokens are 0
  o.s = a.s * f;
  o.t = ENT ? (a.t + a.s * d) * f : a.t * f;
#pragma unroll
  for (int n = LANES / 2; n > 0; n /= 2) {
    o.s += __shfl_xor_sync(0xffffffffu, o.s, n);
    o.t += __shfl_xor_sync(0xffffffffu, o.t, n);
  }
  return o;
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
  // This thread's vectors of the oldest batch, kNT apart; fetch() overwrites them.
  __device__ const uint4* oldest() {
    copies_wait<kStages - 1>();
    return ring + slot * kU * kNT;
  }
};

struct Sums {
  Stat warp[2][kWarps];           // by the parity of the CTA's row
  Stat part;                      // this CTA's
};
struct Shared : Sums {
  uint64_t best[kNT];             // the threads' best keys, sorted in each warp
  uint64_t cand[kCand];
  uint64_t top[2][kMaxTop];       // this CTA's best, sorted
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

// A barrier of the warps that read, and one that counts.
__device__ __forceinline__ void sync_readers() { asm volatile("bar.sync 1, %0;" ::"n"(kNT) : "memory"); }
__device__ __forceinline__ int sync_readers_count(bool x) {
  int n;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.u32 p, %1, 0;\n"
      "barrier.cta.red.popc.aligned.u32 %0, 1, %2, p;\n"
      "}\n"
      : "=r"(n)
      : "r"((uint32_t)x), "n"(kNT)
      : "memory");
  return n;
}

// Each warp's statistics of a row into `sums`, TOP: this thread's best.
template <typename T, bool ENT, bool TOP, bool TAIL>
__device__ void scan(const T* x, const Slice<T>& sl, float c, Feed<T>& feed, const uint32_t* given, const int* ids, int K,
                     Stat* sums, Best& best) {
  constexpr int VEC = Slice<T>::VEC;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Stat st = {-INFINITY, 0.f, 0.f};
  best = {0.f, -1};
  auto single = [&](int j) {
    const float v = DT<T>::to_f(x[j]);
    bool is_given = false;
    if constexpr (TAIL)
      for (int k = 0; k < K; ++k) is_given |= ids[k] == j;
    Stat one = {v, 1.f, 0.f};
    const float y = held(Base(v, c).exponent(v, c));
    one.s = ex2(y);
    if (ENT) one.t = one.s * y;
    else if (TAIL && !is_given) one.t = one.s;
    if (v != v) one = {-INFINITY, v, v};
    st = join<ENT>(st, one, c);
    if (TOP && (best.at == -1 || order_key(v, 0) > order_key(best.v, 0))) best = {v, -2 - j};
  };
  if (tid < sl.h) single(tid);
  // as the feed does: at least one batch a row, whether it holds vectors or not
  Base base(st.m, c);
  for (int at = sl.v0; at == sl.v0 || at < sl.v1; at += kNT * kU) {
    const uint4* w = feed.oldest();
    if (at + tid >= sl.v1) {
      feed.fetch();
      continue;
    }
    const int n = min(kU, (sl.v1 - at - tid + kNT - 1) / kNT);    // vectors of this thread
    float mx = n == kU ? largest_of<T, true>(w, n) : largest_of<T, false>(w, n);
    const Base now(fmaxf(st.m, mx), c);
    const float down = shift(base, now, c), fac = ex2(down);
    // CAREFUL: with exponents held, for what hides tokens, and of any size
    auto sums = [&](auto careful, auto whole, float& s, float& t) {
      constexpr bool CAREFUL = decltype(careful)::value, WHOLE = decltype(whole)::value;
      float sa[2] = {0.f, 0.f}, ta[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (!WHOLE && u >= n) break;
        float f[VEC], e[VEC], v[2] = {0.f, 0.f};
        unpack<T>(w[u * kNT], f);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          if (CAREFUL) {
            f[i] = held(now.exponent(f[i], c));
            f[i + 1] = held(now.exponent(f[i + 1], c));
          } else {
            exponents2(f[i], f[i + 1], c, -now.to);
          }
          e[i] = ex2(f[i]);
          e[i + 1] = ex2(f[i + 1]);
          add2(v[0], v[1], e[i], e[i + 1]);
          if constexpr (ENT) fma2(ta[0], ta[1], e[i], e[i + 1], f[i], f[i + 1]);
        }
        add2(sa[0], sa[1], v[0], v[1]);
        if constexpr (TAIL) {
          const int pos = (at + u * kNT + tid - sl.v0) * VEC;
          const uint32_t bits = given[pos >> 5] >> (pos & 31) & ((1u << VEC) - 1);
          if (bits == 0) {
            add2(ta[0], ta[1], v[0], v[1]);
          } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) ta[i & 1] += bits >> i & 1 ? 0.f : e[i];
          }
        }
      }
      s = sa[0] + sa[1];
      t = ta[0] + ta[1];
    };
    float s = 0.f, t = 0.f;
    if (now.far) sums(std::true_type(), std::false_type(), s, t);
    else if (n == kU) sums(std::false_type(), std::true_type(), s, t);
    else sums(std::false_type(), std::false_type(), s, t);
    if (ENT && !now.far && t != t) sums(std::true_type(), std::false_type(), s, t);
    if constexpr (ENT) st.t = (st.t + st.s * down) * fac + t;
    else if constexpr (TAIL) st.t = st.t * fac + t;
    st.s = st.s * fac + s;
    st.m = now.m;
    base = now;
    if constexpr (TOP) {
      if (s != s) {
        for (int u = 0; u < n; ++u) {
          float f[VEC];
          unpack<T>(w[u * kNT], f);
#pragma unroll
          for (int i = 0; i < VEC; ++i) mx = f[i] != f[i] ? NAN : mx;
        }
      }
      if (best.at == -1 || mx > best.v || (mx != mx && best.v == best.v)) best = {mx, at + tid};   // as order_key has it
    }
    feed.fetch();
  }
  if (tid >= kNT - sl.t) single(sl.V - (kNT - tid));
  st = join_lanes<ENT, 32>(st, Base(st.m, c), c);
  if (lane == 0) sums[warp] = st;
}

// The warps' statistics joined, in every lane of a warp.
template <bool ENT>
__device__ __forceinline__ Stat join_warps(const Stat* sums, float c) {
  const int lane = threadIdx.x & 31;
  Stat st = {-INFINITY, 0.f, 0.f};
  if (lane < kWarps) st = sums[lane];
  static_assert(kWarps <= 8, "join_lanes");
  st = join_lanes<ENT, 8>(st, Base(st.m, c), c);
  return {__shfl_sync(0xffffffffu, st.m, 0), __shfl_sync(0xffffffffu, st.s, 0), __shfl_sync(0xffffffffu, st.t, 0)};
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
  sync_readers();
  sh.best[threadIdx.x] = k;
#pragma unroll
  for (int n = 4; n > 0; n /= 2) {
    sync_readers();
    if (warp < n && warp + n < kWarps) {
      k = warp_merge(k, sh.best[(warp + n) * 32 + 31 - lane], lane);
      sh.best[threadIdx.x] = k;
    }
  }
  return k;
}

// The `top` largest keys of a slice, sorted, into `out` (0 behind the last element).  The top-th largest of the threads' best keys
// bounds them from below, and only the threads that reach it (top of them, keys being unique) can hold any: their elements are read
// again, sixteen lanes to each, and what reaches the bound is ranked by counting.  Values nearly always decide; where several
// threads have the bound's, these look up where they have it (the lower index comes first).  Where more than kCand elements
// reach it (a few threads hold nearly all large values), the slice is scanned once for each rank instead.
template <typename T>
__device__ void best_tokens(const T* x, const Slice<T>& sl, int top, const Best& best, uint64_t* out, Shared& sh) {
  constexpr int VEC = Slice<T>::VEC;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kMaxTop) out[tid] = 0;
  if (tid == 0) sh.n_cand = sh.n_list = 0;
  uint64_t mine = best.at == -1 ? 0 : order_key(best.v, tid);
  uint64_t k = largest32(mine, sh);
  if (tid == top - 1) sh.thr = k >> 32 << 32;       // the value alone: below every key that has it
  sync_readers();
  uint64_t thr = sh.thr;
  if (sync_readers_count(mine != 0 && mine >= thr) > top) {
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
    sync_readers();
    thr = sh.thr;
  }
  if (mine != 0 && mine >= thr) sh.list[atomicAdd(&sh.n_list, 1)] = tid;
  sync_readers();
  const int n_list = sh.n_list;
  for (int i = tid >> 4; i < n_list; i += kNT / 16)
    elements_of<T>(x, sl, sh.list[i], tid & 15, 16, [&](float v, int j) {
      const uint64_t key = order_key(v, j);
      if (key >= thr) {
        const int at = atomicAdd(&sh.n_cand, 1);
        if (at < kCand) sh.cand[at] = key;
      }
    });
  sync_readers();
  const int n = sh.n_cand;
  if (n <= kCand) {
    for (int i = tid; i < n; i += kNT) {
      const uint64_t key = sh.cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += sh.cand[j] > key;
      if (r < top) out[r] = key;
    }
    sync_readers();
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
    sync_readers();
    b = sh.best[0];
    for (int i = 1; i < kWarps; ++i) b = sh.best[i] > b ? sh.best[i] : b;
    if (tid == 0) out[r] = b;
    under = b;
    sync_readers();
    if (b == 0) break;
  }
}

// A row's statistics, in every lane of the finishing warp: those of its CTA's warps, and where a cluster has the row those of its
// CTAs (between two barriers of the cluster, which the other warps take part in: see meet()).
template <bool ENT>
__device__ __forceinline__ Stat row_stat(Sums& sh, int turn, int parts, float c) {
  Stat a = join_warps<ENT>(sh.warp[turn], c);
  if (parts > 1) {
    if ((threadIdx.x & 31) == 0) sh.part = a;
    __syncwarp();
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    a = *cl.map_shared_rank(&sh.part, 0);
    for (int i = 1; i < parts; ++i) a = join<ENT>(a, *cl.map_shared_rank(&sh.part, i), c);
  }
  return a;
}
// The other warps' share of a row's end in a cluster: sums are there, and shared memory stays until the first CTA has read it.
__device__ __forceinline__ void meet(int parts) {
  if (parts > 1) {
    cg::this_cluster().sync();
    cg::this_cluster().sync();
  }
}

struct ProbArgs {
  Rows rows;
  const int64_t* targets;
  float* logprob;
  float* entropy;      // null: not asked for
  float* stats;        // [rows, 4]: m, 1 / s, log2 s, H
  float* top_logprob;  // [rows, top]
  int64_t* top_id;
  int top, parts;
  int64_t ignore, n;   // n rows
  float temp, inv_t;
  int* err;
};

template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kNT + 32, kCtas) token_logprobs_kernel(ProbArgs a) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Shared sh;
  const int parts = a.parts, rank = parts == 1 ? 0 : (int)(blockIdx.x % parts);
  const int64_t first = blockIdx.x / parts, step = gridDim.x / parts;
  const float c = a.inv_t * kLog2e;
  if (threadIdx.x < kNT) {
    Feed<T> feed(a.rows, reinterpret_cast<uint4*>(dynamic), first, step, a.n, rank, parts);
    int turn = 0;
    for (int64_t row = first; row < a.n; row += step, turn ^= 1) {
      const T* x = row_at<T>(a.rows, row);
      const Slice<T> sl(x, a.rows.V, rank, parts);
      Best best;
      scan<T, ENT, TOP, false>(x, sl, c, feed, nullptr, nullptr, 0, sh.warp[turn], best);
      if constexpr (TOP) best_tokens<T>(x, sl, a.top, best, sh.top[turn], sh);
      __syncthreads();
      meet(parts);
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  int turn = 0;
  for (int64_t row = first; row < a.n; row += step, turn ^= 1) {
    const T* x = row_at<T>(a.rows, row);
    const int64_t t = a.targets[row];
    const bool ignored = t == a.ignore, bad = !ignored && (t < 0 || t >= a.rows.V);
    const float xt = ignored || bad ? 0.f : DT<T>::to_f(x[t]);
    __syncthreads();
    const Stat st = row_stat<ENT>(sh, turn, parts, c);
    if (rank == 0) {
      const bool none = no_token(st);
      const Base base(none ? 0.f : st.m, c);
      const double log2_s = none ? 0.0 : log2((double)st.s), lse = log_sum(base, log2_s, c, a.temp);
      const float H = !ENT || none ? 0.f : (float)((log2_s - (double)st.t / st.s) * kLn2_64);
      auto logp = [&](float v) {
        if (none) return -INFINITY;
        if (base.far) return (float)(((double)v - base.m) / a.temp - lse);
        return fabsf(v) < INFINITY ? (float)(v / (double)a.temp - lse) : v - (float)log2_s;
      };
      if (lane == 0) {
        if (bad) tc5::report(a.err, kErrToken);
        a.logprob[row] = bad ? NAN : ignored ? 0.f : logp(xt);
        if (ENT) a.entropy[row] = ignored ? 0.f : bad ? NAN : H;
        if (a.stats != nullptr) reinterpret_cast<float4*>(a.stats)[row] = make_float4(base.m, none ? 0.f : 1.f / st.s, (float)log2_s, H);
      }
      if constexpr (TOP) {
        uint64_t k = sh.top[turn][lane];
        for (int i = 1; i < parts; ++i)
          k = warp_merge(k, cg::this_cluster().map_shared_rank(&sh, i)->top[turn][31 - lane], lane);
        if (lane < a.top && k != 0) {
          const int id = key_index(k);
          a.top_id[row * a.top + lane] = id;
          a.top_logprob[row * a.top + lane] = logp(DT<T>::to_f(x[id]));
        }
      }
    }
    if (parts > 1) cg::this_cluster().sync();
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
  for (int base = sl.v0 + tid; base < sl.v1; base += kNT * kU) {
    uint4 w[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (base + u * kNT < sl.v1) w[u] = ldg_nc_v4(xv + base + u * kNT);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
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
  const int64_t row = blockIdx.x >> __ffs(a.parts) - 1;
  const T* x = row_at<T>(a.rows, row);
  T* y = reinterpret_cast<T*>(a.dx) + row * a.rows.V;
  const Slice<T> sl(x, a.rows.V, (int)(blockIdx.x & a.parts - 1), a.parts);
  const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
  const int64_t t = a.targets[row];
  const bool ignored = t == a.ignore, bad = !ignored && (t < 0 || t >= a.rows.V);
  float g = ignored || a.g == nullptr ? 0.f : a.g[row], ge = ignored || !ENT ? 0.f : a.g_ent[row];
  if (bad) g = NAN;
  if (st.y == 0.f) g = ge = 0.f;                    // no token in the row
  const float c = a.inv_t * kLog2e, scale = -st.y * a.inv_t, lp0 = st.w - st.z * kLn2;
  if (g == 0.f && ge == 0.f) {                      // nothing flows into this row, whatever its logits hold
    map_row<T>(x, y, sl, [](float) { return 0.f; });
    return;
  }
  const Base base(st.x, c);
  auto of = [&](float y) {
    const float d = ENT ? held(y) : y, e = ex2(d) * scale;
    return ENT ? e * fmaf(ge, fmaf(d, kLn2, lp0), g) : e * g;
  };
  if (base.far) map_row<T>(x, y, sl, [&](float v) { return of((v - base.m) * c); });
  else map_row<T>(x, y, sl, [&](float v) { return of(fmaf(v, c, -base.r)); });
  __syncthreads();
  if (threadIdx.x == 0 && !bad && t >= 0 && t < a.rows.V && !ignored && sl.has((int)t))
    y[t] = DT<T>::from_f(fmaf(g, a.inv_t, of(base.exponent(DT<T>::to_f(x[t]), c))));
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
  int words;               // of a row's bits, a multiple of 4
  float temp, inv_t;
  int* err;
};

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The teacher's part of a row, by the finishing warp, in 64 bits (some K numbers beside V): 1 - sum q cancels, and a loss near 0 is
// a difference.  sum_k q_k (log q_k - log p_id) = own - cross / T + mass log sum e^(x / T) with what follows, so that it need not
// wait for the student's sums.
struct Teacher {
  double own, cross, mass;   // sum q log q, sum q (x_id - from), sum q
  float z, share;            // q_k = e^(t_k / T - z) * share
  bool empty, never;         // no token is given; a given one can never be the student's (its logit is -inf)
};
template <typename T, bool TAIL>
__device__ Teacher teacher_of(const T* x, const int* ids, const float* values, const float* lse, int K, float temp_, double from) {
  const int lane = threadIdx.x & 31;
  const double temp = temp_;
  double z = TAIL ? *lse : -INFINITY;
  bool some = false, never = false;
  for (int k = lane; k < K; k += 32)
    if (ids[k] >= 0) {
      some |= values[k] != -INFINITY;
      if (!TAIL) z = fmax(z, values[k] / temp);
    }
  some = __any_sync(0xffffffffu, some);
  if (!TAIL) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z = fmax(z, __shfl_xor_sync(0xffffffffu, z, o));
    z = (float)z;
  }
  double own = 0.0, cross = 0.0, mass = 0.0;
  if (some)
    for (int k = lane; k < K; k += 32)
      if (ids[k] >= 0) {
        const double d = values[k] / temp - z, q = exp(d);
        const float v = DT<T>::to_f(x[ids[k]]);
        if (q != 0.0) {
          own += q * d;
          if (v == -INFINITY) never = true;
          else cross += q * (v - from);
        }
        mass += q;
      }
  own = warp_sum64(own);
  cross = warp_sum64(cross);
  mass = warp_sum64(mass);
  Teacher t = {own, cross, mass, (float)z, 1.f, !some, __any_sync(0xffffffffu, never) != 0};
  if (!TAIL && some) {                              // normalised
    t.share = (float)(1.0 / mass);
    t.own = own / mass - log(mass);
    t.cross = cross / mass;
    t.mass = mass == mass ? 1.0 : mass;
  }
  return t;
}

template <typename T, bool TAIL>
__global__ void __launch_bounds__(kNT + 32, kCtas) distill_kernel(DistillArgs a) {
  // the feed's ring; TAIL: for this row and the next one, a bit for each element of this CTA's vectors
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Sums sh;
  __shared__ int ids[2][kMaxK];
  uint32_t* given = reinterpret_cast<uint32_t*>(dynamic + kRing);
  const int parts = a.parts, rank = parts == 1 ? 0 : (int)(blockIdx.x % parts), K = a.K;
  const int64_t first = blockIdx.x / parts, step = gridDim.x / parts;
  const float c = a.inv_t * kLog2e;
  constexpr int VEC = Slice<T>::VEC;
  if (threadIdx.x < kNT) {
    Feed<T> feed(a.rows, reinterpret_cast<uint4*>(dynamic), first, step, a.n, rank, parts);
    __syncthreads();
    int turn = 0;
    for (int64_t row = first; row < a.n; row += step, turn ^= 1) {
      const T* x = row_at<T>(a.rows, row);
      const Slice<T> sl(x, a.rows.V, rank, parts);
      Best unused;
      scan<T, false, false, TAIL>(x, sl, c, feed, given + turn * a.words, ids[turn], K, sh.warp[turn], unused);
      __syncthreads();
      meet(parts);
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  // a row's tokens, and their bits; true where one lies outside of the vocabulary
  auto open = [&](int64_t row, int turn) {
    bool bad = false;
    for (int k = lane; k < K; k += 32) {
      const int64_t id = a.ids[row * K + k];
      bad |= id >= a.rows.V;
      ids[turn][k] = id < 0 || id >= a.rows.V ? -1 : (int)id;
    }
    if constexpr (TAIL) {
      const Slice<T> sl(row_at<T>(a.rows, row), a.rows.V, rank, parts);
      uint32_t* bits = given + turn * a.words;
      for (int i = lane; i < a.words / 4; i += 32) reinterpret_cast<uint4*>(bits)[i] = make_uint4(0, 0, 0, 0);
      __syncwarp();
      for (int k = lane; k < K; k += 32) {
        const int pos = ids[turn][k] - sl.head - sl.v0 * VEC;
        if (ids[turn][k] >= 0 && pos >= 0 && pos < (sl.v1 - sl.v0) * VEC) atomicOr(&bits[pos >> 5], 1u << (pos & 31));
      }
    }
    __syncwarp();
    return __any_sync(0xffffffffu, bad) != 0;
  };
  bool bad = open(first, 0);
  __syncthreads();
  int turn = 0;
  for (int64_t row = first; row < a.n; row += step, turn ^= 1) {
    const T* x = row_at<T>(a.rows, row);
    auto teacher = [&](float from) {
      return teacher_of<T, TAIL>(x, ids[turn], a.values + row * K, TAIL ? a.lse + row : nullptr, K, a.temp, from);
    };
    Teacher te = teacher(0.f);
    const bool bad_next = row + step < a.n && open(row + step, turn ^ 1);
    __syncthreads();
    const Stat st = row_stat<false>(sh, turn, parts, c);
    const bool none = no_token(st);
    const Base base(none ? 0.f : st.m, c);
    if (base.far) te = teacher(st.m);          // differences of numbers that far from 0 would cancel
    if (rank == 0 && lane == 0) {
      double mass = te.mass, rest = 0.0;
      double loss = te.never || (none && mass > 0.0) ? INFINITY
                             : te.own - te.cross / a.temp + te.mass * log_sum(base, none ? 0.0 : log2((double)st.s), c, a.temp);
      float ratio = 0.f;
      if constexpr (TAIL) {
        rest = fmax(1.0 - mass, 0.0);
        const float left = none ? 0.f : st.t / st.s;
        if (rest > 0.0 && left > kNothing) {
          ratio = (float)rest / left;
          loss += rest * log(rest * st.s / st.t);
        } else {
          rest = 0.0;                                        // as good as no other token: the term is left out
        }
      }
      if (te.empty) {
        loss = mass = rest = 0.0;
        ratio = 0.f;
      }
      if (bad) {
        tc5::report(a.err, kErrToken);
        loss = mass = NAN;
      }
      a.loss[row] = (float)(loss * a.temp * a.temp);
      if (a.stats != nullptr) {
        float4* s4 = reinterpret_cast<float4*>(a.stats) + 2 * row;
        s4[0] = make_float4(base.m, none ? 0.f : 1.f / st.s, (float)(mass + rest), ratio);
        s4[1] = make_float4(te.z, te.share, 0.f, 0.f);
      }
    }
    bad = bad_next;
    if (parts > 1) cg::this_cluster().sync();
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
  const int64_t row = blockIdx.x >> __ffs(a.parts) - 1;
  const int K = a.K;
  const T* x = row_at<T>(a.rows, row);
  T* y = reinterpret_cast<T*>(a.dx) + row * a.rows.V;
  const Slice<T> sl(x, a.rows.V, (int)(blockIdx.x & a.parts - 1), a.parts);
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
  const Base base(st.x, c);
  if (base.far) map_row<T>(x, y, sl, [&](float v) { return ex2((v - base.m) * c) * other; });
  else map_row<T>(x, y, sl, [&](float v) { return ex2(fmaf(v, c, -base.r)) * other; });
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
    if (first) y[id] = DT<T>::from_f(fmaf(-g, sum, ex2(base.exponent(DT<T>::to_f(x[id]), c)) * own));
  }
}

// ------------------------------------------------------------------------------------------------ host
// CTAs to a row: one where the rows alone fill the SMs, else as many (up to a portable cluster) as do, while each still has a
// batch of requests for its threads.
int parts_of(int64_t rows, int V, int elem) {
  const int64_t batch = (int64_t)kNT * 16 / elem;
  const int sms = sm_count();
  int parts = 1;
  while (parts < kMaxCluster && rows * parts < sms && (int64_t)V > batch * parts) parts *= 2;
  return parts;
}

// CTAs that stay, kCtas to an SM or what its 227 KB of shared memory hold (the bits of a long row's tail take some), or a cluster
// for each row.
template <typename Args>
int launch_rows(void (*kern)(Args), const Args& a, size_t smem, size_t fixed, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  const int sms = sm_count();
  if (sms == 0) return (int)cudaErrorInvalidDevice;
  const size_t fit = (227 << 10) / (smem + fixed + 1024);
  const int64_t stay = (int64_t)(fit < kCtas ? fit : kCtas) * sms;
  cfg.gridDim = dim3((unsigned)(a.parts > 1 || a.n < stay ? a.n * a.parts : stay));
  cfg.blockDim = dim3(kNT + 32);
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
  ProbArgs a = {rows_of(logits, s0, s1, n1, rows, V), targets, logprob, entropy, stats, top_logprob, top_id, top, 0, ignore,
                rows, temp, 1.f / temp, err};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto kern = entropy != nullptr ? (top ? token_logprobs_kernel<T, true, true> : token_logprobs_kernel<T, true, false>)
                                   : (top ? token_logprobs_kernel<T, false, true> : token_logprobs_kernel<T, false, false>);
    static SmemLimit limit[4];
    const cudaError_t e = limit[(entropy != nullptr) * 2 + (top > 0)]((const void*)kern, kRing);
    return e != cudaSuccess ? (int)e : launch_rows<ProbArgs>(kern, a, kRing, sizeof(Shared), (cudaStream_t)stream);
  });
}

// g / g_entropy [rows]: gradients of the log probability and of the entropy (either may be null); dlogits [rows, V].
IPEX_API int ipex_token_logprobs_grad(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* targets,
                                      const float* stats, const float* g, const float* g_entropy, void* dlogits, int64_t rows,
                                      int V, int64_t ignore, float temp, int dtype, void* stream) {
  if (!rows_ok(logits, s0, s1, n1, rows, V, dtype == DT_F32 ? 4 : 2) || !temp_ok(temp) ||
      targets == nullptr || dlogits == nullptr || stats == nullptr || (reinterpret_cast<uintptr_t>(stats) & 15))
    return (int)cudaErrorInvalidValue;
  ProbGradArgs a = {rows_of(logits, s0, s1, n1, rows, V), targets, stats, g, g_entropy, dlogits, ignore, 1.f / temp, 0};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto kern = g_entropy != nullptr ? token_logprobs_grad_kernel<T, true> : token_logprobs_grad_kernel<T, false>;
    kern<<<(unsigned)(rows * a.parts), kNT, 0, (cudaStream_t)stream>>>(a);
    return (int)cudaGetLastError();
  });
}

// ids / values [rows, K]: the teacher's tokens (below 0: none) and their logits, K up to 1024; lse [rows]: logsumexp of the
// teacher's logits / temp, or null; loss [rows]; stats [rows, 8] (16-byte aligned) or null.  V up to 524288 with lse.
IPEX_API int ipex_distill(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* ids, const float* values,
                          const float* lse, float* loss, float* stats, int64_t rows, int V, int K, float temp, int dtype, int* err,
                          void* stream) {
  if (!rows_ok(logits, s0, s1, n1, rows, V, dtype == DT_F32 ? 4 : 2) || K < 1 || K > kMaxK || !temp_ok(temp) ||
      ids == nullptr || values == nullptr || loss == nullptr || (lse != nullptr && V > kMaxTailV) ||
      (reinterpret_cast<uintptr_t>(stats) & 15))
    return (int)cudaErrorInvalidValue;
  DistillArgs a = {rows_of(logits, s0, s1, n1, rows, V), ids, values, lse, loss, stats, rows, K, 0, 0, temp, 1.f / temp, err};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    static SmemLimit limit[2];
    if (lse != nullptr) a.words = (V / a.parts + 64 + 127) / 128 * 4;
    auto kern = lse != nullptr ? distill_kernel<T, true> : distill_kernel<T, false>;
    const cudaError_t e = limit[lse != nullptr]((const void*)kern, kRing + (lse != nullptr ? kMaxBits : 0));
    return e != cudaSuccess ? (int)e
                            : launch_rows<DistillArgs>(kern, a, kRing + a.words * 8, sizeof(Sums) + 8 * kMaxK, (cudaStream_t)stream);
  });
}

IPEX_API int ipex_distill_grad(const void* logits, int64_t s0, int64_t s1, int64_t n1, const int64_t* ids, const float* values,
                               const float* stats, const float* g, void* dlogits, int64_t rows, int V, int K, float temp, int dtype,
                               void* stream) {
  if (!rows_ok(logits, s0, s1, n1, rows, V, dtype == DT_F32 ? 4 : 2) || K < 1 || K > kMaxK || !temp_ok(temp) ||
      ids == nullptr || values == nullptr || dlogits == nullptr || stats == nullptr || g == nullptr ||
      (reinterpret_cast<uintptr_t>(stats) & 15))
    return (int)cudaErrorInvalidValue;
  DistillGradArgs a = {rows_of(logits, s0, s1, n1, rows, V), ids, values, stats, g, dlogits, K, 0, temp, 1.f / temp};
  a.parts = parts_of(rows, V, dtype == DT_F32 ? 4 : 2);
  return by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    distill_grad_kernel<T><<<(unsigned)(rows * a.parts), kNT, 0, (cudaStream_t)stream>>>(a);
    return (int)cudaGetLastError();
  });
}
