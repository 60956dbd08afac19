// The update of many tensors at once: AdamW with moments in 32 or in 8 bits, and the norm of all gradients.  sm_100a.
//
//   m' = b1 m + (1 - b1) g       v' = b2 v + (1 - b2) g^2       g: times the clipping factor min(1, max_norm / (norm + 1e-6))
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// All of it is bound by memory: an element's numbers are read once and written once (26 bytes for bf16 with 32-bit moments and the
// 16 bits below bf16, 14 with 8-bit moments).  Tensors lie anywhere; what is kept of them (moments, exponents, the rest of the
// parameters) lies in flat buffers, each tensor's from a multiple of 256 on.  One launch takes up to kMost tensors: their addresses and
// sizes come with the launch, as its parameters, and CTAs take tiles of 2048 elements, each of one tensor.
//
// Every operation is one of IEEE's, rounded to nearest, in the order written above, none contracted: results do not depend on how
// the work is split, and 8-bit moments can be told bit by bit.
//
// Moments in 8 bits: 256 elements (a warp's) share an exponent e, that of the largest of them; m / 2^(e - 134) is held in e4m3, so
// that the largest lies in [2^7, 2^8), and v / 2^(e - 141) in e5m2 (the largest in [2^14, 2^15): v spans twice m's octaves).  A step
// moves v by a thousandth where neighbours are a quarter apart, so that rounding to nearest would hold it for good; it is rounded up
// with the probability of what is cut off (random bits of a hash of the element's place, the step and a seed), which keeps the mean.
// A v that is not 0 is never held as 0, lest m is divided by eps alone.  What is not finite stays so by itself and does not count
// for the exponent.
#include <cuda_fp8.h>

#include <type_traits>

#include "common/utils.cuh"

namespace {

constexpr int kNT = 256;
constexpr int kVec = 8;                     // elements of a thread
constexpr int kTile = kNT * kVec;
constexpr int kBlock = 256;                 // elements with a common exponent: a warp's
static_assert(kBlock == 32 * kVec, "a warp has a block");
constexpr int kLow = 32, kHigh = 254;       // exponents of a block: 2^(e - 127)
constexpr int kMost = 640;                  // tensors of a launch: 25 KB of its 32 KB of parameters

enum { REST_NONE = 0, REST_16 = 1, REST_32 = 2 };

struct Entry {
  void* p;
  const void* g;
  int64_t n;
  uint32_t tile;       // the first of its tiles
  uint32_t block;      // where its moments begin, in blocks
  int32_t step;        // which step counter is its own
};
template <int CAP>
struct Table {
  Entry e[CAP];
  int n;
  uint32_t tiles;
};

// What an update needs beside its numbers, for each step counter.
struct Factors {
  float rate, root, clip, decay;      // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), of the gradient, 1 - lr wd
};

__device__ double power(double b, int64_t t) {
  double r = 1.0;
  for (; t > 0; t >>= 1) {
    if (t & 1) r *= b;
    b *= b;
  }
  return r;
}

struct BeginArgs {
  int64_t* step;
  const float* norm;      // of all gradients, or null
  const float* lr_at;     // or null: lr
  Factors* out;
  double max_norm, lr, b1, b2, decay;
};

template <int CAP>
__global__ void adamw_begin(const __grid_constant__ Table<CAP> tab, BeginArgs a) {
  pdl_launch_dependents();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= tab.n) return;
  const int at = tab.e[i].step;
  if (i > 0 && tab.e[i - 1].step == at) return;     // one counter for all
  const int64_t t = a.step[at] + 1;
  a.step[at] = t;
  const double lr = a.lr_at != nullptr ? (double)*a.lr_at : a.lr;
  Factors f;
  f.rate = (float)(lr / (1.0 - power(a.b1, t)));
  f.root = (float)(1.0 / sqrt(1.0 - power(a.b2, t)));
  f.decay = (float)(1.0 - lr * a.decay);
  f.clip = 1.f;
  if (a.norm != nullptr) {
    const float c = __fdiv_rn((float)a.max_norm, __fadd_rn(*a.norm, 1e-6f));
    f.clip = c > 1.f ? 1.f : c;                     // NaN stays
  }
  a.out[at] = f;
}

template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& tab, uint32_t tile, int from) {
  int lo = from, hi = tab.n;                        // the last one whose first tile is not behind it
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.e[mid].tile <= tile) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Eight elements at a multiple of 16 bytes, as 32-bit numbers.
__device__ __forceinline__ void load8(const float* x, float* f) {
  const float4 a = reinterpret_cast<const float4*>(x)[0], b = reinterpret_cast<const float4*>(x)[1];
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* x, float* f) {
  const uint4 w = *reinterpret_cast<const uint4*>(x);
  const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = DT<T>::to_f(e[i]);
}
__device__ __forceinline__ void store8(float* x, const float* f) {
  reinterpret_cast<float4*>(x)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(x)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T* x, const float* f) {
  __align__(16) T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = DT<T>::from_f(f[i]);
  *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(e);
}

// 2^k for the exponents that occur here (-126 to 127).
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }
// A block's exponent as it is held: 0 in moments that no step has seen.
__device__ __forceinline__ int held(uint8_t e) { return min(max((int)e, kLow), kHigh); }

// The exponent of the largest finite number of a warp's, of 32 x 8.
__device__ __forceinline__ int block_exponent(const float* x) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    top = max(top, b < 0x7F800000u ? b : 0u);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  return held((uint8_t)(top >> 23));
}

__device__ __forceinline__ uint32_t mixed(uint32_t x) {
  x = (x ^ (x >> 16)) * 0xBB67AE85u;                // fractions of the roots of 3 and 2
  x = (x ^ (x >> 15)) * 0x6A09E667u;
  return x ^ (x >> 16);
}

// A 32-bit number's bits are its exponent and fraction in a row, whatever its size: scaled so that its exponent field is the small
// format's, adding random bits below the last kept place and cutting there rounds it up with the probability of what is cut off.
__device__ __forceinline__ uint32_t to_e4m3(float x, float up, uint32_t chance) {
  const float a = fabsf(x);
  const uint32_t bits = __float_as_uint(__fmul_rn(__fmul_rn(a, up), 0x1p-120f));
  const uint32_t code = (bits + (chance << 4) + 8) >> 20 | (x < 0.f ? 0x80u : 0u);
  return a < INFINITY ? code : 0x7Fu;               // the format has no infinity
}
__device__ __forceinline__ uint32_t to_e5m2(float x, float up, uint32_t chance) {
  const uint32_t bits = __float_as_uint(__fmul_rn(__fmul_rn(x, up), 0x1p-112f));
  const uint32_t code = (bits + (chance << 5) + 16) >> 21;
  if (!(x < INFINITY)) return x == INFINITY ? 0x7Cu : 0x7Fu;
  return x > 0.f ? max(code, 1u) : code;
}
template <__nv_fp8_interpretation_t KIND>
__device__ __forceinline__ void from_fp8(uint2 w, float down, float* f) {
  const uint32_t v[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v[i >> 1] >> (16 * (i & 1))), KIND);
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&h));
    f[2 * i] = __fmul_rn(p.x, down);
    f[2 * i + 1] = __fmul_rn(p.y, down);
  }
}

struct StepArgs {
  void* m;
  void* v;
  uint8_t* m_scale;    // exponents of blocks of 8-bit moments
  uint8_t* v_scale;
  void* rest;          // the 16 bits below bf16, or copies in 32 bits
  const Factors* factors;
  const int64_t* step;
  float b1, c1, b2, c2, eps;     // c: 1 - b
  uint32_t seed;
};

template <typename T, bool SMALL, int REST, int CAP>
__global__ void __launch_bounds__(kNT) adamw_step(const __grid_constant__ Table<CAP> tab, StepArgs a) {
  const int lane = threadIdx.x & 31;
  int i = 0;
  pdl_wait();
  for (uint32_t tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x) {
    i = tensor_of(tab, tile, i);
    const Entry& e = tab.e[i];
    const int64_t off = (int64_t)(tile - e.tile) * kTile + threadIdx.x * kVec;      // in the tensor
    const int64_t warp_off = off - lane * kVec;
    if (warp_off >= e.n) continue;                                                  // whole warps: no block of theirs
    const Factors f = a.factors[e.step];
    const int64_t at = (int64_t)e.block * kBlock + off;                             // in the flat buffers
    const int have = off >= e.n ? 0 : (int)min((int64_t)kVec, e.n - off);
    T* p_at = reinterpret_cast<T*>(e.p) + off;
    const T* g_at = reinterpret_cast<const T*>(e.g) + off;
    const bool vec = have == kVec && ((reinterpret_cast<uintptr_t>(e.p) | reinterpret_cast<uintptr_t>(e.g)) & 15) == 0;
    float p[kVec], g[kVec], m[kVec], v[kVec];
    if (vec) {
      load8(g_at, g);
      if constexpr (REST != REST_32) load8(p_at, p);
    } else {
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        g[k] = k < have ? DT<T>::to_f(g_at[k]) : 0.f;
        if constexpr (REST != REST_32) p[k] = k < have ? DT<T>::to_f(p_at[k]) : 0.f;
      }
    }
    if constexpr (REST == REST_32) load8(reinterpret_cast<const float*>(a.rest) + at, p);
    if constexpr (REST == REST_16) {
      const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const int16_t*>(a.rest) + at);
      const int16_t* r = reinterpret_cast<const int16_t*>(&w);
#pragma unroll
      for (int k = 0; k < kVec; ++k) p[k] = __uint_as_float(__float_as_uint(p[k]) + (uint32_t)(int)r[k]);
    }
    if constexpr (SMALL) {
      const int64_t blk = at / kBlock;
      from_fp8<__NV_E4M3>(*reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(a.m) + at), pow2(held(a.m_scale[blk]) - 134), m);
      from_fp8<__NV_E5M2>(*reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(a.v) + at), pow2(held(a.v_scale[blk]) - 141), v);
    } else {
      load8(reinterpret_cast<const float*>(a.m) + at, m);
      load8(reinterpret_cast<const float*>(a.v) + at, v);
    }
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const float x = __fmul_rn(g[k], f.clip);
      m[k] = __fadd_rn(__fmul_rn(m[k], a.b1), __fmul_rn(x, a.c1));
      v[k] = __fadd_rn(__fmul_rn(v[k], a.b2), __fmul_rn(__fmul_rn(x, x), a.c2));
      const float d = __fadd_rn(__fmul_rn(__fsqrt_rn(v[k]), f.root), a.eps);
      p[k] = __fsub_rn(__fmul_rn(p[k], f.decay), __fdiv_rn(__fmul_rn(m[k], f.rate), d));
      if (k >= have) m[k] = v[k] = p[k] = 0.f;      // behind the tensor's end: 0 / eps, or 0 / 0
    }
    if constexpr (SMALL) {
      const int em = block_exponent(m), ev = block_exponent(v);
      const float up_m = pow2(134 - em), up_v = pow2(141 - ev);
      const uint32_t t = (uint32_t)a.step[e.step];
      const uint32_t key = mixed(mixed(t) + a.seed * 0x9E3779B1u) + (uint32_t)(at >> 32) * 0xBB67AE85u;
      uint32_t wm[2] = {0, 0}, wv[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const uint32_t h = mixed((uint32_t)(at + k) * 0x9E3779B1u + key);
        wm[k >> 2] |= to_e4m3(m[k], up_m, h & 0xFFFFu) << (8 * (k & 3));
        wv[k >> 2] |= to_e5m2(v[k], up_v, h >> 16) << (8 * (k & 3));
      }
      *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.m) + at) = make_uint2(wm[0], wm[1]);
      *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.v) + at) = make_uint2(wv[0], wv[1]);
      if (lane == 0) {
        a.m_scale[at / kBlock] = (uint8_t)em;
        a.v_scale[at / kBlock] = (uint8_t)ev;
      }
    } else {
      store8(reinterpret_cast<float*>(a.m) + at, m);
      store8(reinterpret_cast<float*>(a.v) + at, v);
    }
    if constexpr (REST == REST_32) store8(reinterpret_cast<float*>(a.rest) + at, p);
    if constexpr (REST == REST_16) {
      // bf16 nearest to p (halves up) and the difference of their bits; p is made that bf16
      __align__(16) int16_t r[kVec];
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const uint32_t bits = __float_as_uint(p[k]);
        uint32_t high = (bits + 0x8000u) & 0xFFFF0000u;
        r[k] = (int16_t)(bits - high);
        if (p[k] != p[k]) {                         // its bits may run over
          high = 0x7FFF0000u;
          r[k] = 0;
        }
        p[k] = __uint_as_float(high);
      }
      *reinterpret_cast<uint4*>(reinterpret_cast<int16_t*>(a.rest) + at) = *reinterpret_cast<const uint4*>(r);
    }
    if (vec) {
      store8(p_at, p);
    } else {
#pragma unroll
      for (int k = 0; k < kVec; ++k)
        if (k < have) p_at[k] = DT<T>::from_f(p[k]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ the norm of all gradients
// Eight squares are added in 32 bits, their sums in 64: a thread's, then a CTA's, then those of all CTAs in their order.  Where a sum
// of eight is too large or too small for 32 bits, they are taken in 64.
template <typename T, int CAP>
__global__ void __launch_bounds__(kNT) grad_squares(const __grid_constant__ Table<CAP> tab, double* sums) {
  __shared__ double part[kNT / 32];
  pdl_launch_dependents();
  double total = 0.0;
  int i = 0;
  for (uint32_t tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x) {
    i = tensor_of(tab, tile, i);
    const Entry& e = tab.e[i];
    const int64_t off = (int64_t)(tile - e.tile) * kTile + threadIdx.x * kVec;
    if (off >= e.n) continue;
    const int have = (int)min((int64_t)kVec, e.n - off);
    const T* at = reinterpret_cast<const T*>(e.g) + off;
    float g[kVec];
    if (have == kVec && (reinterpret_cast<uintptr_t>(e.g) & 15) == 0) {
      load8(at, g);
    } else {
#pragma unroll
      for (int k = 0; k < kVec; ++k) g[k] = k < have ? DT<T>::to_f(at[k]) : 0.f;
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kVec; ++k) s = fmaf(g[k], g[k], s);
    if (s > 1e-25f && s < 1e38f) {
      total += (double)s;
    } else {
      for (int k = 0; k < kVec; ++k) total += (double)g[k] * g[k];
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kNT / 32; ++w) total += part[w];
    sums[blockIdx.x] = total;
  }
}

__global__ void __launch_bounds__(kNT) grad_norm_kernel(const double* sums, int n, float* norm) {
  __shared__ double part[kNT / 32];
  pdl_wait();
  double total = 0.0;
  for (int i = threadIdx.x; i < n; i += kNT) total += sums[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kNT / 32; ++w) total += part[w];
    *norm = (float)sqrt(total);
  }
}

// ------------------------------------------------------------------------------------------------ host
int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) != 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// The tensors [from, to) that have a gradient, at most CAP of them, as a table; `block`: where the moments of tensor `from` begin.
// Returns the tensor behind the last one, -1 for a size that is not allowed.
template <int CAP>
int64_t fill(Table<CAP>& tab, const int64_t* p, const int64_t* g, const int64_t* n, int64_t from, int64_t to, int steps, uint64_t& block) {
  tab.n = 0;
  tab.tiles = 0;
  int64_t i = from;
  for (; i < to && tab.n < CAP; ++i) {
    const uint64_t blocks = ((uint64_t)n[i] + kBlock - 1) / kBlock, tiles = ((uint64_t)n[i] + kTile - 1) / kTile;
    if (n[i] < 0 || block + blocks > 0xFFFFFFFFull) return -1;
    if (g[i] != 0 && n[i] > 0) {
      if (tiles + tab.tiles > 0x7FFFFFFFull) {
        if (tab.n == 0) return -1;
        return i;
      }
      tab.e[tab.n++] = {p == nullptr ? nullptr : reinterpret_cast<void*>(p[i]), reinterpret_cast<const void*>(g[i]), n[i], tab.tiles,
                        (uint32_t)block, steps > 1 ? (int)i : 0};
      tab.tiles += (uint32_t)tiles;
    }
    block += blocks;
  }
  return i;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == DT_F16) return f((__half*)nullptr);
  if (dtype == DT_BF16) return f((__nv_bfloat16*)nullptr);
  if (dtype == DT_F32) return f((float*)nullptr);
  return (int)cudaErrorInvalidValue;
}

constexpr int kCtas = 4;      // to an SM

int grid_of(uint32_t tiles, int sms) { return (int)(tiles < (uint32_t)(sms * kCtas) ? tiles : (uint32_t)(sms * kCtas)); }

template <int CAP>
int step_all(const int64_t* p, const int64_t* g, const int64_t* n, int64_t count, const BeginArgs& b, const StepArgs& a, int steps,
             int dtype, bool small, int rest, cudaStream_t s) {
  const int sms = sm_count();
  if (sms == 0) return (int)cudaErrorInvalidDevice;
  Table<CAP> tab;
  uint64_t block = 0;
  bool begun = false;
  for (int64_t at = 0; at < count;) {
    at = fill(tab, p, g, n, at, count, steps, block);
    if (at < 0) return (int)cudaErrorInvalidValue;
    if (tab.n == 0) continue;
    if (!begun || steps > 1) {                      // a common counter moves once
      adamw_begin<CAP><<<(tab.n + 127) / 128, 128, 0, s>>>(tab, b);
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return (int)e;
      begun = true;
    }
    const int rc = by_type(dtype, [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      void (*kern)(Table<CAP>, StepArgs) = nullptr;
      if (rest == REST_NONE) kern = small ? adamw_step<T, true, REST_NONE, CAP> : adamw_step<T, false, REST_NONE, CAP>;
      if constexpr (!std::is_same<T, float>::value)
        if (rest == REST_32) kern = small ? adamw_step<T, true, REST_32, CAP> : adamw_step<T, false, REST_32, CAP>;
      if constexpr (std::is_same<T, __nv_bfloat16>::value)
        if (rest == REST_16) kern = small ? adamw_step<T, true, REST_16, CAP> : adamw_step<T, false, REST_16, CAP>;
      if (kern == nullptr) return (int)cudaErrorInvalidValue;
      return (int)launch_kernel(kern, dim3(grid_of(tab.tiles, sms)), dim3(kNT), 0, s, true, tab, a);
    });
    if (rc != 0) return rc;
  }
  return 0;
}

template <int CAP>
int norm_all(const int64_t* g, const int64_t* n, int64_t count, double* sums, float* norm, int dtype, cudaStream_t s) {
  const int sms = sm_count();
  if (sms == 0) return (int)cudaErrorInvalidDevice;
  Table<CAP> tab;
  uint64_t block = 0;
  int parts = 0;
  for (int64_t at = 0; at < count;) {
    at = fill(tab, nullptr, g, n, at, count, 1, block);
    if (at < 0) return (int)cudaErrorInvalidValue;
    if (tab.n == 0) continue;
    const int grid = grid_of(tab.tiles, sms);
    const int rc = by_type(dtype, [&](auto* tag) {
      grad_squares<std::remove_pointer_t<decltype(tag)>, CAP><<<grid, kNT, 0, s>>>(tab, sums + parts);
      return (int)cudaGetLastError();
    });
    if (rc != 0) return rc;
    parts += grid;
  }
  return (int)launch_kernel(grad_norm_kernel, dim3(1), dim3(kNT), 0, s, true, (const double*)sums, parts, norm);
}

constexpr int kFew = 32;

}  // namespace

// How many sums (64-bit) ipex_grad_norm needs for `count` tensors.
IPEX_API int64_t ipex_grad_norm_sums(int64_t count) {
  return (int64_t)sm_count() * kCtas * ((count + kMost - 1) / kMost + 1);
}

// p, g, n [count] (host): addresses and sizes of parameters and gradients of `dtype` (a gradient of 0: its parameter is left as it is,
// and so is its step counter).  Flat buffers of sum(ceil(n / 256)) * 256 elements, aligned to 16 bytes: m, v in 32 bits or (small) in 8,
// with an exponent for each 256 of them; rest: none (0), int16 (1, bf16 alone) or 32-bit (2, 16-bit parameters).  step: one counter, or
// `count` of them; factors: 16 bytes for each.  lr_at (device) stands for lr.  Returns a cudaError_t.
IPEX_API int ipex_adamw_step(const int64_t* p, const int64_t* g, const int64_t* n, int64_t count, void* m, void* v, uint8_t* m_scale,
                             uint8_t* v_scale, void* rest, int rest_kind, int64_t* step, int steps, void* factors, const float* norm,
                             double max_norm, double lr, const float* lr_at, double b1, double b2, double eps, double decay,
                             uint32_t seed, int dtype, int small, void* stream) {
  if (count < 0 || p == nullptr || g == nullptr || n == nullptr || m == nullptr || v == nullptr || step == nullptr || factors == nullptr ||
      (small != 0 && (m_scale == nullptr || v_scale == nullptr)) || (rest_kind != REST_NONE && rest == nullptr) || rest_kind < 0 ||
      rest_kind > 2 || (steps != 1 && steps != count) ||
      ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(rest) |
        reinterpret_cast<uintptr_t>(factors)) & 15))
    return (int)cudaErrorInvalidValue;
  const BeginArgs b = {step, norm, lr_at, (Factors*)factors, max_norm, lr, b1, b2, decay};
  const StepArgs a = {m, v, m_scale, v_scale, rest, (const Factors*)factors, step, (float)b1, (float)(1.0 - b1), (float)b2,
                      (float)(1.0 - b2), (float)eps, seed};
  return count <= kFew ? step_all<kFew>(p, g, n, count, b, a, steps, dtype, small != 0, rest_kind, (cudaStream_t)stream)
                       : step_all<kMost>(p, g, n, count, b, a, steps, dtype, small != 0, rest_kind, (cudaStream_t)stream);
}

// norm: the root of the sum of all gradients' squares; sums: room for ipex_grad_norm_sums(count).
IPEX_API int ipex_grad_norm(const int64_t* g, const int64_t* n, int64_t count, double* sums, float* norm, int dtype, void* stream) {
  if (count < 0 || g == nullptr || n == nullptr || sums == nullptr || norm == nullptr) return (int)cudaErrorInvalidValue;
  return count <= kFew ? norm_all<kFew>(g, n, count, sums, norm, dtype, (cudaStream_t)stream)
                       : norm_all<kMost>(g, n, count, sums, norm, dtype, (cudaStream_t)stream);
}
