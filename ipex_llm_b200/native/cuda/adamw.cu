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
// the work is split, and 8-bit moments can be told bit by bit.  The one exception: a change below 2^-62 in size, which no parameter
// from 2^-37 on notices, may be off in its last bits (see change_usual).
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
constexpr int kNormParts = 2;               // of a thread's in a tile of the norm: both are asked for before the first is worked on
constexpr int kBlock = 256;                 // elements with a common exponent: a warp's
static_assert(kBlock == 32 * kVec, "a warp has a block");
constexpr int kLow = 32, kHigh = 254;       // exponents of a block: 2^(e - 127)
// To an SM: 64 registers, at which the forms with 8-bit moments spill 16 to 24 bytes a thread.  Three, with up to 80 and no spills, are
// slower all the same: 240 x 40960 with 32-bit moments 40.9 -> 42.2 us, with 8-bit ones 31.7 -> 34.1, 202M with 8-bit ones 537 -> 658.
constexpr int kCtas = 4;
// SMs do not all run at one speed: 32 times as many CTAs are launched at most, of a few tiles each (one tile to a CTA where there are
// fewer).  202M elements with 8-bit moments took 597 us with the CTAs that stay and 547 so, 240 x 40960 with 32-bit ones 46 and 42, 12.6M
// of fp16 with copies and 8-bit moments 56 and 44.  A CTA's tiles lie far apart: with two neighbours to a CTA, what is read at a time has
// gaps, and the first of these took 1210 us.
constexpr int kDealt = 32;
constexpr int kNormCtas = 8;                // of the norm's
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
struct __align__(16) Factors {
  float rate, root, clip, decay;      // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), of the gradient, 1 - lr wd
  uint32_t key;                       // of the random bits
  int usual;                          // whether change_usual() holds, as far as they go
};

// A hash: multiplications by the fractions of the roots of 3 and 2, upper bits brought down before each and behind them.
__device__ __forceinline__ uint32_t almost_mixed(uint32_t x) {
  x = (x ^ (x >> 16)) * 0xBB67AE85u;
  return (x ^ (x >> 15)) * 0x6A09E667u;
}
__device__ __forceinline__ uint32_t mixed(uint32_t x) {
  x = almost_mixed(x);
  return x ^ (x >> 16);
}

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
  float eps;
  uint32_t seed;
};

template <int CAP>
__global__ void adamw_begin(const __grid_constant__ Table<CAP> tab, BeginArgs a) {
  pdl_wait();
  pdl_launch_dependents();      // not before the wait: the step's first loads do not wait for more than this launch's begin
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
  f.key = mixed(mixed((uint32_t)t) + a.seed * 0x9E3779B1u);
  f.usual = a.eps >= 0x1p-38f && a.eps <= 0x1p20f && f.root <= 0x1p6f && (f.rate == 0.f || (f.rate >= 0x1p-60f && f.rate <= 0x1p10f));
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

// ---- pairs of 32-bit numbers: one instruction, each half rounded to nearest by itself
using Pair = float2;
__device__ __forceinline__ Pair both(float x) { return make_float2(x, x); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 x, x, y, z;\n"
      "mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// A product that goes into a sum.  The compiler contracts mul.rn.f32x2 and add.rn.f32x2 (and a fused product with a -0 that it knows);
// it does not know that `zero`, an argument of the launch, is -0.
__device__ __forceinline__ Pair term2(Pair a, Pair b, float zero) { return fma2(a, b, both(zero)); }
__device__ __forceinline__ float rcp_near(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rsqrt_near(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The largest of three by size; NaN if one is NaN.
__device__ __forceinline__ float largest3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// ---- eight elements: as they lie in memory, and as 32-bit numbers
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) == 4 ? 2 : 1];
  __device__ __forceinline__ void load(const T* x) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(w) / 16); ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(x) + i);
  }
  __device__ __forceinline__ void load(const T* x, int have) {      // of any alignment; 0 behind the last one
    __align__(16) T e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = k < have ? x[k] : DT<T>::from_f(0.f);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(w) / 16); ++i) w[i] = reinterpret_cast<const uint4*>(e)[i];
  }
  __device__ __forceinline__ void store(T* x) const {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(w) / 16); ++i) __stcs(reinterpret_cast<uint4*>(x) + i, w[i]);
  }
  __device__ __forceinline__ void store(T* x, int have) const {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < have) x[k] = e[k];
  }
  __device__ __forceinline__ void get(Pair* f) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, float>::value) {
        const float* e = reinterpret_cast<const float*>(w);
        f[k] = make_float2(e[2 * k], e[2 * k + 1]);
      } else {
        const uint32_t x = reinterpret_cast<const uint32_t*>(w)[k];
        if constexpr (std::is_same<T, __nv_bfloat16>::value) f[k] = make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
        else f[k] = __half22float2(*reinterpret_cast<const __half2*>(&x));
      }
    }
  }
  __device__ __forceinline__ void put(const Pair* f) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, float>::value) {
        reinterpret_cast<float2*>(w)[k] = f[k];
      } else {
        uint32_t& x = reinterpret_cast<uint32_t*>(w)[k];
        if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(&x) = __floats2bfloat162_rn(f[k].x, f[k].y);
        else *reinterpret_cast<__half2*>(&x) = __floats2half2_rn(f[k].x, f[k].y);
      }
    }
  }
};

// 2^k for the exponents that occur here (-126 to 127).
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }
// A block's exponent as it is held: 0 in moments that no step has seen.
__device__ __forceinline__ int held(int e) { return min(max(e, kLow), kHigh); }

// The exponent of the largest finite number of a warp's, of 32 x 8.
__device__ __noinline__ int finite_exponent(Pair a, Pair b, Pair c, Pair d) {
  const float x[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  uint32_t top = 0;
  for (int i = 0; i < 8; ++i) {
    const uint32_t bits = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    top = max(top, bits < 0x7F800000u ? bits : 0u);
  }
  return held(__reduce_max_sync(0xffffffffu, top) >> 23);
}

// A 32-bit number's bits are its exponent and fraction in a row, whatever its size: scaled so that its exponent field is the small
// format's, adding random bits below the last kept place and cutting there rounds it up with the probability of what is cut off.
// The codes, in the uppermost bytes; `chance` is the hash but for its last step: that leaves the upper half (v's bits) as it is, and
// for the lower one (m's) it is taken here, with the shift.
__device__ __forceinline__ uint32_t to_e4m3(float x, float scaled, uint32_t chance) {
  const uint32_t t = (__float_as_uint(scaled) + ((chance << 4 ^ chance >> 12) & 0xFFFF0u) + 8u) << 4;      // its sign is shifted out
  return t | (__float_as_uint(x) & 0x80000000u);
}
__device__ __forceinline__ uint32_t to_e5m2(float x, float scaled, uint32_t chance) {
  const uint32_t t = (__float_as_uint(scaled) + ((chance >> 11 & 0x1FFFE0u) | 16u)) << 3;
  return x > 0.f ? max(t, 1u << 24) : t;            // what is not 0 does not become 0
}
// Of what no power of two takes there at once: numbers from 2^8 (m) and 2^15 (v) on, and what is not finite.
__device__ __noinline__ uint32_t to_e4m3_any(float x, int e, uint32_t chance) {
  const float a = fabsf(x);
  return a < INFINITY ? to_e4m3(x, __fmul_rn(__fmul_rn(a, pow2(134 - e)), 0x1p-120f), chance) : 0x7F000000u;
}
__device__ __noinline__ uint32_t to_e5m2_any(float x, int e, uint32_t chance) {
  if (!(x < INFINITY)) return x == INFINITY ? 0x7C000000u : 0x7F000000u;
  return to_e5m2(x, __fmul_rn(__fmul_rn(x, pow2(141 - e)), 0x1p-112f), chance);
}
template <__nv_fp8_interpretation_t KIND>
__device__ __forceinline__ void from_fp8(uint2 w, float down, Pair* f) {
  const uint32_t v[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v[i >> 1] >> (16 * (i & 1))), KIND);
    f[i] = mul2(__half22float2(*reinterpret_cast<const __half2*>(&h)), both(down));
  }
}
// The uppermost bytes of eight words.
__device__ __forceinline__ uint2 upper_bytes(const uint32_t* t) {
  return make_uint2(__byte_perm(__byte_perm(t[0], t[1], 0x0073), __byte_perm(t[2], t[3], 0x0073), 0x5410),
                    __byte_perm(__byte_perm(t[4], t[5], 0x0073), __byte_perm(t[6], t[7], 0x0073), 0x5410));
}

struct StepArgs {
  void* m;
  void* v;
  uint8_t* m_scale;    // exponents of blocks of 8-bit moments
  uint8_t* v_scale;
  void* rest;          // the 16 bits below bf16, or copies in 32 bits
  const Factors* factors;
  float b1, c1, b2, c2, eps;     // c: 1 - b
  float zero;                    // -0
};

__device__ __forceinline__ float change_any(float m, float v, const Factors& f, float eps) {
  return -__fdiv_rn(__fmul_rn(m, f.rate), __fadd_rn(__fmul_rn(__fsqrt_rn(v), f.root), eps));
}

// The update's change, -m rate / (sqrt(v) root + eps), where every number is of a usual size: roots by Newton's step from an
// approximate 1 / sqrt, quotients by Newton's step for the reciprocal and Markstein's for the quotient, with signs such that none has
// to be turned.  All are the nearest numbers: the root and the reciprocal for every fraction there is (tested), the quotient by
// Markstein's theorem, as long as remainders are exact: while m rate is 0 or above 2^-100 in size (below, the quotient by a divisor of
// 2^-38 or more is below 2^-62, and its last bits may be others); v is taken times 2^64, with 2^-102 for 0, which no other v
// notices, or eps absorbs.  17 instructions for two elements; the general root and division take three
// times as many, and a branch each.
__device__ __forceinline__ Pair change_usual(Pair m, Pair v, const Factors& f, float eps, float zero) {
  const Pair u = fma2(v, both(-0x1p64f), both(-0x1p-102f));       // -2^64 v
  const Pair y = make_float2(rsqrt_near(-u.x), rsqrt_near(-u.y));
  const Pair g = mul2(u, y);                                      // about -sqrt
  const Pair s = fma2(fma2(g, g, u), mul2(y, both(0.5f)), g);     // -sqrt
  const Pair d = add2(term2(s, both(f.root * 0x1p-32f), zero), both(-eps));
  const Pair n = mul2(m, both(-f.rate));
  const Pair r0 = make_float2(rcp_near(-d.x), rcp_near(-d.y));
  const Pair r = fma2(fma2(d, r0, both(1.f)), r0, r0);
  const Pair q = mul2(n, r);
  return fma2(fma2(d, q, n), r, q);
}

// A pair of bf16 numbers with what their 32-bit numbers have below them, from -2^15 to 2^15 - 1.
__device__ __forceinline__ Pair with_rest(uint32_t p, uint32_t r) {
  uint32_t lo;
  asm("prmt.b32 %0, %1, 0, 0x9910;" : "=r"(lo) : "r"(r));        // the lower half with its sign
  return make_float2(__uint_as_float(p * 65536u + lo), __uint_as_float((p & 0xFFFF0000u) + (uint32_t)((int)r >> 16)));
}

// Eight elements of a thread: what is read of them, and their update.
template <typename T, bool SMALL, int REST>
struct Eight {
  Raw8<T> g, p;
  Raw8<float> copy, wide_m, wide_v;
  uint4 low;
  uint2 m, v;
  int em, ev;

  __device__ __forceinline__ void load(const StepArgs& a, const T* g_at, const T* p_at, int64_t at, int have, bool vec) {
    if (vec) {
      g.load(g_at);
      if constexpr (REST != REST_32) p.load(p_at);
    } else {
      g.load(g_at, have);
      if constexpr (REST != REST_32) p.load(p_at, have);
    }
    if constexpr (REST == REST_32) copy.load(reinterpret_cast<const float*>(a.rest) + at);
    if constexpr (REST == REST_16) low = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const int16_t*>(a.rest) + at));
    if constexpr (SMALL) {
      m = __ldcs(reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(a.m) + at));
      v = __ldcs(reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(a.v) + at));
      em = a.m_scale[at / kBlock];
      ev = a.v_scale[at / kBlock];
    } else {
      wide_m.load(reinterpret_cast<const float*>(a.m) + at);
      wide_v.load(reinterpret_cast<const float*>(a.v) + at);
    }
  }

  __device__ __forceinline__ void update(const StepArgs& a, const Factors& f, T* p_at, int64_t at, int have, bool vec) {
    Pair w[4], d[4], mm[4], vv[4];
    g.get(d);
    if constexpr (REST == REST_32) {
      copy.get(w);
    } else if constexpr (REST == REST_16) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = with_rest(reinterpret_cast<const uint32_t*>(p.w)[k], reinterpret_cast<const uint32_t*>(&low)[k]);
    } else {
      p.get(w);
    }
    if constexpr (SMALL) {
      from_fp8<__NV_E4M3>(m, pow2(held(em) - 134), mm);
      from_fp8<__NV_E5M2>(v, pow2(held(ev) - 141), vv);
    } else {
      wide_m.get(mm);
      wide_v.get(vv);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const Pair y = mul2(d[k], both(f.clip));
      mm[k] = add2(term2(mm[k], both(a.b1), a.zero), term2(y, both(a.c1), a.zero));
      vv[k] = add2(term2(vv[k], both(a.b2), a.zero), term2(mul2(y, y), both(a.c2), a.zero));
    }
    if (have < kVec) {                                // behind the tensor's end
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (2 * k >= have) mm[k].x = vv[k].x = 0.f;
        if (2 * k + 1 >= have) mm[k].y = vv[k].y = 0.f;
      }
    }
    float top_m = 0.f, top_v = 0.f, top_p = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      top_m = largest3(top_m, mm[k].x, mm[k].y);
      top_v = largest3(top_v, vv[k].x, vv[k].y);
    }
    if (f.usual && top_m < 0x1p60f && top_v < 0x1p60f) {
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k] = change_usual(mm[k], vv[k], f, a.eps, a.zero);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        d[k] = make_float2(change_any(mm[k].x, vv[k].x, f, a.eps), change_any(mm[k].y, vv[k].y, f, a.eps));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = add2(term2(w[k], both(f.decay), a.zero), d[k]);
      if constexpr (REST == REST_16) top_p = largest3(top_p, w[k].x, w[k].y);
    }
    if (REST != REST_NONE && have < kVec) {           // 0 / eps, or 0 / 0
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (2 * k >= have) w[k].x = 0.f;
        if (2 * k + 1 >= have) w[k].y = 0.f;
      }
    }
    if constexpr (SMALL) {
      int e = held(__reduce_max_sync(0xffffffffu, __float_as_uint(top_m)) >> 23);
      int h = held(__reduce_max_sync(0xffffffffu, __float_as_uint(top_v)) >> 23);
      const uint32_t first = (uint32_t)at * 0x9E3779B1u + (uint32_t)(at >> 32) * 0xBB67AE85u + f.key;
      uint32_t tm[8], tv[8];
      if (e <= 134 && h <= 141) {                     // all of the block below 2^8 and 2^15: one power of two is enough
        const float up_m = pow2(14 - e), up_v = pow2(29 - h);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t c0 = almost_mixed(first + 2 * k * 0x9E3779B1u), c1 = almost_mixed(first + (2 * k + 1) * 0x9E3779B1u);
          const Pair sv = mul2(vv[k], both(up_v)), sm = mul2(mm[k], both(up_m));
          tm[2 * k] = to_e4m3(mm[k].x, sm.x, c0);
          tm[2 * k + 1] = to_e4m3(mm[k].y, sm.y, c1);
          tv[2 * k] = to_e5m2(vv[k].x, sv.x, c0);
          tv[2 * k + 1] = to_e5m2(vv[k].y, sv.y, c1);
        }
      } else {
        e = finite_exponent(mm[0], mm[1], mm[2], mm[3]);
        h = finite_exponent(vv[0], vv[1], vv[2], vv[3]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t c0 = almost_mixed(first + 2 * k * 0x9E3779B1u), c1 = almost_mixed(first + (2 * k + 1) * 0x9E3779B1u);
          tm[2 * k] = to_e4m3_any(mm[k].x, e, c0);
          tm[2 * k + 1] = to_e4m3_any(mm[k].y, e, c1);
          tv[2 * k] = to_e5m2_any(vv[k].x, h, c0);
          tv[2 * k + 1] = to_e5m2_any(vv[k].y, h, c1);
        }
      }
      __stcs(reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.m) + at), upper_bytes(tm));
      __stcs(reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.v) + at), upper_bytes(tv));
      if ((threadIdx.x & 31) == 0) {
        a.m_scale[at / kBlock] = (uint8_t)e;
        a.v_scale[at / kBlock] = (uint8_t)h;
      }
    } else {
      wide_m.put(mm);
      wide_m.store(reinterpret_cast<float*>(a.m) + at);
      wide_v.put(vv);
      wide_v.store(reinterpret_cast<float*>(a.v) + at);
    }
    if constexpr (REST == REST_16) {
      // bf16 nearest to p (halves up): its upper half, one more where the lower half is 2^15 or more.  What is left, from -2^15 to
      // 2^15 - 1, is the lower half as it stands.
      uint32_t* to = reinterpret_cast<uint32_t*>(p.w);
      uint32_t* r = reinterpret_cast<uint32_t*>(&low);
      if (!(top_p < INFINITY)) {                      // NaN's bits may run over
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (w[k].x != w[k].x) w[k].x = __uint_as_float(0x7FFF0000u);
          if (w[k].y != w[k].y) w[k].y = __uint_as_float(0x7FFF0000u);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = __float_as_uint(w[k].x), hi = __float_as_uint(w[k].y);
        r[k] = __byte_perm(lo, hi, 0x5410);
        to[k] = __byte_perm(lo + 0x8000u, hi + 0x8000u, 0x7632);
      }
      __stcs(reinterpret_cast<uint4*>(reinterpret_cast<int16_t*>(a.rest) + at), low);
    } else {
      if constexpr (REST == REST_32) {
        copy.put(w);
        copy.store(reinterpret_cast<float*>(a.rest) + at);
      }
      p.put(w);
    }
    if (vec) p.store(p_at);
    else p.store(p_at, have);
  }
};

template <typename T, bool SMALL, int REST, int CAP>
__global__ void __launch_bounds__(kNT, kCtas) adamw_step(const __grid_constant__ Table<CAP> tab, StepArgs a) {
  int i = 0;
  bool first = true;
  for (uint32_t tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x) {
    i = tensor_of(tab, tile, i);
    const Entry& e = tab.e[i];
    const int64_t off = (int64_t)(tile - e.tile) * kTile + threadIdx.x * kVec, at = (int64_t)e.block * kBlock + off;
    const int64_t left = e.n - off;
    if (left + (int)(threadIdx.x & 31) * kVec <= 0) continue;      // no block of the warp's
    T* p_at = reinterpret_cast<T*>(e.p) + off;
    const T* g_at = reinterpret_cast<const T*>(e.g) + off;
    const int have = (int)max((int64_t)0, min((int64_t)kVec, left));
    const bool vec = have == kVec && ((reinterpret_cast<uintptr_t>(e.p) | reinterpret_cast<uintptr_t>(e.g)) & 15) == 0;
    Eight<T, SMALL, REST> x;
    x.load(a, g_at, p_at, at, have, vec);
    if (first) pdl_wait();                            // what the launch in front of this one writes is not among it
    first = false;
    const Factors f = a.factors[e.step];
    x.update(a, f, p_at, at, have, vec);
  }
}

// ------------------------------------------------------------------------------------------------ the norm of all gradients
// Eight squares are added in 32 bits, their sums in 64: a thread's, then a CTA's, then those of all CTAs in their order.  Where a sum
// of eight is too large or too small for 32 bits, they are taken in 64.
template <typename T, int CAP>
__global__ void __launch_bounds__(kNT) grad_squares(const __grid_constant__ Table<CAP> tab, double* sums) {
  __shared__ double part[kNT / 32];
  pdl_wait();
  pdl_launch_dependents();
  double total = 0.0;
  int i = 0;
  for (uint32_t tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x) {
    i = tensor_of(tab, tile, i);
    const Entry& e = tab.e[i];
    const int64_t off = (int64_t)(tile - e.tile) * (kTile * kNormParts) + threadIdx.x * kVec;
    const T* at = reinterpret_cast<const T*>(e.g) + off;
    const bool aligned = (reinterpret_cast<uintptr_t>(e.g) & 15) == 0;
    Raw8<T> w[kNormParts];
#pragma unroll
    for (int h = 0; h < kNormParts; ++h) {
      const int have = (int)max((int64_t)0, min((int64_t)kVec, e.n - off - h * kTile));
      if (have == kVec && aligned) w[h].load(at + h * kTile);
      else w[h].load(at + h * kTile, have);
    }
#pragma unroll
    for (int h = 0; h < kNormParts; ++h) {
      Pair g[4], s = both(0.f);
      w[h].get(g);
#pragma unroll
      for (int k = 0; k < 4; ++k) s = fma2(g[k], g[k], s);
      const float sum = s.x + s.y;
      if (sum > 1e-25f && sum < 1e38f) {
        total += (double)sum;
      } else {
        for (int k = 0; k < 4; ++k) total += (double)g[k].x * g[k].x + (double)g[k].y * g[k].y;
      }
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

// The tensors [from, to) that have a gradient, at most CAP of them, as a table of tiles of `tile` elements; `block`: where the moments of tensor `from` begin.
// Returns the tensor behind the last one, -1 for a size that is not allowed.
template <int CAP>
int64_t fill(Table<CAP>& tab, const int64_t* p, const int64_t* g, const int64_t* n, int64_t from, int64_t to, int steps, int tile,
             uint64_t& block) {
  tab.n = 0;
  tab.tiles = 0;
  int64_t i = from;
  for (; i < to && tab.n < CAP; ++i) {
    const uint64_t blocks = ((uint64_t)n[i] + kBlock - 1) / kBlock, tiles = ((uint64_t)n[i] + tile - 1) / tile;
    if (n[i] < 0 || n[i] > (int64_t)1 << 40 || block + blocks > 0xFFFFFFFFull) return -1;
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

int grid_of(uint32_t tiles, int ctas) { return (int)(tiles < (uint32_t)ctas ? tiles : (uint32_t)ctas); }

template <int CAP>
int step_all(const int64_t* p, const int64_t* g, const int64_t* n, int64_t count, const BeginArgs& b, const StepArgs& a, int steps,
             int dtype, bool small, int rest, cudaStream_t s) {
  const int sms = sm_count();
  if (sms == 0) return (int)cudaErrorInvalidDevice;
  Table<CAP> tab;
  uint64_t block = 0;
  bool begun = false;
  for (int64_t at = 0; at < count;) {
    at = fill(tab, p, g, n, at, count, steps, kTile, block);
    if (at < 0) return (int)cudaErrorInvalidValue;
    if (tab.n == 0) continue;
    if (!begun || steps > 1) {                      // a common counter moves once
      cudaError_t e;
      if (steps > 1) {
        e = launch_kernel(adamw_begin<CAP>, dim3((tab.n + 127) / 128), dim3(128), 0, s, true, tab, b);
      } else {                                      // and needs no table: 25 KB of parameters less
        Table<1> one = {};
        one.n = 1;
        e = launch_kernel(adamw_begin<1>, dim3(1), dim3(32), 0, s, true, one, b);
      }
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
      return (int)launch_kernel(kern, dim3(grid_of(tab.tiles, sms * kCtas * kDealt)), dim3(kNT), 0, s, true, tab, a);
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
    at = fill(tab, nullptr, g, n, at, count, 1, kTile * kNormParts, block);
    if (at < 0) return (int)cudaErrorInvalidValue;
    if (tab.n == 0) continue;
    const int grid = grid_of(tab.tiles, sms * kNormCtas);
    const int rc = by_type(dtype, [&](auto* tag) {
      return (int)launch_kernel(grad_squares<std::remove_pointer_t<decltype(tag)>, CAP>, dim3(grid), dim3(kNT), 0, s, true, tab, sums + parts);
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
  return (int64_t)sm_count() * kNormCtas * ((count + kMost - 1) / kMost + 1);
}

// p, g, n [count] (host): addresses and sizes of parameters and gradients of `dtype` (a gradient of 0: its parameter is left as it is,
// and so is its step counter).  Flat buffers of sum(ceil(n / 256)) * 256 elements, aligned to 16 bytes: m, v in 32 bits or (small) in 8,
// with an exponent for each 256 of them; rest: none (0), int16 (1, bf16 alone) or 32-bit (2, 16-bit parameters).  step: one counter, or
// `count` of them; factors: 32 bytes for each.  lr_at (device) stands for lr.  Returns a cudaError_t.
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
  const BeginArgs b = {step, norm, lr_at, (Factors*)factors, max_norm, lr, b1, b2, decay, (float)eps, seed};
  const StepArgs a = {m, v, m_scale, v_scale, rest, (const Factors*)factors, (float)b1, (float)(1.0 - b1), (float)b2,
                      (float)(1.0 - b2), (float)eps, -0.f};
  return count <= kFew ? step_all<kFew>(p, g, n, count, b, a, steps, dtype, small != 0, rest_kind, (cudaStream_t)stream)
                       : step_all<kMost>(p, g, n, count, b, a, steps, dtype, small != 0, rest_kind, (cudaStream_t)stream);
}

// norm: the root of the sum of all gradients' squares; sums: room for ipex_grad_norm_sums(count).
IPEX_API int ipex_grad_norm(const int64_t* g, const int64_t* n, int64_t count, double* sums, float* norm, int dtype, void* stream) {
  if (count < 0 || g == nullptr || n == nullptr || sums == nullptr || norm == nullptr) return (int)cudaErrorInvalidValue;
  return count <= kFew ? norm_all<kFew>(g, n, count, sums, norm, dtype, (cudaStream_t)stream)
                       : norm_all<kMost>(g, n, count, sums, norm, dtype, (cudaStream_t)stream);
}
