// Rows of logits: where they lie, their vectors, and sums of exponentials that hold at any size.
//
// With c = log2(e) / T and r = rint(c max x), exponents are y = c x - r: one fma, whose rounding of r is common to a row and cancels.
// r is whole, so that sums are rescaled by powers of two, exactly.  From |c max x| = 2^24 on, r is no longer within a half of it:
// there y = (x - max x) c.
#pragma once
#include <type_traits>

#include "common/utils.cuh"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr double kLn2_64 = 0.693147180559945309;
constexpr int kErrToken = 61;     // a token outside of the vocabulary

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// An exponent, held above -1e25 (2^-1e25 is 0), so that its product with a sum of up to 2^30 stays finite and 0 times it is 0 for
// hidden tokens (-inf, or the type's lowest value); NaN stays NaN.
__device__ __forceinline__ float held(float y) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(y), "f"(-1.0e25f));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two 32-bit numbers an instruction: x += a, y += b; x += a u, y += b v; x = x c - r, y = y c - r.
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  asm("{\n.reg .b64 u, v;\nmov.b64 u, {%0, %1};\nmov.b64 v, {%2, %3};\nadd.rn.f32x2 u, u, v;\nmov.b64 {%0, %1}, u;\n}\n"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float u, float v) {
  asm("{\n.reg .b64 p, q, r;\nmov.b64 p, {%2, %3};\nmov.b64 q, {%4, %5};\nmov.b64 r, {%0, %1};\n"
      "fma.rn.f32x2 r, p, q, r;\nmov.b64 {%0, %1}, r;\n}\n"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b), "f"(u), "f"(v));
}
__device__ __forceinline__ void exponents2(float& x, float& y, float c, float minus_r) {
  asm("{\n.reg .b64 p, q, r;\nmov.b64 p, {%0, %1};\nmov.b64 q, {%2, %2};\nmov.b64 r, {%3, %3};\n"
      "fma.rn.f32x2 p, p, q, r;\nmov.b64 {%0, %1}, p;\n}\n"
      : "+f"(x), "+f"(y)
      : "f"(c), "f"(minus_r));
}
struct Rows {
  const void* x;
  int64_t s0, s1;      // strides of the outer and the inner row index, in elements
  int64_t n1;          // rows to an outer index
  int V;
};

template <typename T>
__device__ __forceinline__ const T* row_at(const Rows& r, int64_t row) {
  const T* x = reinterpret_cast<const T*>(r.x);
  if (row < r.n1) return x + row * r.s1;           // as all rows are where one stride goes through them (see rows_of)
  const uint32_t outer = (uint32_t)row / (uint32_t)r.n1;
  return x + outer * r.s0 + ((uint32_t)row - outer * (uint32_t)r.n1) * r.s1;
}

// A vector's elements.  bf16 by shifts: a conversion would go through the unit that the exponentials need.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& w, float* f) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      f[i] = __uint_as_float(v[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
    } else {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}

// The larger ones of two pairs of 16-bit numbers; a number before NaN.
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// m: the largest logit (-inf: no token), s: sum of 2^y, t: that sum weighted by y (ENT), or over the tokens not given (TAIL).
struct Stat {
  float m, s, t;
};
// What exponents are taken from: r = rint(c m), or c m itself where m is far from 0.
constexpr float kFar = 0x1p24f;
struct Base {
  float m, r, to;      // to: r, and 0 for no token
  bool far;
  __device__ __forceinline__ Base(float m_, float c) {
    m = m_;
    r = rintf(__fmul_rn(m, c));
    to = r == -INFINITY ? 0.f : r;
    far = !(fabsf(r) < kFar) && m != -INFINITY;
  }
  __device__ __forceinline__ float exponent(float x, float c) const { return far ? (x - m) * c : fmaf(x, c, -to); }
};
// The exponent of the factor that takes sums from one base to another that is not below it.
__device__ __forceinline__ float shift(const Base& from, const Base& to, float c) {
  float d = from.r - to.to;
  if (from.far || to.far)
    d = !to.far ? fmaf(from.m, c, -to.to) : from.far ? (from.m - to.m) * c : -fmaf(to.m, c, -from.r);
  return held(d);
}
template <bool ENT>
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float c) {
  Stat o;
  o.m = fmaxf(a.m, b.m);
  const Base to(o.m, c);
  const float da = shift(Base(a.m, c), to, c), db = shift(Base(b.m, c), to, c);     // sums of a side without tokens are 0
  const float ea = ex2(da), eb = ex2(db);
  o.s = a.s * ea + b.s * eb;
  o.t = ENT ? (a.t + a.s * da) * ea + (b.t + b.s * db) * eb : a.t * ea + b.t * eb;
  return o;
}

// A row whose largest logit is not above -2^127 has no token: -inf, or the lowest values of bf16 and of 32 bits, hide them all.
__device__ __forceinline__ bool no_token(const Stat& st) { return st.s == st.s && !(st.m > -0x1p127f); }

// log sum e^((x - from) / T), from = 0, or m where that is far.  A row's few last operations are done in 64 bits: in 32, they made
// the error of a log probability 1.7 times what its own rounding is.  c is log2(e) / T rounded to 32 bits, and r, rounded from
// c max x, is taken back to the unrounded factor: what is left of c's error is that of the differences to the largest logit.
__device__ __forceinline__ double log_sum(const Base& base, double log2_s, float c, float temp) {
  return (base.far ? 0.0 : base.r * (1.0 / ((double)temp * c))) + log2_s * kLn2_64;
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

bool rows_ok(const void* x, int64_t s0, int64_t s1, int64_t n1, int64_t rows, int V, int elem) {
  return x != nullptr && rows >= 1 && rows <= (1ll << 27) && n1 >= 1 && V >= 1 && V <= (1 << 30) && s0 >= 0 && s1 >= 0 &&
         (reinterpret_cast<uintptr_t>(x) % elem) == 0;
}

bool temp_ok(float t) { return t >= 1e-6f && t <= 1e6f; }

// Rows that follow one another at one stride count as one run of them.
Rows rows_of(const void* x, int64_t s0, int64_t s1, int64_t n1, int64_t rows, int V) {
  return {x, s0, s1, s0 == s1 * n1 || n1 > rows ? rows : n1, V};
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == DT_F16) return f((__half*)nullptr);
  if (dtype == DT_BF16) return f((__nv_bfloat16*)nullptr);
  if (dtype == DT_F32) return f((float*)nullptr);
  return (int)cudaErrorInvalidValue;
}

}  // namespace
