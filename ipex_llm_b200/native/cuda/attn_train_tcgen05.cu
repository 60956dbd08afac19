// Attention with a gradient on the 5th-generation tensor cores, sm_100a: forward keeps one number a row (the logarithm of the
// soft-max's sum), backward computes the probabilities from it again.
//
//   s_ij = scale q_i . k_j     P_ij = e^(s_ij - L_i)     o_i = sum_j P_ij v_j          L_i = log sum_j e^(s_ij) over seen keys
//   dP_ij = dO_i . v_j         delta_i = dO_i . o_i      dS_ij = P_ij (dP_ij - delta_i)
//   dq_i = scale sum_j dS_ij k_j      dk_j = scale sum_i dS_ij q_i      dv_j = sum_i P_ij dO_i
//
// Query i sees key j if the key is not hidden and, when causal, j <= i + Skv - Sq, and with a window also
// j > i + Skv - Sq - window.  A row that sees nothing gives zeros and gets no gradient.  Key heads are shared by Hq / Hkv
// query heads; their gradients are summed over those inside one CTA, in a fixed order: no result depends on an order of atomics.
//
// Tiles are 128 x 128.  All operands come by TMA from 4-D maps (width, rows, heads, sequences) of the tensors as they lie, in
// the 128-byte swizzle; what lies outside of a sequence, or past a head's width, reads as zero.  One tile in shared memory
// serves as a K-major operand (rows are M or N: q, k in s; dO, v in dP) and as an MN-major one (rows are summed over: v in o,
// k in dq, q and dO in dk and dv).  Probabilities and dS go back to tensor memory in 16 bits, over the scores that they were
// made from, and are the products' first operand there.
//
// The products are issued by one warp in an order that leaves the arithmetic of one tile under the products of another:
//   forward     two tiles of queries with eight warps each take turns, two threads to a row
//   dk and dv   transposed scores (rows are keys), so that P^T and dS^T are what the products want; s of the next step runs
//               under this step's dS, dP of the next under the next P
//   dq          a pass of its own over the keys, which computes s and dP once more (7 products in all where 5 would do): the
//               sums then need no atomics, whose order would change results, and no 32-bit dq in global memory
// Sixteen warps of arithmetic hide each other's latencies: with eight, two to a scheduler, an exponential's chain (product,
// special function, conversion) showed, and a block of 128 x 128 took 2900 clocks forward, 3800 for dk and dv and 3250 for dq, of
// which the products alone are 1030, 2180 and 1540.  Now they are 2530, 3570 and 3060: 4096 tokens, 64 heads of 128 over 8 of keys,
// causal, bf16 take 332, 515 and 395 us (37 for the pass before the backward) at 1.78 GHz, where one CTA has at most 233, 256 and 229
// blocks (228 on average).
// With all arithmetic taken out a block still takes 1700 (forward) and 2870 clocks (dk and dv): the products' issue and arrivals
// between the roles are what is left to win.
//
// In the transposed scores L_i and delta_i belong to columns, not to the threads' rows.  Read from shared memory, four numbers a
// request, they took a third of its bandwidth, which the products need.  So they are summed by the products too: one more step
// of 16 columns, in which a query's row holds -L_i / scale (or -delta_i) in pieces of 16 bits, and every key's row the pieces'
// weights.
//
// In fp16 the range of dS is what is short, not its precision: P is taken times 2^12, and dP - delta times a power of two that a
// bound on |dO_i| |v_j| gives for each group of heads, so that the largest dS comes near 2^15.  Both go out of the results again.
//
// Every wait is bounded; one that runs out raises the CTA's abort flag, all roles leave, and the error word gets 71 (loader), 72
// (products), 73 (soft-max).  No cluster multicast.
#include "common/utils.cuh"
#include "tcgen05_common.cuh"

namespace {

using namespace tc5;

constexpr int kT = 128;           // rows of a tile of queries or keys
constexpr int kArith = 16;        // warps of arithmetic
constexpr int kLoader = kArith, kIssuer = kArith + 1;
constexpr int kThreads = 32 * (kArith + 2);
constexpr uint32_t kTmemCols = 512;
constexpr int kShiftF16 = 12;     // P is stored times 2^12 in fp16
template <typename T> __host__ __device__ constexpr float shift_of() { return std::is_same<T, __half>::value ? kShiftF16 : 0; }
template <typename T> __host__ __device__ constexpr float scale_of() { return std::is_same<T, __half>::value ? 1 << kShiftF16 : 1; }
// delta_i is the difference of all dP_ij of a row: with the rounded o its error reaches every dS_ij of the row with the same sign
// and adds a third to the error of dq and dk (measured: 1.53 times the final rounding's instead of 1.42).  So what rounding takes
// from o is kept too, rounded once more, times 2^11 so that it does not fall among fp16's subnormals.
constexpr float kLowScale = 2048.f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four-dimensional tile load: 64 columns from x on of 128 rows from y on of head h, sequence b.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* tm, int x, int y, int h, int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(h), "r"(b), "r"(smem_u32(bar))
      : "memory");
}
// A tile of D columns: D / 64 blocks of [128 rows x 128 bytes] behind one another.
template <int D>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* tm, int row, int h, int b, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c) tma_load_4d(dst + c * (kT * 128), tm, c * 64, row, h, b, bar);
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 32 lanes x 32 columns without the wait, and the wait; values are there only behind it.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld_wait(float (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < N; ++j) asm volatile("" : "+f"(v[j]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] . B[smem]; issued by one thread.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// The same tile read with its rows as the summed-over dimension (MN-major): 64 columns of 128 bytes are one swizzle atom wide,
// atoms of further columns follow after a block of 128 rows (leading offset), groups of eight rows after 1024 bytes (stride).
__device__ __forceinline__ uint64_t make_desc_mn(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((kT * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
constexpr uint32_t kBMajorMN = 1u << 16;
// 16 columns of a K-major operand without a swizzle: rows of eight columns, 16 bytes, lie behind one another; the second eight
// columns begin `second` bytes behind the first (leading offset), eight rows take 128 bytes (stride).
__device__ __forceinline__ uint64_t make_desc_rows16(uint32_t smem_addr, uint32_t second) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(second >> 4) << 16;
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  return d;
}

// acc = A . B^T over D columns, both tiles K-major.
template <int D>
__device__ __forceinline__ void mma_rows(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      umma_f16(d, a + c * (kT * 128 >> 4) + 2 * kk, b + c * (kT * 128 >> 4) + 2 * kk, idesc, (c | kk) != 0);
}
// acc (+)= A . B over 128 rows of B: A in tensor memory, 16 bits, each 2 * RUN of its columns (RUN of tensor memory) packed into
// the front of the PITCH columns of scores that they were made from.
template <int RUN, int PITCH>
__device__ __forceinline__ void mma_sum(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    umma_ts(d, a + kk * 8 / RUN * PITCH + kk * 8 % RUN, b + kk * (16 * 128 >> 4), idesc, accumulate || kk != 0);
}
// What a warp has written to tensor memory goes to the products: one arrival a warp.
__device__ __forceinline__ void hand_over(uint64_t* bar, int lane) {
  tmem_st_wait();
  tcgen05_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// A number that is the same in the whole warp, for the compiler to know: products take their operands from uniform registers, and
// with bounds or offsets that came out of a division every one of them took 64 clocks to issue, as long as it runs.
__device__ __forceinline__ int uniform(int x) { return (int)__reduce_max_sync(0xffffffffu, (unsigned)x); }

// Two 32-bit numbers an instruction.
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b) {   // x *= a, y *= b
  asm("{\n"
      ".reg .b64 u, v;\n"
      "mov.b64 u, {%0, %1};\n"
      "mov.b64 v, {%2, %3};\n"
      "mul.rn.f32x2 u, u, v;\n"
      "mov.b64 {%0, %1}, u;\n"
      "}\n"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {   // x += a, y += b
  asm("{\n"
      ".reg .b64 u, v;\n"
      "mov.b64 u, {%0, %1};\n"
      "mov.b64 v, {%2, %3};\n"
      "add.rn.f32x2 u, u, v;\n"
      "mov.b64 {%0, %1}, u;\n"
      "}\n"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b) {   // x = x a + b, y = y a + b
  asm("{\n"
      ".reg .b64 u, v, w;\n"
      "mov.b64 u, {%0, %1};\n"
      "mov.b64 v, {%2, %2};\n"
      "mov.b64 w, {%3, %3};\n"
      "fma.rn.f32x2 u, u, v, w;\n"
      "mov.b64 {%0, %1}, u;\n"
      "}\n"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// What rounding to 16 bits took from two numbers, in 16 bits.
template <typename T>
__device__ __forceinline__ uint32_t rest2(uint32_t rounded, float lo, float hi) {
  const T* v = reinterpret_cast<const T*>(&rounded);
  return pack2<T>(lo - to_float<T>(v[0]), hi - to_float<T>(v[1]));
}

// 32 rows x 32 columns of a warp, a row to a lane, times `f`, in 16 bits to shared memory (2 KB, the 64-byte swizzle), from where a
// TMA store takes them to [b][h] of a tensor: whole sectors, where every lane storing its own row cost 2 to 6 us a tile.  What lies
// past the tensor is not stored.
template <typename T>
__device__ __forceinline__ void stage32(uint8_t* st, const float (&v)[32], float f, int lane) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 w;
    w.x = pack2<T>(v[8 * q] * f, v[8 * q + 1] * f);
    w.y = pack2<T>(v[8 * q + 2] * f, v[8 * q + 3] * f);
    w.z = pack2<T>(v[8 * q + 4] * f, v[8 * q + 5] * f);
    w.w = pack2<T>(v[8 * q + 6] * f, v[8 * q + 7] * f);
    *reinterpret_cast<uint4*>(st + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4)) = w;
  }
  fence_proxy_async_smem();
  __syncwarp();
}
__device__ __forceinline__ void store32(const CUtensorMap* tm, const uint8_t* st, int x, int y, int h, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(tm)),
               "r"(smem_u32(st)), "r"(x), "r"(y), "r"(h), "r"(b)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until at most N of this thread's stores have yet to read shared memory.
template <int N>
__device__ __forceinline__ void stores_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

struct Shape {
  int B, Hq, Hkv, Sq, Skv, D;
  int causal, window;        // window 0: none
  int q_pad;                 // row stride of the statistics: Sq rounded up to 128
  int k_words;               // 32-bit words of a sequence's mask of keys
  const uint32_t* mask;      // [B, k_words] or null: bit j: key j is real
  float scale, scale_log2;
  int* err;
};

// Bits [lo, hi) of the 32 from bit `at` on.
__device__ __forceinline__ uint32_t range_bits(int lo, int hi, int at) {
  lo = min(max(lo - at, 0), 32);
  hi = min(max(hi - at, 0), 32);
  const uint32_t below_hi = hi >= 32 ? 0xFFFFFFFFu : (1u << hi) - 1;
  const uint32_t below_lo = lo >= 32 ? 0xFFFFFFFFu : (1u << lo) - 1;
  return below_hi & ~below_lo;
}

// Blocks of keys that rows [q0, q0 + 128) may see.
__device__ __forceinline__ void key_blocks(const Shape& s, int q0, int& j0, int& j1) {
  const int off = s.Skv - s.Sq, last = min(q0 + kT, s.Sq) - 1;
  const int hi = last < q0 ? 0 : s.causal ? min(s.Skv, last + off + 1) : s.Skv;
  const int lo = s.window > 0 ? max(0, q0 + off - s.window + 1) : 0;
  j0 = lo / kT;
  j1 = hi > lo ? (hi + kT - 1) / kT : j0;
}
// The keys of a row: [lo, hi).
__device__ __forceinline__ void row_keys(const Shape& s, int q, int& lo, int& hi) {
  const int off = s.Skv - s.Sq;
  hi = s.causal ? min(s.Skv, q + off + 1) : s.Skv;
  lo = s.window > 0 ? max(0, q + off - s.window + 1) : 0;
}

// Rows before this one may see fewer than kFew keys (those of a window with holes apart); the whole warp calls it.
//
// P and dS are rounded to 16 bits on their way into a product.  That alone takes dq and dk from one rounding to two (1.41 times
// the error); the error of P in o, and so in delta, adds 1 / keys of a row to it, and short rows are also those with the largest
// gradients: sequences of a few to 64 tokens came to 1.45 to 1.6 times.  So tiles with such rows give the products what rounding
// took, too, in a second step over columns that the scores have left: the first tile of a causal sequence, or all of a short one.
constexpr int kFew = 64;
__device__ __forceinline__ int few_queries(const Shape& s, int b, int lane) {
  constexpr int kAll = 0x7FFFFFFF;
  if (s.window > 0 && s.window < kFew) return kAll;
  int enough = s.Skv >= kFew ? kFew : kAll;        // so many keys from the front hold kFew real ones
  if (s.mask != nullptr) {
    const uint32_t* words = s.mask + (int64_t)b * s.k_words;
    enough = kAll;
    for (int w = 0, seen = 0; w < s.k_words && enough == kAll; w += 32) {
      int n = w + lane < s.k_words ? __popc(__ldg(words + w + lane)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int before = __shfl_up_sync(0xffffffffu, n, o);
        n += lane >= o ? before : 0;
      }
      const uint32_t there = __ballot_sync(0xffffffffu, seen + n >= kFew);
      if (there != 0) enough = min(s.Skv, (w + __ffs(there)) * 32);
      seen += __shfl_sync(0xffffffffu, n, 31);
    }
  }
  return enough == kAll ? kAll : s.causal ? max(0, enough - 1 - (s.Skv - s.Sq)) : 0;
}

// So do all rows of dq in heads below 64.  The keys that a row sees have a part along its query in common, over which dS sums to 0
// while its rounding does not, and the fewer the dimensions the larger that part: 1.44 times the final rounding's error with 128,
// 1.5 with 32 (1.03 so; dk, whose sums run over queries, has 1.41 to 1.44).  It costs 14 % of dq: 79 us for 4 x 1024 tokens and 32
// heads of 56, 69 for heads of 64.
__device__ __forceinline__ bool rest_of_dq(const Shape& s) { return s.D < 64; }

// A CTA stays on its SM and takes tiles of work, sorted from long to short, in turn with the others, every second round
// backwards.  (A CTA to a tile cost 5 us between the last product of one and the first of the next, for barriers, tensor memory,
// cold loads; here the ring of tiles runs on.)
__device__ __forceinline__ unsigned item_of(int round) {
  return round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// What a CTA takes down in every case.
__device__ __forceinline__ void finish(uint32_t tmem_base, int warp) {
  tcgen05_fence_before();
  __syncthreads();
  if (warp == kIssuer) tmem_dealloc(tmem_base, kTmemCols);
}

// ------------------------------------------------------------------------------------------------ forward
// Outputs go by the maps tm_o and, with nlse, tm_low: what rounding took from them, times kLowScale.
struct FwdArgs {
  Shape s;
  float* nlse;        // [B, Hq, q_pad]: -L log2(e) (+ the shift of fp16); -inf for rows that see nothing and past Sq; or null
  unsigned items;
};

template <int D>
struct FwdSmem {
  static constexpr int kTile = kT * D * 2;
  static constexpr int kStages = D == 128 ? 4 : 6;
  static constexpr int kXch = (2 + kStages) * kTile;            // maxima and sums of half rows, two of each
  static constexpr int kBars = kXch + 2 * 2 * 2 * kT * 4;
  static constexpr int kSize = 1024 + kBars + 512;
};

// Two tiles of queries [q0, q0 + 256) of a head.
struct FwdItem {
  int q0, h, b, kvh, j0[2], j1[2], ja, jb;
  __device__ __forceinline__ FwdItem(const Shape& s, unsigned i) {
    const int pairs = (s.Sq + 2 * kT - 1) / (2 * kT);
    const unsigned rest = i / s.Hq;
    h = (int)(i % s.Hq);
    b = (int)(rest % s.B);
    q0 = (pairs - 1 - (int)(rest / s.B)) * 2 * kT;
    kvh = h / (s.Hq / s.Hkv);
    key_blocks(s, q0, j0[0], j1[0]);
    key_blocks(s, q0 + kT, j0[1], j1[1]);
    const bool two = j1[1] > j0[1];
    ja = two ? (j1[0] > j0[0] ? min(j0[0], j0[1]) : j0[1]) : j0[0];
    jb = two ? max(j1[0], j1[1]) : j1[0];
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                const __grid_constant__ CUtensorMap tm_low, const __grid_constant__ FwdArgs a) {
  using L = FwdSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + 2 * L::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* kv_full = bars + 2;
  uint64_t* kv_empty = kv_full + L::kStages;
  uint64_t* s_full = kv_empty + L::kStages;    // [2]
  uint64_t* p_full = s_full + 2;               // [2]
  uint64_t* o_full = p_full + 2;               // [2]
  uint64_t* x_full = o_full + 2;               // [8]: the two warps of 32 rows
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(x_full + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const Shape& s = a.s;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, kArith);
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kArith / 2);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&x_full[i], 2);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kIssuer) tmem_alloc(tmem_slot, kTmemCols);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);

  if (warp == kLoader) {
    // ---------------- loader: keys and values of a block take a stage each, in turn ----------------
    if (lane == 0) {
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
      bool ok = true;
      int n = 0, w = 0;
      for (; ok && item_of(w) < a.items; ++w) {
        const FwdItem it(s, item_of(w));
        if (!mbar_wait(q_empty, (w & 1) ^ 1, abort_flag)) { ok = false; report(s.err, 71); break; }
        const int n_tiles = it.ja >= it.jb ? 0 : it.q0 + kT < s.Sq ? 2 : 1;
        mbar_expect_tx(q_full, n_tiles * L::kTile);
        for (int t = 0; t < n_tiles; ++t) load_tile<D>(sQ + t * L::kTile, &tm_q, it.q0 + t * kT, it.h, it.b, q_full);
        for (int m = 0; m < 2 * (it.jb - it.ja); ++m, ++n) {
          const int st = n % L::kStages;
          if (!mbar_wait(&kv_empty[st], (n / L::kStages & 1) ^ 1, abort_flag)) { ok = false; report(s.err, 71); break; }
          mbar_expect_tx(&kv_full[st], L::kTile);
          load_tile<D>(sKV + st * L::kTile, m & 1 ? &tm_v : &tm_k, (it.ja + (m >> 1)) * kT, it.kvh, it.b, &kv_full[st]);
        }
      }
      if (!ok) {
        mbar_wait_quiet(q_full, w & 1, 1 << 12);
        for (int i = n - L::kStages < 0 ? 0 : n - L::kStages; i < n; ++i)
          mbar_wait_quiet(&kv_full[i % L::kStages], i / L::kStages & 1, 1 << 12);
      }
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    // ---------------- products ----------------
    const uint32_t idesc_s = make_idesc_f16<T>(kT, kT), idesc_o = make_idesc_f16<T>(kT, D) | kBMajorMN;
    const uint64_t qd = make_desc_sw128(smem_u32(sQ)), kd = make_desc_sw128(smem_u32(sKV)), vd = make_desc_mn(smem_u32(sKV));
    auto slot = [&](int n) { return (uint64_t)(n % L::kStages * (L::kTile >> 4)); };
    auto wait_kv = [&](int n) { return warp_wait(&kv_full[n % L::kStages], n / L::kStages & 1, abort_flag); };
    auto free_kv = [&](int n) {
      if (elect_one()) umma_commit(&kv_empty[n % L::kStages]);
      __syncwarp();
    };
    bool ok = true;
    int n = 0, made[2] = {0, 0};                 // tiles of keys and values before this item; probabilities waited for
    int few_to = 0, last_b = -1;
    for (int w = 0; ok && item_of(w) < a.items; ++w) {
      FwdItem it(s, item_of(w));
      it.ja = uniform(it.ja);
      it.jb = uniform(it.jb);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        it.j0[t] = uniform(it.j0[t]);
        it.j1[t] = uniform(it.j1[t]);
      }
      if (it.b != last_b) {
        few_to = uniform(few_queries(s, it.b, lane));
        last_b = it.b;
      }
      const int q0 = uniform(it.q0);
      ok = warp_wait(q_full, w & 1, abort_flag);
      if (!ok) break;
      auto has = [&](int t, int j) { return j >= it.j0[t] && j < it.j1[t]; };
      auto scores = [&](int t, int nk) {
        if (elect_one()) {
          mma_rows<D>(tmem + t * kT, qd + t * (L::kTile >> 4), kd + slot(nk), idesc_s);
          umma_commit(&s_full[t]);
        }
        __syncwarp();
      };
      if (it.ja < it.jb) {
        ok = wait_kv(n);
        tcgen05_fence_after();
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (ok && has(t, it.ja)) scores(t, n);
        if (ok) free_kv(n);
      }
      for (int j = it.ja; j < it.jb && ok; ++j, n += 2) {
        ok = wait_kv(n + 1);
        if (ok && j + 1 < it.jb) ok = wait_kv(n + 2);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (ok && has(t, j)) ok = warp_wait(&p_full[t], made[t]++ & 1, abort_flag);
          if (!ok) break;
          if (has(t, j)) {
            tcgen05_fence_after();
            if (elect_one()) {
              mma_sum<16, 32>(tmem + 2 * kT + t * kT, tmem + t * kT, vd + slot(n + 1), idesc_o, j > it.j0[t]);
              if (q0 + t * kT < few_to) mma_sum<16, 32>(tmem + 2 * kT + t * kT, tmem + t * kT + 16, vd + slot(n + 1), idesc_o, true);
              umma_commit(&o_full[t]);
            }
            __syncwarp();
          }
          // over the probabilities that the product in front has read
          if (j + 1 < it.jb && has(t, j + 1)) scores(t, n + 2);
        }
        if (!ok) break;
        free_kv(n + 1);
        if (j + 1 < it.jb) free_kv(n + 2);
      }
    }
    if (!ok && lane == 0) report(s.err, 72);
    __syncwarp();
  } else {
    // ---------------- soft-max: two threads to a row, 64 columns each ----------------
    const int t = warp >> 3, hf = warp >> 2 & 1, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + t * kT, tO = tmem + lanes + 2 * kT + t * kT;
    uint64_t* x_bar = &x_full[t * 4 + (warp & 3)];
    float* xch = reinterpret_cast<float*>(smem + L::kXch) + t * 4 * kT;   // [2 turns][2 halves][128]
    uint8_t* stage = sQ + t * L::kTile + (warp & 7) * (L::kTile / 8);     // behind the tile's last scores
    const float c = s.scale_log2;
    bool ok = true;
    int made = 0, turns = 0;                       // scores and exchanges before this one
    int few_to = 0, last_b = -1;
    for (int w = 0; ok && item_of(w) < a.items; ++w) {
      const FwdItem item(s, item_of(w));
      const int first = t ? item.j0[1] : item.j0[0], n = (t ? item.j1[1] : item.j1[0]) - first;
      const int q = item.q0 + t * kT + r, b = item.b;
      if (b != last_b) few_to = few_queries(s, b, lane);
      last_b = b;
      const bool few = item.q0 + t * kT < few_to;
      int klo, khi;
      row_keys(s, q, klo, khi);
      float m = -INFINITY, l = 0.f;
      for (int it = 0; it < n; ++it, ++made, ++turns) {
        const int k0 = (first + it) * kT + hf * 64;
        if (!warp_wait(&s_full[t], made & 1, abort_flag)) { ok = false; break; }
        tcgen05_fence_after();
        uint32_t see[2] = {range_bits(klo, khi, k0), range_bits(klo, khi, k0 + 32)};
        if (s.mask != nullptr) {
          const uint32_t* words = s.mask + (int64_t)b * s.k_words + (k0 >> 5);
          see[0] &= __ldg(words);
          see[1] &= __ldg(words + 1);
        }
        // The scores are read twice, for the maximum and for the exponentials: 64 of them do not stay in registers beside the rest.
        const bool whole = __all_sync(0xffffffffu, (see[0] & see[1]) == 0xFFFFFFFFu);
        auto read = [&](int g, float (&v)[32]) {
          tmem_ld32(tS + hf * 64 + 32 * g, v);
          tmem_ld_wait(v);
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = see[g] >> i & 1 ? v[i] : -INFINITY;
          }
        };
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          float v[32];
          read(g, v);
          float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int i = 4; i < 28; i += 8)
#pragma unroll
            for (int u = 0; u < 4; ++u) mx[u] = max3(mx[u], v[i + u], v[i + u + 4]);
          top = max3(max3(top, v[28], v[29]), max3(mx[0], mx[1], v[30]), max3(mx[2], mx[3], v[31]));
        }
        // the other half's maximum
        float* turn = xch + (turns & 1) * 2 * kT;
        turn[hf * kT + r] = top;
        __syncwarp();
        if (lane == 0) mbar_arrive(x_bar);
        if (!warp_wait(x_bar, turns & 1, abort_flag)) { ok = false; break; }
        top = fmaxf(m, fmaxf(top, turn[(hf ^ 1) * kT + r]));
        // The reference moves only when it falls behind by a factor of 2^8: until then sums and products stay below 2^8 times
        // what they would be, far from the end of their range, and the outputs need not be read.
        const bool move = (top - m) * c > 8.f;
        if (__any_sync(0xffffffffu, move)) {
          const float f = move ? ex2((m - top) * c) : 1.f;
          l *= f;
          if (move) m = top;
          if (it > 0) {
            if (!warp_wait(&o_full[t], (made - 1) & 1, abort_flag)) { ok = false; break; }
            tcgen05_fence_after();
#pragma unroll
            for (int cc = 0; cc < D / 2; cc += 16) {
              float o[16];
              tmem_ld16(tO + hf * (D / 2) + cc, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= f;
              tmem_st16(tO + hf * (D / 2) + cc, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        const float mc = m == -INFINITY ? 0.f : -m * c;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          float v[32], sum[4] = {0.f, 0.f, 0.f, 0.f};
          read(g, v);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float &p0 = v[2 * i], &p1 = v[2 * i + 1];
            fma2(p0, p1, c, mc);
            p0 = ex2(p0);
            p1 = ex2(p1);
            add2(sum[2 * (i & 1)], sum[2 * (i & 1) + 1], p0, p1);
            pk[i] = pack2<T>(p0, p1);
          }
          tmem_st16(tS + hf * 64 + 32 * g, pk);          // over scores that have been read
          if (few) {
#pragma unroll
            for (int i = 0; i < 16; ++i) pk[i] = rest2<T>(pk[i], v[2 * i], v[2 * i + 1]);
            tmem_st16(tS + hf * 64 + 32 * g + 16, pk);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        hand_over(&p_full[t], lane);
      }
      if (ok && n > 0) {
        // the row's sum, and the last product
        float* turn = xch + (turns & 1) * 2 * kT;
        turn[hf * kT + r] = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(x_bar);
        ok = warp_wait(x_bar, turns & 1, abort_flag) && warp_wait(&o_full[t], (made - 1) & 1, abort_flag);
        tcgen05_fence_after();
        if (ok) l += turn[(hf ^ 1) * kT + r];
        ++turns;
      } else if (ok) {
        ok = warp_wait(q_full, w & 1, abort_flag);            // nothing is loaded: the stage is free
      }
      if (!ok) break;
      const float inv = l > 0.f ? 1.f / l : l == l ? 0.f : NAN;   // a row without keys: zeros
      if (a.nlse != nullptr && hf == 0 && item.q0 + t * kT < s.Sq) {
        const bool none = q >= s.Sq || m == -INFINITY;
        a.nlse[((int64_t)b * s.Hq + item.h) * s.q_pad + q] = none ? -INFINITY : shift_of<T>() - m * c - log2f(l);
      }
      const int row = item.q0 + t * kT + (warp & 3) * 32;
      if (row < s.Sq) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const int col = i * 64 + hf * 32;
          if (col >= s.D) break;
          float o[32];
          if (n > 0) {
            tmem_ld32(tO + col, o);
            tmem_ld_wait(o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          if (lane == 0) stores_read<0>();
          __syncwarp();
          stage32<T>(stage, o, inv, lane);
          if (lane == 0) store32(&tm_o, stage, col, row, item.h, b);
          if (a.nlse != nullptr) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float x = o[e] * inv;
              o[e] = x - to_float<T>(from_float<T>(x));
            }
            uint8_t* second = stage + (D == 128 ? 2048 : 0);
            if (lane == 0 && D != 128) stores_read<0>();
            __syncwarp();
            stage32<T>(second, o, kLowScale, lane);
            if (lane == 0) store32(&tm_low, second, col, row, item.h, b);
          }
        }
      }
      tcgen05_fence_before();
      if (lane == 0) {
        stores_read<0>();
        mbar_arrive(q_empty);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) report(s.err, 73);
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  finish(tmem, warp);
}

// ------------------------------------------------------------------------------------------------ before the backward pass
// Pieces of 16 bits whose weighted sum is x, in a row of eight numbers: each takes what those before it leave, the last below
// 2^-24 of x.  fp16's weights spread its pieces over numbers up to 65504 x 2^15, to 2^-45: a first piece x / 2^15 leaves at most
// 2^-12 |x| or 2^-10, and so on.  (Three pieces with weights of 2^8 and less end at 2^24, which dO_i . o_i passes where a loss is
// scaled; a column more costs nothing, the product takes sixteen anyway.)
template <typename T> struct Pieces;
template <> struct Pieces<__nv_bfloat16> {
  static constexpr int kN = 3;
  static __device__ float weight(int) { return 1.f; }
};
template <> struct Pieces<__half> {
  static constexpr int kN = 4;
  static __device__ float weight(int i) { return i == 0 ? 0x1p15f : i == 1 ? 0x1p4f : i == 2 ? 0x1p-8f : 0x1p-20f; }
};
template <typename T>
__device__ __forceinline__ uint4 in_pieces(float x) {
  __align__(16) T v[8];
#pragma unroll
  for (int i = 0; i < Pieces<T>::kN; ++i) {
    const float w = Pieces<T>::weight(i);
    v[i] = from_float<T>(x / w);
    x -= to_float<T>(v[i]) * w;
  }
#pragma unroll
  for (int i = Pieces<T>::kN; i < 8; ++i) v[i] = from_float<T>(0.f);
  return *reinterpret_cast<const uint4*>(v);
}

struct PrepArgs {
  const void* out;         // [B, Sq, Hq, D]
  const void* low;
  const void* grad;        // by strides
  const void* v;
  int64_t g_b, g_h, g_s, v_b, v_h, v_s;
  const float* nlse;       // [B, Hq, q_pad]
  float* delta;            // [B, Hq, q_pad]
  uint4* pieces;           // [B, Hq, q_pad / 128][2][128]: of -L / scale and of -delta; rows that see nothing: 0
  float inv_scale_log2;
  uint32_t* bound;         // [B, Hkv, 2] zeros, or null
  int B, Hq, Hkv, Sq, Skv, D, q_pad;
};

template <typename T>
__device__ __forceinline__ float dot8(const uint4& x, const uint4& y) {
  const T *a = reinterpret_cast<const T*>(&x), *b = reinterpret_cast<const T*>(&y);
  float d = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) d = fmaf(to_float<T>(a[i]), to_float<T>(b[i]), d);
  return d;
}

// delta_i = dO_i . o_i (and zeros behind Sq); in fp16 also the largest |dO_i|^2 and |v_j|^2 of each group of
// heads that share keys.  The maxima are of non-negative numbers, whose bits order like integers: any order gives the same.
//
// A CTA to 128 rows of a head, LANES lanes to a row (eight columns each), the rows of a group of lanes in flight four at a time.
// What a row gets is written by a lane of its own (in fp16 12.5 us instead of 15 for 2 x 1031 tokens in 32 heads of
// 80, where one lane loads -L / scale and cuts numbers into pieces for all rows of its group; in bf16 the same).  blockIdx.y counts
// the query heads, then (fp16) the key heads, whose rows only go into the bound.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) attn_prep_kernel(PrepArgs a) {
  constexpr int kRows = kT * LANES / 256;
  __shared__ uint32_t most[256 / LANES];
  const int sub = threadIdx.x % LANES, group = threadIdx.x / LANES, b = blockIdx.z;
  const bool is_q = (int)blockIdx.y < a.Hq, in = 8 * sub < a.D;
  const int h = is_q ? blockIdx.y : blockIdx.y - a.Hq, rows = is_q ? a.Sq : a.Skv, r0 = blockIdx.x * kT + group * kRows;
  const T* x = is_q ? (const T*)a.grad + b * a.g_b + h * a.g_h : (const T*)a.v + b * a.v_b + h * a.v_h;
  const int64_t stride = is_q ? a.g_s : a.v_s, o_row = (int64_t)a.Hq * a.D;
  const int64_t o_at = ((int64_t)b * a.Sq * a.Hq + h) * a.D + 8 * sub;
  if ((int)blockIdx.x * kT >= rows) return;
  const bool writes = is_q && sub < kRows;
  const int64_t row = ((int64_t)b * a.Hq + h) * a.q_pad + r0 + sub;
  const float nl = writes ? a.nlse[row] : 0.f;
  float largest = 0.f, delta = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; i += 4) {
    uint4 g[4], o[4], lo[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + i + u;
      g[u] = o[u] = lo[u] = make_uint4(0, 0, 0, 0);
      if (in && r < rows) {
        g[u] = ldg_nc_v4(x + r * stride + 8 * sub);
        if (is_q) {
          o[u] = ldg_nc_v4((const T*)a.out + o_at + r * o_row);
          lo[u] = ldg_nc_v4((const T*)a.low + o_at + r * o_row);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float d = is_q ? dot8<T>(g[u], o[u]) + dot8<T>(g[u], lo[u]) * (1.f / kLowScale) : 0.f;
      float n = std::is_same<T, __half>::value ? dot8<T>(g[u], g[u]) : 0.f;
#pragma unroll
      for (int s = LANES / 2; s > 0; s >>= 1) {
        d += __shfl_xor_sync(0xffffffffu, d, s);
        if (std::is_same<T, __half>::value) n += __shfl_xor_sync(0xffffffffu, n, s);
      }
      largest = fmaxf(largest, n);
      if (sub == i + u) delta = d;
    }
  }
  if (writes) {
    a.delta[row] = delta;
    uint4* at = a.pieces + row / kT * (2 * kT) + row % kT;
    at[0] = in_pieces<T>(nl == -INFINITY ? 0.f : nl * a.inv_scale_log2);
    at[kT] = in_pieces<T>(-delta);
  }
  if (std::is_same<T, __half>::value) {
    if (sub == 0) most[group] = __float_as_uint(largest);
    __syncthreads();
    if (threadIdx.x < 32) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, threadIdx.x < 256 / LANES ? most[threadIdx.x] : 0u);
      if (threadIdx.x == 0) atomicMax(&a.bound[(b * a.Hkv + (is_q ? h / (a.Hq / a.Hkv) : h)) * 2 + (is_q ? 0 : 1)], top);
    }
  }
}

// fp16: the power of two for dP - delta; bf16: none.  |dP_ij - delta_i| <= 2 max |dO_i| max |v_j| (o_i is a mean of the v_j).
template <typename T>
__device__ __forceinline__ float grad_factor(const uint32_t* bound, int group) {
  if constexpr (!std::is_same<T, __half>::value) return 1.f;
  const float n2 = 4.f * __uint_as_float(bound[2 * group]) * __uint_as_float(bound[2 * group + 1]);
  if (!(n2 > 0.f && n2 < INFINITY)) return 1.f;
  const int e = (int)floorf(15.f - 0.5f * log2f(n2) - kShiftF16);
  return exp2f((float)min(max(e, -100), 100));
}

struct BwdArgs {
  Shape s;
  const float* nlse;      // [B, Hq, q_pad]
  const float* delta;     // [B, Hq, q_pad]
  const uint4* pieces;
  const uint32_t* bound;  // [B, Hkv, 2] or null
  void *out0, *out1;      // dk and dv, or dq: [B, rows, heads, D]
  unsigned items;
};
// Zeros in rows [row, row + 128) of a head of [B, rows, heads, D], by the 512 threads of the arithmetic: what no query (or key) sees.
template <typename T>
__device__ __forceinline__ void zero_rows(void* out, int b, int row, int rows, int h, int heads, int D) {
  T* at = reinterpret_cast<T*>(out) + ((int64_t)b * rows * heads + h) * D;
  const int per = D / 8, n = min(kT, rows - row) * per;
  for (int i = threadIdx.x; i < n; i += 32 * kArith)
    *reinterpret_cast<uint4*>(at + (int64_t)(row + i / per) * heads * D + i % per * 8) = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------------------------------------ dk and dv
template <int D>
struct BwdSmem {
  static constexpr int kTile = kT * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kPieces = (2 + 2 * kStages) * kTile;     // of -L / scale, then of -delta, of the tiles' queries
  static constexpr int kWeights = kPieces + kStages * 4096;     // 16 columns of the pieces' weights, eight of them zeros
  static constexpr int kBars = kWeights + 4096;
  static constexpr int kSize = 1024 + kBars + 256;
};

// A block of keys [k0, k0 + 128), and the blocks of queries [i0, i0 + ni) of each head of its group that may see it.
struct DkvItem {
  int k0, kvh, b, i0, ni, total;
  __device__ __forceinline__ DkvItem(const Shape& s, unsigned i) {
    const unsigned rest = i / s.Hkv;
    kvh = (int)(i % s.Hkv);
    b = (int)(rest % s.B);
    k0 = (int)(rest / s.B) * kT;                 // the first keys are seen by most queries, and come first
    const int off = s.Skv - s.Sq;
    const int qlo = s.causal ? max(0, k0 - off) : 0;
    const int qhi = s.window > 0 ? (int)min((int64_t)s.Sq, (int64_t)min(k0 + kT, s.Skv) - 1 + s.window - off) : s.Sq;
    i0 = qlo / kT;
    ni = qhi > qlo ? (qhi + kT - 1) / kT - i0 : 0;
    total = ni * (s.Hq / s.Hkv);
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
attn_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_g,
                const __grid_constant__ CUtensorMap tm_dk, const __grid_constant__ CUtensorMap tm_dv,
                const __grid_constant__ BwdArgs a) {
  using L = BwdSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = smem + L::kTile;
  uint8_t* sQG = smem + 2 * L::kTile;            // tiles of q, and as many of dO
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* kv_full = bars;
  uint64_t* kv_empty = bars + 1;
  uint64_t* full = bars + 2;                     // [2][kStages]: q, dO
  uint64_t* empty = full + 2 * L::kStages;
  uint64_t* s_full = empty + 2 * L::kStages;
  uint64_t* p_full = s_full + 1;
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_full = s_full + 3;
  uint64_t* done = s_full + 4;
  uint64_t* staged = done + 1;                   // [2]: by the parity of the item
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(staged + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const Shape& s = a.s;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int group = s.Hq / s.Hkv, off = s.Skv - s.Sq;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(kv_empty, 1);
    mbar_init(&staged[0], kArith);
    mbar_init(&staged[1], kArith);
    for (int i = 0; i < 2 * L::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, kArith);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, kArith);
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < 256) {
    __align__(16) T w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = from_float<T>(threadIdx.x < kT && i < Pieces<T>::kN ? Pieces<T>::weight(i) : 0.f);
    reinterpret_cast<uint4*>(smem + L::kWeights)[threadIdx.x] = *reinterpret_cast<const uint4*>(w);
    fence_proxy_async_smem();
  }
  if (warp == kIssuer) tmem_alloc(tmem_slot, kTmemCols);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = uniform(*tmem_slot), tP = tmem + kT, tV = tmem + 2 * kT, tK = tmem + 3 * kT;

  if (warp == kLoader) {
    if (lane == 0) {
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_g);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
      // A tile of dO is free again half a step before the tile of q beside it: each has barriers of its own, and goes as its
      // turn comes.
      // An item's outputs are staged where its last step's tiles were: that place is taken again by the step kStages later, in the
      // next item or behind it.  In the place of k and v it kept the next item's from coming (4 x 512 tokens, 40 heads of 128: 61 us
      // instead of 52.5; dq, staged over q, 48.5 instead of 45).
      bool ok = true;
      int n = 0, z = 0, waited = 0;                // steps and items before this item; items whose staging has been waited for
      auto staged_before = [&](int item) {
        for (; ok && waited < item; ++waited) ok = mbar_wait(&staged[waited & 1], waited >> 1 & 1, abort_flag);
        if (!ok) report(s.err, 71);
      };
      for (int w = 0; ok && item_of(w) < a.items; ++w) {
        const DkvItem it(s, item_of(w));
        if (it.total == 0) continue;
        staged_before(z - 1);                      // so a barrier of these is never two items ahead
        if (!ok) break;
        if (!mbar_wait(kv_empty, (z & 1) ^ 1, abort_flag)) { ok = false; report(s.err, 71); break; }
        mbar_expect_tx(kv_full, 2 * L::kTile);
        load_tile<D>(sK, &tm_k, it.k0, it.kvh, it.b, kv_full);
        load_tile<D>(sV, &tm_v, it.k0, it.kvh, it.b, kv_full);
        for (int m = 0; m < 2 * it.total; ++m) {
          const int i = m >> 1, x = (m & 1) ^ (n + i == 0 ? 0 : 1), st = (n + i) % L::kStages, at = x * L::kStages + st;
          const int h = it.kvh * group + i / it.ni, q0 = (it.i0 + i % it.ni) * kT;
          if (i >= L::kStages - 1) staged_before(z);
          if (!ok) break;
          if (!mbar_wait(&empty[at], ((n + i) / L::kStages & 1) ^ 1, abort_flag)) { ok = false; report(s.err, 71); break; }
          mbar_expect_tx(&full[at], L::kTile + 2048);
          load_tile<D>(sQG + at * L::kTile, x ? &tm_g : &tm_q, q0, h, it.b, &full[at]);
          bulk_load(smem + L::kPieces + at * 2048, a.pieces + (((int64_t)it.b * s.Hq + h) * s.q_pad + q0) * 2 + x * kT, 2048,
                    &full[at]);
        }
        n += it.total;
        ++z;
      }
      if (!ok) {                                   // loads in flight end before the CTA does
        mbar_wait_quiet(kv_full, 0, 1 << 12);
        mbar_wait_quiet(kv_full, 1, 1 << 12);
        for (int i = 0; i < 2 * L::kStages; ++i) {
          mbar_wait_quiet(&full[i], 0, 1 << 12);
          mbar_wait_quiet(&full[i], 1, 1 << 12);
        }
      }
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    const uint32_t idesc_s = make_idesc_f16<T>(kT, kT), idesc_o = make_idesc_f16<T>(kT, D) | kBMajorMN;
    const uint64_t kd = make_desc_sw128(smem_u32(sK)), vd = make_desc_sw128(smem_u32(sV));
    const uint64_t qg_rows = make_desc_sw128(smem_u32(sQG)), qg_sum = make_desc_mn(smem_u32(sQG));
    const uint64_t weights = make_desc_rows16(smem_u32(smem + L::kWeights), 2048);
    const uint64_t pieces = make_desc_rows16(smem_u32(smem + L::kPieces), 0);   // their second eight columns: the first once more
    auto slot = [&](int n, int w) { return w * L::kStages + n % L::kStages; };
    auto tile = [&](int n, int w) { return (uint64_t)(slot(n, w) * (L::kTile >> 4)); };
    bool ok = true;
    int base = 0, z = 0, few_to = 0, last_b = -1;
    // Half of step n of an item's `total`, of q (W 0: k q^T, and P^T dO of the step before) or of dO (W 1: v dO^T, and dS^T q): the
    // sum, whose first operand lies where the new scores go, in front of these.
    auto half = [&](auto which, int n, int total, bool few) {
      constexpr int W = decltype(which)::value;
      const uint32_t tS = W ? tP : tmem, tO = W ? tK : tV;
      const int at = base + n;
      if (n > 0) {
        if (!warp_wait(W ? ds_full : p_full, (at - 1) & 1, abort_flag)) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          mma_sum<16, 32>(tO, tS, qg_sum + tile(at - 1, 1 - W), idesc_o, n > 1);
          if (few) mma_sum<16, 32>(tO, tS + 16, qg_sum + tile(at - 1, 1 - W), idesc_o, true);
          umma_commit(&empty[slot(at - 1, 1 - W)]);
        }
        __syncwarp();
      }
      if (n < total) {
        if (!warp_wait(&full[slot(at, W)], at / L::kStages & 1, abort_flag)) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          mma_rows<D>(tS, W ? vd : kd, qg_rows + tile(at, W), idesc_s);
          umma_f16(tS, weights, pieces + (slot(at, W) * 2048 >> 4), idesc_s, true);
          umma_commit(W ? dp_full : s_full);
          if (W && n + 1 == total) umma_commit(kv_empty);      // k and v have been read: the next item's come
        }
        __syncwarp();
      }
      return true;
    };
    for (int w = 0; ok && item_of(w) < a.items; ++w) {
      const DkvItem it(s, item_of(w));
      const int total = uniform(it.total), ni = uniform(it.ni);
      if (it.b != last_b) few_to = few_queries(s, it.b, lane);
      last_b = it.b;
      const int few_n = uniform(max(0, min(it.ni, few_to / kT + (few_to % kT != 0) - it.i0)));   // blocks of each head
      if (total == 0) continue;
      ok = warp_wait(kv_full, z++ & 1, abort_flag);
      for (int n = 0, i = -1; n <= total && ok; ++n, i = i + 1 < ni ? i + 1 : 0)         // i: the block of step n - 1
        ok = half(std::integral_constant<int, 0>(), n, total, i < few_n) &&
             half(std::integral_constant<int, 1>(), n, total, i < few_n);
      if (ok && elect_one()) umma_commit(done);
      __syncwarp();
      base += total;
    }
    if (!ok && lane == 0) report(s.err, 72);
    __syncwarp();
  } else {
    // ---------------- a key and a quarter of the queries to a thread ----------------
    const int qd = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t mine = (uint32_t)((warp & 3) * 32) << 16, lanes = mine + qd * 32;
    const float c = s.scale_log2;
    bool ok = true;
    int made = 0, items = 0, few_to = 0, last_b = -1;
    for (int w = 0; ok && item_of(w) < a.items; ++w) {
      const DkvItem it(s, item_of(w));
      if (it.b != last_b) few_to = few_queries(s, it.b, lane);
      last_b = it.b;
      if (it.total == 0) {
        zero_rows<T>(a.out0, it.b, it.k0, s.Skv, it.kvh, s.Hkv, s.D);
        zero_rows<T>(a.out1, it.b, it.k0, s.Skv, it.kvh, s.Hkv, s.D);
        continue;
      }
      const int k = it.k0 + r;
      const float f = grad_factor<T>(a.bound, it.b * s.Hkv + it.kvh);
      auto step = [&](auto few, int q0) {
        constexpr bool FEW = decltype(few)::value;
        const uint32_t par = made & 1;
        if (!warp_wait(s_full, par, abort_flag)) return false;
        tcgen05_fence_after();
        float p[32];
        tmem_ld32(tmem + lanes, p);
        // this key is seen by queries [lo, hi)
        const int lo = s.causal ? k - off - q0 : -kT;
        const int hi = s.window > 0 ? (int)min((int64_t)kT, (int64_t)k - off - q0 + s.window) : kT;
        const uint32_t see = range_bits(lo, hi, qd * 32);
        tmem_ld_wait(p);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          mul2(p[i], p[i + 1], c, c);
          p[i] = ex2(p[i]);
          p[i + 1] = ex2(p[i + 1]);
        }
        if (!__all_sync(0xffffffffu, see == 0xFFFFFFFFu)) {
#pragma unroll
          for (int i = 0; i < 32; ++i) p[i] = see >> i & 1 ? p[i] : 0.f;
        }
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = pack2<T>(p[2 * i], p[2 * i + 1]);
        tmem_st16(tmem + lanes, pk);
        if constexpr (FEW) {
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = rest2<T>(pk[i], p[2 * i], p[2 * i + 1]);
          tmem_st16(tmem + lanes + 16, pk);
        }
        hand_over(p_full, lane);
        if (!warp_wait(dp_full, par, abort_flag)) return false;
        tcgen05_fence_after();
#pragma unroll
        for (int g = 0; g < 2; ++g) {              // 16 at a time: the probabilities stay in registers
          float d[16];
          tmem_ld16(tP + lanes + 16 * g, d);
          tmem_ld_wait(d);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            mul2(d[2 * i], d[2 * i + 1], p[16 * g + 2 * i], p[16 * g + 2 * i + 1]);
            if constexpr (std::is_same<T, __half>::value) mul2(d[2 * i], d[2 * i + 1], f, f);
            pk[8 * g + i] = pack2<T>(d[2 * i], d[2 * i + 1]);
          }
          if constexpr (FEW) {                               // in the place of probabilities that have been used
#pragma unroll
            for (int i = 0; i < 8; ++i) p[8 * g + i] = __uint_as_float(rest2<T>(pk[8 * g + i], d[2 * i], d[2 * i + 1]));
          }
        }
        tmem_st16(tP + lanes, pk);
        if constexpr (FEW) tmem_st16(tP + lanes + 16, reinterpret_cast<const uint32_t*>(p));
        hand_over(ds_full, lane);
        return true;
      };
      for (int n = 0, i = 0; n < it.total && ok; ++n, ++made) {
        const int q0 = (it.i0 + i) * kT;
        i = i + 1 < it.ni ? i + 1 : 0;
        ok = q0 < few_to ? step(std::true_type(), q0) : step(std::false_type(), q0);
      }
      if (ok) ok = warp_wait(done, items & 1, abort_flag);
      tcgen05_fence_after();
      if (!ok) break;
      bool real = k < s.Skv;
      if (real && s.mask != nullptr) real = s.mask[(int64_t)it.b * s.k_words + (k >> 5)] >> (k & 31) & 1;
      const int row = it.k0 + (warp & 3) * 32;
      const float un = 1.f / scale_of<T>();
      const int slot = (made + L::kStages - 1) % L::kStages, mine_at = warp * (2 * L::kTile / kArith);
      uint8_t* stage = sQG + (mine_at / L::kTile * L::kStages + slot) * L::kTile + mine_at % L::kTile;
      if (row < s.Skv) {
        // 32 columns at a time: those of dv, then those of dk
#pragma unroll 1
        for (int i = 0; i < 2 * D / 128; ++i) {
          const int x = qd + 4 * i;
          const bool is_v = x < D / 32;
          const int col = x % (D / 32) * 32;
          float o[32];
          tmem_ld32((is_v ? tV : tK) + mine + col, o);
          tmem_ld_wait(o);
          if (!real) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          stage32<T>(stage + i * 2048, o, is_v ? un : s.scale * un / f, lane);
          if (lane == 0 && col < s.D) store32(is_v ? &tm_dv : &tm_dk, stage + i * 2048, col, row, it.kvh, it.b);
        }
      }
      tcgen05_fence_before();
      if (lane == 0) {
        stores_read<0>();
        mbar_arrive(&staged[items & 1]);
      }
      ++items;
      __syncwarp();
    }
    if (!ok && lane == 0) report(s.err, 73);
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  finish(tmem, warp);
}

// ------------------------------------------------------------------------------------------------ dq
template <int D>
struct DqSmem {
  static constexpr int kTile = kT * D * 2;
  static constexpr int kK = D == 128 ? 3 : 4, kV = D == 128 ? 2 : 4;     // tiles of k are kept for longer
  static constexpr int kBars = (2 + kK + kV) * kTile;
  static constexpr int kSize = 1024 + kBars + 256;
};

// A tile of queries [q0, q0 + 128) of a head, and the blocks of keys that it may see.
struct DqItem {
  int q0, h, b, kvh, j0, total;
  __device__ __forceinline__ DqItem(const Shape& s, unsigned i) {
    const unsigned rest = i / s.Hq;
    h = (int)(i % s.Hq);
    b = (int)(rest % s.B);
    q0 = ((s.Sq + kT - 1) / kT - 1 - (int)(rest / s.B)) * kT;
    kvh = h / (s.Hq / s.Hkv);
    int j1;
    key_blocks(s, q0, j0, j1);
    total = j1 - j0;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
attn_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_g,
               const __grid_constant__ CUtensorMap tm_dq, const __grid_constant__ BwdArgs a) {
  using L = DqSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sG = smem + L::kTile;
  uint8_t* sKV = smem + 2 * L::kTile;            // tiles of k, then of v
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* full = bars + 2;                     // [kK] and [kV]
  uint64_t* empty = full + L::kK + L::kV;
  uint64_t* s_full = empty + L::kK + L::kV;      // [2]
  uint64_t* s_free = s_full + 2;                 // [2]
  uint64_t* dp_full = s_full + 4;
  uint64_t* ds_full = s_full + 5;
  uint64_t* done = s_full + 6;
  uint64_t* staged = done + 1;                   // [2]: by the parity of the item
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(staged + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const Shape& s = a.s;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(&staged[0], kArith);
    mbar_init(&staged[1], kArith);
    for (int i = 0; i < L::kK + L::kV; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], kArith);
    }
    mbar_init(dp_full, 1);
    mbar_init(ds_full, kArith);
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kIssuer) tmem_alloc(tmem_slot, kTmemCols);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  // two tiles of scores in turn, dP (and dS over it), the sum
  const uint32_t tmem = uniform(*tmem_slot), tP = tmem + 2 * kT, tQ = tmem + 3 * kT;

  if (warp == kLoader) {
    if (lane == 0) {
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_g);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
      // outputs are staged where the last step's keys were, as in the other pass
      bool ok = true;
      int n = 0, z = 0, waited = 0;                // steps and items before this item; items whose staging has been waited for
      auto staged_before = [&](int item) {
        for (; ok && waited < item; ++waited) ok = mbar_wait(&staged[waited & 1], waited >> 1 & 1, abort_flag);
        if (!ok) report(s.err, 71);
      };
      for (int w = 0; ok && item_of(w) < a.items; ++w) {
        const DqItem it(s, item_of(w));
        if (it.total == 0) continue;
        staged_before(z - 1);
        if (!ok) break;
        if (!mbar_wait(q_empty, (z & 1) ^ 1, abort_flag)) { ok = false; report(s.err, 71); break; }
        mbar_expect_tx(q_full, 2 * L::kTile);
        load_tile<D>(sQ, &tm_q, it.q0, it.h, it.b, q_full);
        load_tile<D>(sG, &tm_g, it.q0, it.h, it.b, q_full);
        for (int m = 0; m < 2 * it.total; ++m) {
          const int i = n + (m >> 1), x = m & 1, of = x ? L::kV : L::kK, at = x * L::kK + i % of;
          if (x == 0 && (m >> 1) >= L::kK - 1) staged_before(z);
          if (!ok) break;
          if (!mbar_wait(&empty[at], (i / of & 1) ^ 1, abort_flag)) { ok = false; report(s.err, 71); break; }
          mbar_expect_tx(&full[at], L::kTile);
          load_tile<D>(sKV + at * L::kTile, x ? &tm_v : &tm_k, (it.j0 + (m >> 1)) * kT, it.kvh, it.b, &full[at]);
        }
        n += it.total;
        ++z;
      }
      if (!ok) {                                   // loads in flight end before the CTA does
        mbar_wait_quiet(q_full, 0, 1 << 12);
        mbar_wait_quiet(q_full, 1, 1 << 12);
        for (int i = 0; i < L::kK + L::kV; ++i) {
          mbar_wait_quiet(&full[i], 0, 1 << 12);
          mbar_wait_quiet(&full[i], 1, 1 << 12);
        }
      }
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    const uint32_t idesc_s = make_idesc_f16<T>(kT, kT), idesc_o = make_idesc_f16<T>(kT, D) | kBMajorMN;
    const uint64_t qd = make_desc_sw128(smem_u32(sQ)), gd = make_desc_sw128(smem_u32(sG));
    const uint64_t kv_rows = make_desc_sw128(smem_u32(sKV)), kv_sum = make_desc_mn(smem_u32(sKV));
    auto k_at = [&](int n) { return n % L::kK; };
    auto v_at = [&](int n) { return L::kK + n % L::kV; };
    bool ok = true;
    int base = 0, z = 0, few_to = 0, last_b = -1;
    for (int w = 0; ok && item_of(w) < a.items; ++w) {
      const DqItem it(s, item_of(w));
      const int total = uniform(it.total);
      if (it.b != last_b) few_to = few_queries(s, it.b, lane);
      last_b = it.b;
      const bool few = uniform(rest_of_dq(s) || it.q0 < few_to);
      if (total == 0) continue;
      ok = warp_wait(q_full, z++ & 1, abort_flag);
      const int end = base + total;
      auto scores = [&](int n) {                  // q k^T, into the other tile
        if (!warp_wait(&full[k_at(n)], n / L::kK & 1, abort_flag) || !warp_wait(&s_free[n & 1], (n >> 1 & 1) ^ 1, abort_flag))
          return false;
        tcgen05_fence_after();
        if (elect_one()) {
          mma_rows<D>(tmem + (n & 1) * kT, qd, kv_rows + (uint64_t)(k_at(n) * (L::kTile >> 4)), idesc_s);
          umma_commit(&s_full[n & 1]);
        }
        __syncwarp();
        return true;
      };
      auto grads = [&](int n) {                   // dO v^T
        if (!warp_wait(&full[v_at(n)], n / L::kV & 1, abort_flag)) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          mma_rows<D>(tP, gd, kv_rows + (uint64_t)(v_at(n) * (L::kTile >> 4)), idesc_s);
          umma_commit(dp_full);
          umma_commit(&empty[v_at(n)]);
          if (n + 1 == end) umma_commit(q_empty);          // behind all scores: the next item's q and dO come
        }
        __syncwarp();
        return true;
      };
      // What the arithmetic waits for goes first: dS of a step, its sum (dS lies over dP), the next dP.  Scores are two steps ahead.
      ok = scores(base) && grads(base) && (base + 1 == end || scores(base + 1));
      for (int n = base; n < end && ok; ++n) {
        ok = warp_wait(ds_full, n & 1, abort_flag);
        if (!ok) break;
        tcgen05_fence_after();
        if (elect_one()) {
          mma_sum<16, 32>(tQ, tP, kv_sum + (uint64_t)(k_at(n) * (L::kTile >> 4)), idesc_o, n > base);
          if (few) mma_sum<16, 32>(tQ, tP + 16, kv_sum + (uint64_t)(k_at(n) * (L::kTile >> 4)), idesc_o, true);
          umma_commit(&empty[k_at(n)]);
        }
        __syncwarp();
        if (n + 1 < end) ok = grads(n + 1);
        if (ok && n + 2 < end) ok = scores(n + 2);
      }
      if (ok && elect_one()) umma_commit(done);
      __syncwarp();
      base = end;
    }
    if (!ok && lane == 0) report(s.err, 72);
    __syncwarp();
  } else {
    // ---------------- a quarter of a query's keys to a thread ----------------
    const int qd = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t mine = (uint32_t)((warp & 3) * 32) << 16, lanes = mine + qd * 32;
    const float c = s.scale_log2;
    bool ok = true;
    int made = 0, items = 0, few_to = 0, last_b = -1;
    for (int w = 0; ok && item_of(w) < a.items; ++w) {
      const DqItem it(s, item_of(w));
      if (it.b != last_b) few_to = few_queries(s, it.b, lane);
      last_b = it.b;
      const bool few = rest_of_dq(s) || it.q0 < few_to;
      if (it.total == 0) {
        zero_rows<T>(a.out0, it.b, it.q0, s.Sq, it.h, s.Hq, s.D);
        continue;
      }
      const int q = it.q0 + r;
      int klo, khi;
      row_keys(s, q, klo, khi);
      const float f = grad_factor<T>(a.bound, it.b * s.Hkv + it.kvh);
      const int64_t at = ((int64_t)it.b * s.Hq + it.h) * s.q_pad + q;
      const float nl = a.nlse[at], dl = a.delta[at] * -f;
      for (int n = 0; n < it.total; ++n, ++made) {
        const int kb = (it.j0 + n) * kT + qd * 32;
        if (!warp_wait(&s_full[made & 1], made >> 1 & 1, abort_flag)) { ok = false; break; }
        tcgen05_fence_after();
        float p[32];
        tmem_ld32(tmem + lanes + (made & 1) * kT, p);
        uint32_t see = range_bits(klo, khi, kb);
        if (s.mask != nullptr) see &= __ldg(s.mask + (int64_t)it.b * s.k_words + (kb >> 5));
        tmem_ld_wait(p);
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[made & 1]);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          fma2(p[i], p[i + 1], c, nl);
          p[i] = ex2(p[i]);
          p[i + 1] = ex2(p[i + 1]);
        }
        if (!__all_sync(0xffffffffu, see == 0xFFFFFFFFu)) {
#pragma unroll
          for (int i = 0; i < 32; ++i) p[i] = see >> i & 1 ? p[i] : 0.f;
        }
        if (!warp_wait(dp_full, made & 1, abort_flag)) { ok = false; break; }
        tcgen05_fence_after();
        float d[32];
        tmem_ld32(tP + lanes, d);
        tmem_ld_wait(d);
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          fma2(d[2 * i], d[2 * i + 1], f, dl);
          mul2(d[2 * i], d[2 * i + 1], p[2 * i], p[2 * i + 1]);
          pk[i] = pack2<T>(d[2 * i], d[2 * i + 1]);
        }
        tmem_st16(tP + lanes, pk);
        if (few) {
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = rest2<T>(pk[i], d[2 * i], d[2 * i + 1]);
          tmem_st16(tP + lanes + 16, pk);
        }
        hand_over(ds_full, lane);
      }
      if (ok) ok = warp_wait(done, items & 1, abort_flag);
      tcgen05_fence_after();
      if (!ok) break;
      const int row = it.q0 + (warp & 3) * 32;
      uint8_t* stage = sKV + (made + L::kK - 1) % L::kK * L::kTile + (qd % (D / 32) * 4 + (warp & 3)) * 2048;
      if (qd < D / 32 && qd * 32 < s.D && row < s.Sq) {
        float o[32];
        tmem_ld32(tQ + mine + qd * 32, o);
        tmem_ld_wait(o);
        stage32<T>(stage, o, s.scale / (scale_of<T>() * f), lane);
        if (lane == 0) store32(&tm_dq, stage, qd * 32, row, it.h, it.b);
      }
      tcgen05_fence_before();
      if (lane == 0) {
        stores_read<0>();
        mbar_arrive(&staged[items & 1]);
      }
      ++items;
      __syncwarp();
    }
    if (!ok && lane == 0) report(s.err, 73);
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  finish(tmem, warp);
}

// ------------------------------------------------------------------------------------------------ hidden keys
// The mask of keys as bits, and keys and values with zeros in hidden rows, so that what those hold (infinities, NaN) takes no
// part in products where they are summed over.
struct HideArgs {
  const uint8_t* mask;     // [B, Skv] by strides
  int64_t m_b, m_s;
  const void *k, *v;
  int64_t k_b, k_h, k_s, v_b, v_h, v_s;
  uint4 *ko, *vo;          // [B, Skv, Hkv, D]
  uint32_t* words;         // [B, k_words]
  int Hkv, Skv, D, k_words;
};

__global__ void __launch_bounds__(256) attn_hide_kernel(HideArgs a) {
  __shared__ uint32_t word;
  const int b = blockIdx.z, s0 = blockIdx.x * 32, tid = threadIdx.x;
  if (tid < 32) {
    const bool real = s0 + tid < a.Skv && a.mask[b * a.m_b + (s0 + tid) * a.m_s] != 0;
    const uint32_t w = __ballot_sync(0xffffffffu, real);
    if (tid == 0) {
      word = w;
      if (blockIdx.y == 0) a.words[(int64_t)b * a.k_words + blockIdx.x] = w;
    }
  }
  __syncthreads();
  const uint32_t w = word;
  const int per = a.D / 8, row = a.Hkv * per, n = min(32, a.Skv - s0) * row;
  for (int i = blockIdx.y * 256 + tid; i < n; i += 256 * gridDim.y) {
    const int sl = i / row, h = i % row / per, c = i % per * 8;
    const bool real = w >> sl & 1;
    const int64_t at = ((int64_t)b * a.Skv + s0) * row + i;
    const uint16_t* k = reinterpret_cast<const uint16_t*>(a.k) + b * a.k_b + h * a.k_h + (int64_t)(s0 + sl) * a.k_s + c;
    const uint16_t* v = reinterpret_cast<const uint16_t*>(a.v) + b * a.v_b + h * a.v_h + (int64_t)(s0 + sl) * a.v_s + c;
    a.ko[at] = real ? *reinterpret_cast<const uint4*>(k) : make_uint4(0, 0, 0, 0);
    a.vo[at] = real ? *reinterpret_cast<const uint4*>(v) : make_uint4(0, 0, 0, 0);
  }
}

// ------------------------------------------------------------------------------------------------ host
// [sequences, heads, rows, D] by strides in elements: rows of D (a multiple of 8) elements.
struct Tensor4 {
  const void* p;
  int64_t b, h, s;
};

bool encode(CUtensorMap* tm, CUtensorMapDataType dt, const Tensor4& t, int D, int rows, int heads, int B, bool store = false) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  // strides of dimensions of size 1 are never taken, but have to be multiples of 16 bytes
  const int64_t s = rows > 1 ? t.s : D, h = heads > 1 ? t.h : D, b = B > 1 ? t.b : D;
  if ((reinterpret_cast<uintptr_t>(t.p) & 15) || t.p == nullptr || s <= 0 || h <= 0 || b <= 0 || ((s | h | b) & 7)) return false;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)B};
  cuuint64_t strides[3] = {(cuuint64_t)s * 2, (cuuint64_t)h * 2, (cuuint64_t)b * 2};
  cuuint32_t box[4] = {store ? 32u : 64u, store ? 32u : (cuuint32_t)kT, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(tm, dt, 4, const_cast<void*>(t.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             store ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// A contiguous [B, rows, heads, D], written by tiles of 32 x 32.
bool encode_out(CUtensorMap* tm, CUtensorMapDataType dt, void* p, int D, int rows, int heads, int B) {
  return encode(tm, dt, {p, (int64_t)rows * heads * D, D, (int64_t)heads * D}, D, rows, heads, B, true);
}

int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) != 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}
// Tiles of work of 128 (or 256) rows: their number, 0 where it is past what a CTA counts.
unsigned items_of(const Shape& s, int heads, int rows, int of) {
  const int64_t n = (int64_t)heads * ((rows + of - 1) / of) * s.B;
  return n < (1ll << 30) ? (unsigned)n : 0;
}
unsigned grid_of(unsigned items) {
  const unsigned n = (unsigned)sm_count();
  return items < n ? items : n;
}

// The driver's encoder wants a current context, which a thread that has launched nothing yet (autograd's) need not have.
bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

bool shape_ok(int B, int Hq, int Hkv, int Sq, int Skv, int D, int window, float scale) {
  return B >= 1 && B <= 65535 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hq <= (1 << 20) && Sq >= 1 && Skv >= 1 &&
         Sq <= (1 << 23) && Skv <= (1 << 23) && D >= 8 && D <= 128 && D % 8 == 0 && window >= 0 && scale >= 1e-4f && scale <= 1e4f;
}

Shape make_shape(int B, int Hq, int Hkv, int Sq, int Skv, int D, int causal, int window, const uint32_t* mask, float scale,
                 int* err) {
  Shape s;
  s.B = B; s.Hq = Hq; s.Hkv = Hkv; s.Sq = Sq; s.Skv = Skv; s.D = D; s.causal = causal;
  s.window = window < Skv ? window : 0;      // one of all keys hides none, and limits stay in 32 bits
  s.q_pad = (Sq + kT - 1) / kT * kT;
  s.k_words = (Skv + kT - 1) / kT * (kT / 32);
  s.mask = mask; s.scale = scale; s.scale_log2 = scale * 1.4426950408889634f; s.err = err;
  return s;
}

template <typename T> constexpr CUtensorMapDataType map_type() {
  return std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// One CTA to an SM whatever the tiles take: each allocates all of the tensor memory.
constexpr int one_cta(int bytes) { return bytes > 120 * 1024 ? bytes : 120 * 1024; }

template <typename T, int D>
int run_fwd(const Shape& s, const Tensor4& q, const Tensor4& k, const Tensor4& v, void* out, void* low, float* nlse,
            cudaStream_t stream) {
  CUtensorMap tq, tk, tv, to, tl;
  const CUtensorMapDataType dt = map_type<T>();
  if (!bind_context() || !encode(&tq, dt, q, s.D, s.Sq, s.Hq, s.B) || !encode(&tk, dt, k, s.D, s.Skv, s.Hkv, s.B) ||
      !encode(&tv, dt, v, s.D, s.Skv, s.Hkv, s.B) || !encode_out(&to, dt, out, s.D, s.Sq, s.Hq, s.B) ||
      (nlse != nullptr && !encode_out(&tl, dt, low, s.D, s.Sq, s.Hq, s.B)))
    return (int)cudaErrorInvalidValue;
  if (nlse == nullptr) tl = to;                    // not used
  constexpr int smem = one_cta(FwdSmem<D>::kSize);
  static SmemLimit limit;
  const cudaError_t e = limit((const void*)attn_fwd_kernel<T, D>, smem);
  if (e != cudaSuccess) return (int)e;
  const FwdArgs a = {s, nlse, items_of(s, s.Hq, s.Sq, 2 * kT)};
  if (a.items == 0) return (int)cudaErrorInvalidValue;
  attn_fwd_kernel<T, D><<<grid_of(a.items), kThreads, smem, stream>>>(tq, tk, tv, to, tl, a);
  return (int)cudaGetLastError();
}

template <typename T, int D>
int run_bwd(const Shape& s, const Tensor4& q, const Tensor4& k, const Tensor4& v, const Tensor4& g, const void* out,
            const void* low, const float* nlse, float* work, void* dq, void* dk, void* dv, cudaStream_t stream) {
  CUtensorMap tq, tk, tv, tg, tdq, tdk, tdv;
  const CUtensorMapDataType dt = map_type<T>();
  if (!bind_context() || !encode(&tq, dt, q, s.D, s.Sq, s.Hq, s.B) || !encode(&tk, dt, k, s.D, s.Skv, s.Hkv, s.B) ||
      !encode(&tv, dt, v, s.D, s.Skv, s.Hkv, s.B) || !encode(&tg, dt, g, s.D, s.Sq, s.Hq, s.B) ||
      !encode_out(&tdq, dt, dq, s.D, s.Sq, s.Hq, s.B) || !encode_out(&tdk, dt, dk, s.D, s.Skv, s.Hkv, s.B) ||
      !encode_out(&tdv, dt, dv, s.D, s.Skv, s.Hkv, s.B))
    return (int)cudaErrorInvalidValue;
  constexpr int smem = one_cta(BwdSmem<D>::kSize), smem_q = one_cta(DqSmem<D>::kSize);
  static SmemLimit limit_kv, limit_q;
  cudaError_t e = limit_kv((const void*)attn_dkv_kernel<T, D>, smem);
  if (e == cudaSuccess) e = limit_q((const void*)attn_dq_kernel<T, D>, smem_q);
  if (e != cudaSuccess) return (int)e;
  uint4* pieces = reinterpret_cast<uint4*>(work);
  float* delta = work + (int64_t)s.B * s.Hq * s.q_pad * 8;
  uint32_t* bound = nullptr;
  if (std::is_same<T, __half>::value) {
    bound = reinterpret_cast<uint32_t*>(work + (int64_t)s.B * s.Hq * s.q_pad * 9);
    e = cudaMemsetAsync(bound, 0, (size_t)s.B * s.Hkv * 8, stream);
    if (e != cudaSuccess) return (int)e;
  }
  const PrepArgs p = {out, low, g.p, v.p, g.b, g.h, g.s, v.b, v.h, v.s, nlse, delta, pieces, 1.f / s.scale_log2, bound,
                      s.B, s.Hq, s.Hkv, s.Sq, s.Skv, s.D, s.q_pad};
  if (items_of(s, s.Hkv, s.Skv, kT) == 0 || items_of(s, s.Hq, s.Sq, kT) == 0 || s.Hq + s.Hkv > 65535)
    return (int)cudaErrorInvalidValue;
  const int longest = bound != nullptr && s.Skv > s.Sq ? s.Skv : s.Sq;
  const dim3 prep_grid((longest + kT - 1) / kT, s.Hq + (bound != nullptr ? s.Hkv : 0), s.B);
  attn_prep_kernel<T, D / 8><<<prep_grid, 256, 0, stream>>>(p);
  BwdArgs a = {s, nlse, delta, pieces, bound, dk, dv, items_of(s, s.Hkv, s.Skv, kT)};
  attn_dkv_kernel<T, D><<<grid_of(a.items), kThreads, smem, stream>>>(tq, tk, tv, tg, tdk, tdv, a);
  a.items = items_of(s, s.Hq, s.Sq, kT);
  a.out0 = dq;
  attn_dq_kernel<T, D><<<grid_of(a.items), kThreads, smem_q, stream>>>(tq, tk, tv, tg, tdq, a);
  return (int)cudaGetLastError();
}

}  // namespace

// q [B, Hq, Sq, D], k and v [B, Hkv, Skv, D] by the strides of sequences, heads and rows (elements; multiples of 8, rows
// contiguous, pointers 16-byte aligned), fp16 or bf16, D a multiple of 8 up to 128.  window > 0 needs causal.  mask_words: the
// real keys' bits [B, ceil(Skv / 128) * 4] or null (ipex_attn_hide writes them).  out [B, Sq, Hq, D] contiguous; low, the same
// shape, and nlse [B, Hq, Sq
// rounded up to 128] (16-byte aligned) for the backward pass, or null.  Returns a cudaError_t.
IPEX_API int ipex_attn_train_fwd(const void* q, int64_t q_b, int64_t q_h, int64_t q_s, const void* k, int64_t k_b, int64_t k_h,
                                 int64_t k_s, const void* v, int64_t v_b, int64_t v_h, int64_t v_s, const uint32_t* mask_words,
                                 void* out, void* low, float* nlse, int B, int Hq, int Hkv, int Sq, int Skv, int D, int causal,
                                 int window, float scale, int dtype, int* err, void* stream) {
  if (!shape_ok(B, Hq, Hkv, Sq, Skv, D, window, scale) || (window > 0 && !causal) || out == nullptr ||
      (nlse != nullptr && low == nullptr) ||
      ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(low) | reinterpret_cast<uintptr_t>(nlse)) & 15))
    return (int)cudaErrorInvalidValue;
  const Shape s = make_shape(B, Hq, Hkv, Sq, Skv, D, causal, window, mask_words, scale, err);
  const Tensor4 tq = {q, q_b, q_h, q_s}, tk = {k, k_b, k_h, k_s}, tv = {v, v_b, v_h, v_s};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == DT_F16)
    return D <= 64 ? run_fwd<__half, 64>(s, tq, tk, tv, out, low, nlse, st) : run_fwd<__half, 128>(s, tq, tk, tv, out, low, nlse, st);
  if (dtype == DT_BF16)
    return D <= 64 ? run_fwd<__nv_bfloat16, 64>(s, tq, tk, tv, out, low, nlse, st)
                   : run_fwd<__nv_bfloat16, 128>(s, tq, tk, tv, out, low, nlse, st);
  return (int)cudaErrorInvalidValue;
}

// g: the gradient of out, by strides like q.  work: scratch, 16-byte aligned, 9 floats for each of nlse and 2 B Hkv.
// dq [B, Sq, Hq, D], dk and dv [B, Skv, Hkv, D] contiguous.
IPEX_API int ipex_attn_train_bwd(const void* q, int64_t q_b, int64_t q_h, int64_t q_s, const void* k, int64_t k_b, int64_t k_h,
                                 int64_t k_s, const void* v, int64_t v_b, int64_t v_h, int64_t v_s, const uint32_t* mask_words,
                                 const void* out, const void* low, const float* nlse, const void* g, int64_t g_b, int64_t g_h,
                                 int64_t g_s, float* work, void* dq, void* dk, void* dv, int B, int Hq, int Hkv, int Sq,
                                 int Skv, int D, int causal, int window, float scale, int dtype, int* err, void* stream) {
  if (!shape_ok(B, Hq, Hkv, Sq, Skv, D, window, scale) || (window > 0 && !causal) || out == nullptr || low == nullptr ||
      nlse == nullptr || work == nullptr || dq == nullptr || dk == nullptr || dv == nullptr ||
      ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(low) | reinterpret_cast<uintptr_t>(nlse) |
        reinterpret_cast<uintptr_t>(work) |
        reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv)) & 15))
    return (int)cudaErrorInvalidValue;
  const Shape s = make_shape(B, Hq, Hkv, Sq, Skv, D, causal, window, mask_words, scale, err);
  const Tensor4 tq = {q, q_b, q_h, q_s}, tk = {k, k_b, k_h, k_s}, tv = {v, v_b, v_h, v_s}, tg = {g, g_b, g_h, g_s};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == DT_F16)
    return D <= 64 ? run_bwd<__half, 64>(s, tq, tk, tv, tg, out, low, nlse, work, dq, dk, dv, st)
                   : run_bwd<__half, 128>(s, tq, tk, tv, tg, out, low, nlse, work, dq, dk, dv, st);
  if (dtype == DT_BF16)
    return D <= 64 ? run_bwd<__nv_bfloat16, 64>(s, tq, tk, tv, tg, out, low, nlse, work, dq, dk, dv, st)
                   : run_bwd<__nv_bfloat16, 128>(s, tq, tk, tv, tg, out, low, nlse, work, dq, dk, dv, st);
  return (int)cudaErrorInvalidValue;
}

// mask [B, Skv] of bytes by strides (0: hidden); k, v by strides as above; k_out, v_out [B, Skv, Hkv, D] contiguous, words [B,
// ceil(Skv / 128) * 4].
IPEX_API int ipex_attn_hide(const uint8_t* mask, int64_t m_b, int64_t m_s, const void* k, int64_t k_b, int64_t k_h, int64_t k_s,
                            const void* v, int64_t v_b, int64_t v_h, int64_t v_s, void* k_out, void* v_out, uint32_t* words, int B,
                            int Hkv, int Skv, int D, void* stream) {
  if (B < 1 || B > 65535 || Hkv < 1 || Skv < 1 || Skv > (1 << 23) || D < 8 || D > 128 || D % 8 ||
      mask == nullptr || k == nullptr || v == nullptr || k_out == nullptr || v_out == nullptr || words == nullptr ||
      ((k_b | k_h | k_s | v_b | v_h | v_s) & 7) ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_out) |
        reinterpret_cast<uintptr_t>(v_out)) & 15))
    return (int)cudaErrorInvalidValue;
  HideArgs a = {mask, m_b, m_s, k, v, k_b, k_h, k_s, v_b, v_h, v_s, (uint4*)k_out, (uint4*)v_out, words, Hkv, Skv, D,
                (Skv + kT - 1) / kT * (kT / 32)};
  // two vectors of k and of v to a thread
  const int shares = (32 * Hkv * (D / 8) + 511) / 512;
  attn_hide_kernel<<<dim3(a.k_words, shares < 65535 ? shares : 65535, B), 256, 0, (cudaStream_t)stream>>>(a);
  return (int)cudaGetLastError();
}
