// Shared pieces of the attention kernels (fl_attn.cu, fl_attn_bwd.cu).
//
// Row i of a sequence sees the keys begin[i] <= j < end[i].  Scores:
//   x_ij = scale q_i . k_j,  [cap tanh(x / cap)],  [- slope_h |i + Sk - Sq - j|]
// and o_i = sum_j softmax(x_i)_j v_j over the seen keys (0 for a row that sees
// none).  Query heads share key/value heads in groups of Hq / Hkv.
//
// Packed rows: where a group's size is a power of two, a tile's rows are the
// group's heads of consecutive tokens (row r = token r >> lgp, head r & (pg - 1)),
// so a key/value tile is read once for the whole group and a few tokens still
// fill a tile.
#pragma once
#include <cuda_bf16.h>
#include <cstdint>

#include "fl_host.h"
#include "fl_ptx.cuh"

namespace fl {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTile = 128;        // rows or keys of a tile
constexpr int kNone = 0x7fffffff;

struct Shape {
  int B, Sq, Sk, Hq, Hkv, D;
  int lgp;       // log2 of the packed heads pg
  int groups;    // Hq / Hkv / pg
  float scale;   // of q . k
  float sl2;     // scale * log2(e)
  float cap2;    // cap * log2(e), 0 = no cap
  float icap2;   // 2 log2(e) scale / cap: tanh's argument as a power of two
  const int* begin;
  const int* end;
  const float* slopes;  // [Hq] or null
};

// What the rows of a tile see: {min begin, max end} over its rows that see
// anything, {max begin, min end} over all its rows inside the sequence (a row
// that sees nothing makes those impossible to cover).
struct Range {
  int min_lo, max_hi, max_lo, min_hi;
};

__device__ __forceinline__ void row_range(const Shape& s, int b, int tok, int& lo, int& hi) {
  const int64_t i = static_cast<int64_t>(b) * s.Sq + tok;
  lo = max(s.begin[i], 0);
  hi = min(s.end[i], s.Sk);
  if (lo >= hi) lo = hi = 0;
}

// Range of the tokens [t0, t0 + n): one warp, every lane gets the result.
__device__ __forceinline__ Range tile_range(const Shape& s, int b, int t0, int n) {
  Range r{kNone, 0, 0, kNone};
  for (int i = threadIdx.x & 31; i < n; i += 32) {
    if (t0 + i >= s.Sq) break;
    int lo, hi;
    row_range(s, b, t0 + i, lo, hi);
    if (lo < hi) {
      r.min_lo = min(r.min_lo, lo);
      r.max_hi = max(r.max_hi, hi);
      r.max_lo = max(r.max_lo, lo);
      r.min_hi = min(r.min_hi, hi);
    } else {
      r.max_lo = kNone;
      r.min_hi = 0;
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    r.min_lo = min(r.min_lo, __shfl_xor_sync(0xffffffffu, r.min_lo, o));
    r.max_hi = max(r.max_hi, __shfl_xor_sync(0xffffffffu, r.max_hi, o));
    r.max_lo = max(r.max_lo, __shfl_xor_sync(0xffffffffu, r.max_lo, o));
    r.min_hi = min(r.min_hi, __shfl_xor_sync(0xffffffffu, r.min_hi, o));
  }
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x of two values without the special-function unit, whose 16 results a
// cycle and SM bound the exponentials: x = i + f with i the nearest integer
// (by adding 1.5 * 2^23), 2^f on [-1/2, 1/2] by the polynomial of degree 5 with
// value 1 at 0 whose largest relative error is smallest (1.1e-7; 1.7e-7 with these
// steps in FP32: less than the special-function unit's 2^-22), times 2^i, whose
// bits are made from those of i.  x under -126.5 gives 0; a product and not an
// addition to the exponent's bits, so that NaN stays NaN.
__device__ __forceinline__ void ex2_pair(float x0, float x1, float& y0, float& y1) {
  const float round = 12582912.0f;
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x0) : "f"(-127.0f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x1) : "f"(-127.0f));
  const uint64_t x = pair(x0, x1);
  const uint64_t i = add2(x, pair(round, round));
  const uint64_t f = fma2(add2(i, pair(-round, -round)), pair(-1.0f, -1.0f), x);
  uint64_t p = fma2(f, pair(0.001326472731307149f, 0.001326472731307149f),
                    pair(0.009671512991189957f, 0.009671512991189957f));
  p = fma2(f, p, pair(0.05550733581185341f, 0.05550733581185341f));
  p = fma2(f, p, pair(0.24022242426872253f, 0.24022242426872253f));
  p = fma2(f, p, pair(0.6931470036506653f, 0.6931470036506653f));
  p = fma2(f, p, pair(1.0f, 1.0f));
  float i0, i1;
  unpair(i, i0, i1);
  i0 = __int_as_float((__float_as_int(i0) << 23) + 0x3F800000);
  i1 = __int_as_float((__float_as_int(i1) << 23) + 0x3F800000);
  unpair(mul2(p, pair(i0, i1)), y0, y1);
}

// What is done to a score before the softmax.
enum Mode : int { kPlain = 0, kSlopes = 1, kCapped = 2, kCappedSlopes = 3 };
__host__ __device__ constexpr bool has_cap(int mode) { return mode >= kCapped; }
__host__ __device__ constexpr bool has_slopes(int mode) { return mode == kSlopes || mode == kCappedSlopes; }

// The cap, from u = 2^(2 y log2 e) and r = 1 / (1 + u): tanh(y) = 1 - 2 r with an
// absolute error of a few 1e-7 everywhere, which the cap multiplies (the hardware's
// tanh would leave 2^-11 of the cap); its derivative is 1 - tanh^2(y) = 4 r (u r),
// to a few 1e-6 of itself on either side (1 - r would leave nothing of it where r
// is near 1).  2 y log2 e of two scores, and r of it:
__device__ __forceinline__ uint64_t cap_arg2(const Shape& s, uint64_t qk) {
  return mul2(qk, pair(s.icap2, s.icap2));
}
__device__ __forceinline__ uint64_t cap_u2(uint64_t arg) {
  float y0, y1;
  unpair(arg, y0, y1);
  return pair(ex2(y0), ex2(y1));
}
__device__ __forceinline__ uint64_t cap_r2(uint64_t u) {
  float y0, y1;
  unpair(add2(u, pair(1.0f, 1.0f)), y0, y1);
  return pair(rcp(y0), rcp(y1));
}
// cap log2(e) tanh + add:
__device__ __forceinline__ uint64_t capped2(const Shape& s, uint64_t r, uint64_t add) {
  return fma2(r, pair(-2.0f * s.cap2, -2.0f * s.cap2), add);   // add: with cap2 in it
}
// The derivative times 2^15: between the two places that use it it is held in fp16,
// whose 11 bits then reach down to 2^-29 (scores of 10.7 caps; at 1 they would end at
// 2^-14, 5.5 caps); dp - delta is formed over 2^15 for it.
constexpr float kCapSlope = 32768.0f;
// u of an argument for it: finite, so that r is not 0 and u r is 1 at the far end.
__device__ __forceinline__ uint64_t cap_u2_finite(uint64_t arg) {
  float y0, y1;
  unpair(arg, y0, y1);
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(y0) : "f"(126.0f));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(y1) : "f"(126.0f));
  return pair(ex2(y0), ex2(y1));
}
__device__ __forceinline__ uint64_t cap_slope2(uint64_t r, uint64_t u) {
  return mul2(mul2(r, pair(4.0f * kCapSlope, 4.0f * kCapSlope)), mul2(u, r));
}

// A small non-negative integer as a float without the conversion unit (which
// is the special-function unit).
__device__ __forceinline__ float small_float(int v) { return __int_as_float(0x4B000000 | v) - 8388608.0f; }

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// The lane that issues for a warp: always the same one.
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// The descriptors' address field counts 16-byte units and a tile does not wrap
// it, so a step is an addition: the issuing thread shares its scheduler with
// element warps and has few slots between two products.
//
// D[128 x kRows] = A . B^T, both K-major in shared memory: A 128 rows, B kRows,
// each as HD / 64 chunks of rows of 128 bytes; a and b from sdesc_kmajor_sw128.
template <int HD, int kRows>
__device__ __forceinline__ void mma_rows(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk)
    mma_ss(d, a + (kk / 4) * (kTile * 128 >> 4) + 2 * (kk % 4), b + (kk / 4) * (kRows * 128 >> 4) + 2 * (kk % 4), idesc,
           kk != 0);
}

// D[128 x HD] (+)= A . B: A bf16 [128 x kRows] in TMEM; B [kRows x HD] in shared
// memory (the same chunks, read with the columns as the MN side), b from
// cols_desc<kRows>.
template <int kRows>
__device__ __forceinline__ uint64_t cols_desc(uint32_t addr) {
  return sdesc_mnmajor_sw128(addr, kRows * 128, 1024);
}
template <int HD, int kRows>
__device__ __forceinline__ void mma_cols(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < kRows / 16; ++kk)
    mma_ts(d, a_tmem + kk * 8, b + kk * (2048 >> 4), idesc, accumulate || kk != 0);
}

// The part of that product that takes the first or second 16 of every 32 columns
// of A, which lie in the first half of the 32 columns of FP32 that they were.
template <int HD, int kRows>
__device__ __forceinline__ void mma_cols_half(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, int half,
                                              bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < kRows / 16; kk += 2)
    mma_ts(d, a_tmem + kk * 16 + half * 8, b + (kk + half) * (2048 >> 4), idesc, accumulate || kk + half != 0);
}

int packed_log2(int Hq, int Hkv);
// Row tiles of kTile packed rows over all heads and sequences.
int64_t fwd_ctas(int B, int Sq, int Hq, int Hkv);
// A call of at most 2048 rows (tokens x heads) over at most 512 keys: its results can
// be so few that a second rounding of each shows, and its time is mostly latency.
// The products' rounded operands come in two bf16 parts there, forward and backward.
// With one part 210 of 5788 drawn calls were over 1.5 times as far off as FP32
// rounded once (2 tokens: 2.4 times), all of them this small; with two none.  It
// costs 2 x 128 tokens, 4/2 heads of 64 6.3 + 19.6 us instead of 6.0 + 19.4, and at
// the border (1 x 512 tokens, 4/2 heads of 128) a backward of 37.6 instead of 33.8.
// Beyond it the roundings of more results average out to 1.41 - 1.47 times.
inline bool few_results(int64_t rows, int64_t Sk) { return rows <= 2048 && Sk <= 4 * kTile; }
void fill_shape(Shape& s, int B, int Sq, int Sk, int Hq, int Hkv, int D, const int* begin, const int* end, float scale,
                float cap, const float* slopes);

}  // namespace attn

// Tiled tensor map of any rank: dims and box innermost first, stride_bytes of
// the dimensions from the second on; after current_context (fl_gemm.cu).
int current_context(int* dev);
int make_tensor_map(CUtensorMap* map, const void* base, CUtensorMapDataType dt, int rank, const uint64_t* dims,
                    const uint64_t* stride_bytes, const uint32_t* box, CUtensorMapSwizzle swz);
int allow_smem(const void* kernel, int bytes);

// Argument checks of both directions; bases and strides (batch, token, head) of
// q, k, v and, with tensors = 4, dout.
int attn_check(const char* who, int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int D, const int64_t* strides,
               int tensors, const void* const* bases, const int* begin, const int* end, float scale, float cap);

// bf16 [B, S, H, D] with element strides, as boxes of 64 columns x `heads`
// heads x `tokens` tokens (128-byte swizzle; columns past D read as zero).
int attn_map(CUtensorMap* map, const void* base, int64_t batch_stride, int64_t token_stride, int64_t head_stride, int B,
             int S, int H, int D, int heads, int tokens);

}  // namespace fl
