// Rotary position embedding of queries and keys, with an optional RMS norm of
// every head in the same pass, forward and backward.
//
//   angle(t, p) = position[t] * inv_freq[p],  c = factor cos, s = factor sin
//   (y1, y2) = (c x1 - s x2, c x2 + s x1) for pair p of the first `rot`
//   columns; columns from `rot` on pass through.  Pairs are columns
//   (p, p + rot/2), or (2p, 2p + 1) when interleaved.
//   With a norm x is first x * r * w, r = rsqrt(mean(x^2) + eps).
//   Backward: g = the transposed rotation of dy; without a norm dx = g; with
//   one, xh = x r, dw += g xh, dx = r (g w - xh mean(g w xh)).
//
// Every value is read once and written once; all arithmetic between is FP32
// and each result is rounded once.  HBM bounds it.  Angles are formed in the
// kernel from the positions: a token's rot/2 sines and cosines serve all its
// heads from shared memory, so no table crosses HBM.  The product position *
// inv_freq and its reduction to a fraction of a turn are FP64 (in FP32 a far
// position leaves no fraction), the sine and cosine of the fraction FP32.
//
// Vector form (head size and rot multiples of 16, 16-byte aligned rows): a
// thread owns the two 8-column vectors whose columns pair up, so a rotation
// needs no exchange between threads and a head's sum of squares is a shuffle
// over head_dim/16 neighbouring lanes.  Instructions come next after HBM, so the
// arithmetic works on pairs of FP32 values, angles and weights lie in shared
// memory as neighbouring lanes read them, and rows per block leave few lanes
// idle.  Measured at 8192 tokens: 32 + 8 heads of 128 30 us forward or backward
// (168 MB: 5.5 TB/s, 85% of a copy's rate); with a norm 32 + 4 heads 34.5 us
// forward (4.4 TB/s) and 49 us backward (226 MB: 4.7 TB/s), 61 us with the weights'
// gradients (128 registers, at most 296 blocks).  Other shapes take
// the scalar form, a warp per head, which loads each column's partner as well
// (1027 tokens, 16 heads of 80, 40 columns rotated: 11 us, 1.5 as a copy).
#include <cuda_bf16.h>
#include <cstdint>

#include "fl_host.h"
#include "fl_ptx.cuh"

namespace fl {
namespace rot {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;
constexpr int kChunk = 4;          // items a thread loads before it uses the first
constexpr int kMaxTokens = 16;     // tokens of one block
constexpr int kGradBlocks = 296;   // blocks of a backward that sums weight gradients

struct Side {                      // queries or keys
  const __nv_bfloat16* x;          // the normalized (or rotated) input; backward: read with a norm only
  const __nv_bfloat16* dy;         // backward
  __nv_bfloat16* out;              // contiguous [T, heads, D]
  int64_t x_tok, x_head, dy_tok, dy_head;
  const void* w;                   // [D] norm weight
};

struct Args {
  Side side[2];
  int heads_q, heads;              // query heads, query + key heads
  int64_t T;
  int D, rot;
  const void* pos;
  int pos64, w16;
  const float* inv;
  float factor, eps;
  int tokens;                      // tokens per block
  unsigned heads_magic;            // ceil(2^32 / heads), 0 for one head: row / heads for a block's rows
  int lanes_log2;                  // lanes per head (vector form)
  float* dw_part;                  // [gridDim.x][2][D]
};

__device__ __forceinline__ float2 cos_sin(const Args& a, int64_t t, int p) {
  const double pos = a.pos64 ? static_cast<double>(static_cast<const int64_t*>(a.pos)[t])
                             : static_cast<double>(static_cast<const int32_t*>(a.pos)[t]);
  double turns = pos * static_cast<double>(a.inv[p]) * 0.15915494309189533577;  // 1 / (2 pi)
  turns -= rint(turns);
  float s, c;
  sincospif(2.0f * static_cast<float>(turns), &s, &c);
  return make_float2(c * a.factor, s * a.factor);
}

__device__ __forceinline__ float weight_at(const Args& a, int which, int d) {
  const void* w = a.side[which].w;
  return a.w16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[d]) : static_cast<const float*>(w)[d];
}

// Streamed once: keep the lines out of L1.
__device__ __forceinline__ uint4 load_stream(const __nv_bfloat16* p) {
  return __ldcs(reinterpret_cast<const uint4*>(p));
}

// Eight columns as four pairs of FP32 values; one instruction works on a pair.
struct V8 {
  uint64_t p[4];
};
__device__ __forceinline__ V8 unpack(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = pair(w[i] << 16, w[i] & 0xFFFF0000u);
  return r;
}
__device__ __forceinline__ uint4 pack(const V8& v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    unpair(v.p[i], lo, hi);
    w[i] = pack_bf16x2(lo, hi);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ V8 mul(const V8& a, const V8& b) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = mul2(a.p[i], b.p[i]);
  return r;
}
__device__ __forceinline__ void scale(V8& a, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) a.p[i] = mul2(a.p[i], pair(s, s));
}
__device__ __forceinline__ float dot(const V8& a0, const V8& b0, const V8& a1, const V8& b1) {
  uint64_t s = mul2(a0.p[0], b0.p[0]), t = mul2(a1.p[0], b1.p[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    s = fma2(a0.p[i], b0.p[i], s);
    t = fma2(a1.p[i], b1.p[i], t);
  }
  float lo, hi;
  unpair(add2(s, t), lo, hi);
  return lo + hi;
}
constexpr uint64_t kSigns = 0x8000000080000000ull;

// Turns the pairs of two vectors in place; kBack: by the negative angles.
// cs[i * stride] = {cos, cos, sin, sin} of the pairs 2i and 2i + 1.
template <bool kInter, bool kBack>
__device__ __forceinline__ void turn(V8& a, V8& b, const float4* cs, int stride) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(cs + i * stride);
    const uint64_t c = v.x, s = kBack ? v.y ^ kSigns : v.y, n = kBack ? v.y : v.y ^ kSigns;
    if constexpr (!kInter) {
      const uint64_t x = a.p[i];
      a.p[i] = fma2(c, x, mul2(n, b.p[i]));
      b.p[i] = fma2(c, b.p[i], mul2(s, x));
    } else {
      float c0, c1, s0, s1, n0, n1;
      unpair(c, c0, c1);
      unpair(s, s0, s1);
      unpair(n, n0, n1);
      V8& x = i < 2 ? a : b;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint64_t& y = x.p[2 * (i & 1) + e];
        float lo, hi;
        unpair(y, lo, hi);
        y = fma2(e ? pair(c1, c1) : pair(c0, c0), y, mul2(e ? pair(n1, s1) : pair(n0, s0), pair(hi, lo)));
      }
    }
  }
}

template <bool kNorm, bool kInter, bool kBwd, bool kDw>
__global__ void __launch_bounds__(kThreads, kNorm && kBwd ? 2 : 3) vec_kernel(const Args a) {
  constexpr int kItems = kNorm && kBwd ? kChunk / 2 : kChunk;  // rows loaded before the first is used
  // (cos, cos, sin, sin) of [token][i][slot], weights of [side][i][slot]: the
  // lanes of a head read neighbouring words.
  __shared__ float4 cs4[kMaxTokens * kMaxDim / 4];
  __shared__ float4 w4[kNorm ? 2 * kMaxDim / 4 : 1];
  const int L = 1 << a.lanes_log2, D = a.D, half = a.rot >> 1;
  const int slots = D >> 4, turned = a.rot >> 4;
  const int slot = threadIdx.x & (L - 1);
  const bool live_slot = slot < slots;
  // Columns of a slot's two vectors.
  auto first_col = [&](int sl) { return kInter ? 16 * sl : (sl < turned ? 8 * sl : a.rot + 16 * (sl - turned)); };
  auto second_col = [&](int sl) { return first_col(sl) + (kInter || sl >= turned ? 8 : half); };
  const int c0 = first_col(slot), c1 = second_col(slot);
  uint64_t accq[kDw ? 8 : 1], acck[kDw ? 8 : 1];
  if constexpr (kDw) {
#pragma unroll
    for (int i = 0; i < 8; ++i) accq[i] = acck[i] = 0;
  }
  if constexpr (kNorm) {
    for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
      const int which = i >= D, j = i - which * D, e = j & 15, sl = j >> 4;
      const int col = e < 8 ? first_col(sl) + e : second_col(sl) + e - 8;
      if (which == 0 || a.heads > a.heads_q)
        reinterpret_cast<float*>(w4 + (which * 4 + (e >> 2)) * slots + sl)[e & 3] = weight_at(a, which, col);
    }
  }
  const int step = kThreads >> a.lanes_log2;       // rows a pass of the block covers
  const int row0 = threadIdx.x >> a.lanes_log2;
  const float inv_d = 1.0f / static_cast<float>(D);
  const Side q = a.side[0], k = a.side[1];

  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens; t0 < a.T;
       t0 += static_cast<int64_t>(gridDim.x) * a.tokens) {
    const int n_tokens = static_cast<int>(a.T - t0 < a.tokens ? a.T - t0 : a.tokens);
    const int n_rows = n_tokens * a.heads;         // (token, head) rows of the block
    bool first = true;
    const __nv_bfloat16 *qx = q.x + t0 * q.x_tok, *kx = k.x + t0 * k.x_tok;
    const __nv_bfloat16 *qd = q.dy + t0 * q.dy_tok, *kd = k.dy + t0 * k.dy_tok;
    __nv_bfloat16 *qo = q.out + t0 * (a.heads_q * D), *ko = k.out + t0 * ((a.heads - a.heads_q) * D);
    // Uniform trip counts: every lane takes part in the shuffles of each row.
    for (int rb = 0; rb < n_rows; rb += kItems * step) {
      uint4 xa[kItems], xb[kItems], da[kBwd ? kItems : 1], db[kBwd ? kItems : 1];
      int tok[kItems], head[kItems];
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        if (rb + u * step >= n_rows) continue;
        const int row = rb + u * step + row0;
        tok[u] = a.heads_magic ? __umulhi(row, a.heads_magic) : row;   // row / heads
        head[u] = row - tok[u] * a.heads;
        xa[u] = xb[u] = make_uint4(0, 0, 0, 0);
        if constexpr (kBwd) da[u] = db[u] = make_uint4(0, 0, 0, 0);
        if (live_slot && row < n_rows) {
          const bool is_k = head[u] >= a.heads_q;
          const int h = is_k ? head[u] - a.heads_q : head[u];
          if constexpr (!kBwd || kNorm) {
            const __nv_bfloat16* p = (is_k ? kx : qx) + (tok[u] * static_cast<int>(is_k ? k.x_tok : q.x_tok) +
                                                         h * static_cast<int>(is_k ? k.x_head : q.x_head));
            xa[u] = load_stream(p + c0);
            xb[u] = load_stream(p + c1);
          }
          if constexpr (kBwd) {
            const __nv_bfloat16* p = (is_k ? kd : qd) + (tok[u] * static_cast<int>(is_k ? k.dy_tok : q.dy_tok) +
                                                         h * static_cast<int>(is_k ? k.dy_head : q.dy_head));
            da[u] = load_stream(p + c0);
            db[u] = load_stream(p + c1);
          }
        }
      }
      if (first) {  // the block's angles, formed while the first loads are in flight
        first = false;
        __syncthreads();
        for (int i = threadIdx.x; i < n_tokens * half; i += kThreads) {
          const int tl = i / half, p = i - tl * half;
          const float2 cs = cos_sin(a, t0 + tl, p);
          float* o = reinterpret_cast<float*>(cs4 + (tl * 4 + ((p & 7) >> 1)) * turned + (p >> 3)) + (p & 1);
          o[0] = cs.x;
          o[2] = cs.y;
        }
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        if (rb + u * step >= n_rows) break;
        const bool live = live_slot && rb + u * step + row0 < n_rows;
        const bool is_k = head[u] >= a.heads_q;
        const float4* cs = cs4 + tok[u] * 4 * turned + slot;
        const bool turns = live && slot < turned;
        V8 w0, w1, y0, y1;
        if constexpr (kNorm) {
          const float4* w = w4 + (is_k ? 4 * slots : 0) + (live ? slot : 0);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(w + i * slots);
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(w + (2 + i) * slots);
            w0.p[2 * i] = v.x, w0.p[2 * i + 1] = v.y;
            w1.p[2 * i] = x.x, w1.p[2 * i + 1] = x.y;
          }
        }
        if constexpr (!kBwd) {
          y0 = unpack(xa[u]);
          y1 = unpack(xb[u]);
          if constexpr (kNorm) {
            float ss = dot(y0, y0, y1, y1);
            for (int o = L >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = rsqrtf(ss * inv_d + a.eps);
            y0 = mul(y0, w0);
            y1 = mul(y1, w1);
            scale(y0, r);
            scale(y1, r);
          }
          if (turns) turn<kInter, false>(y0, y1, cs, turned);
        } else {
          y0 = unpack(da[u]);
          y1 = unpack(db[u]);
          if (turns) turn<kInter, true>(y0, y1, cs, turned);
          if constexpr (kNorm) {
            const V8 x0 = unpack(xa[u]), x1 = unpack(xb[u]);
            const V8 g0 = mul(y0, w0), g1 = mul(y1, w1);
            float ss = dot(x0, x0, x1, x1), gx = dot(g0, x0, g1, x1);
            for (int o = L >> 1; o; o >>= 1) {
              ss += __shfl_xor_sync(0xffffffffu, ss, o);
              gx += __shfl_xor_sync(0xffffffffu, gx, o);
            }
            const float r = rsqrtf(ss * inv_d + a.eps);
            const float m = -gx * r * r * inv_d;   // -mean(g w xh) r
            if constexpr (kDw) {
              if (live) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint64_t e0 = mul2(x0.p[i], pair(r, r)), e1 = mul2(x1.p[i], pair(r, r));
                  if (is_k) {
                    acck[i] = fma2(y0.p[i], e0, acck[i]);
                    acck[4 + i] = fma2(y1.p[i], e1, acck[4 + i]);
                  } else {
                    accq[i] = fma2(y0.p[i], e0, accq[i]);
                    accq[4 + i] = fma2(y1.p[i], e1, accq[4 + i]);
                  }
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              y0.p[i] = fma2(x0.p[i], pair(m, m), g0.p[i]);
              y1.p[i] = fma2(x1.p[i], pair(m, m), g1.p[i]);
            }
            scale(y0, r);
            scale(y1, r);
          }
        }
        if (live) {
          const int heads = is_k ? a.heads - a.heads_q : a.heads_q, h = is_k ? head[u] - a.heads_q : head[u];
          __nv_bfloat16* o = (is_k ? ko : qo) + (tok[u] * heads + h) * D;
          __stcs(reinterpret_cast<uint4*>(o + c0), pack(y0));
          __stcs(reinterpret_cast<uint4*>(o + c1), pack(y1));
        }
      }
    }
  }

  if constexpr (kDw) {
    // Per-thread sums -> per-block sums, the threads of a slot in order.
    float* red = reinterpret_cast<float*>(cs4);    // [kThreads][16] floats fit the angles' space
    static_assert(kThreads * 16 <= kMaxTokens * kMaxDim, "the weight sums reuse the angles' space");
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i)
        reinterpret_cast<uint64_t*>(red)[threadIdx.x * 8 + i] = which ? acck[i] : accq[i];
      __syncthreads();
      for (int i = threadIdx.x; i < slots * 16; i += kThreads) {
        const int sl = i >> 4, e = i & 15;
        float sum = 0.f;
        for (int r = 0; r < step; ++r) sum += red[((r << a.lanes_log2) + sl) * 16 + e];
        a.dw_part[(static_cast<int64_t>(blockIdx.x) * 2 + which) * D +
                  (e < 8 ? first_col(sl) + e : second_col(sl) + e - 8)] = sum;
      }
    }
  }
}

// Scalar form: a block per few tokens, a warp per (token, head) row, lane l holding columns l, l + 32, ...
template <bool kNorm, bool kInter, bool kBwd, bool kDw>
__global__ void __launch_bounds__(kThreads) scalar_kernel(const Args a) {
  constexpr int kPer = kMaxDim / 32;
  constexpr int kWarps = kThreads / 32;
  __shared__ float red[kDw ? kWarps * kMaxDim : 1];
  __shared__ float2 angles[kMaxTokens * kMaxDim / 2];   // (cos, sin) of [token][rot / 2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = a.D, half = a.rot >> 1;
  float accq[kDw ? kPer : 1], acck[kDw ? kPer : 1];
  if constexpr (kDw) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) accq[i] = acck[i] = 0.f;
  }
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens; t0 < a.T;
       t0 += static_cast<int64_t>(gridDim.x) * a.tokens) {
    const int n_tokens = static_cast<int>(a.T - t0 < a.tokens ? a.T - t0 : a.tokens);
    __syncthreads();
    for (int i = threadIdx.x; i < n_tokens * half; i += kThreads) angles[i] = cos_sin(a, t0 + i / half, i % half);
    __syncthreads();
    for (int row = warp; row < n_tokens * a.heads; row += kWarps) {
      const int tl = row / a.heads;
      const int64_t t = t0 + tl;
      int h = row - tl * a.heads;
      const int which = h >= a.heads_q;
      const Side& s = a.side[which];
      if (which) h -= a.heads_q;
      const __nv_bfloat16* x = s.x + t * s.x_tok + h * s.x_head;
      const __nv_bfloat16* dy = kBwd ? s.dy + t * s.dy_tok + h * s.dy_head : nullptr;
      __nv_bfloat16* out = s.out + (t * (which ? a.heads - a.heads_q : a.heads_q) + h) * D;
      float r = 1.f;
      if constexpr (kNorm) {
        float ss = 0.f;
        for (int d = lane; d < D; d += 32) {
          const float v = __bfloat162float(x[d]);
          ss += v * v;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        r = rsqrtf(ss / static_cast<float>(D) + a.eps);
      }
      float y[kPer], gx = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int d = lane + 32 * i;
        y[i] = 0.f;
        if (d >= D) continue;
        const __nv_bfloat16* in = kBwd ? dy : x;
        float v = __bfloat162float(in[d]);
        if constexpr (kNorm && !kBwd) v *= r * weight_at(a, which, d);
        if (d < a.rot) {
          const bool left = kInter ? (d & 1) == 0 : d < half;
          const int mate = kInter ? d ^ 1 : (left ? d + half : d - half);
          float m = __bfloat162float(in[mate]);
          if constexpr (kNorm && !kBwd) m *= r * weight_at(a, which, mate);
          const float2 cs = angles[tl * half + (kInter ? d >> 1 : (left ? d : mate))];
          // forward: left -s, right +s; the transposed rotation: left +s, right -s
          v = cs.x * v + ((left == kBwd) ? cs.y : -cs.y) * m;
        }
        y[i] = v;
        if constexpr (kNorm && kBwd) gx += v * weight_at(a, which, d) * __bfloat162float(x[d]);
      }
      if constexpr (kNorm && kBwd) {
#pragma unroll
        for (int o = 16; o; o >>= 1) gx += __shfl_xor_sync(0xffffffffu, gx, o);
        const float m = gx * r * r / static_cast<float>(D);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int d = lane + 32 * i;
          if (d >= D) continue;
          const float xv = __bfloat162float(x[d]);
          if constexpr (kDw) {
            if (which)
              acck[i] += y[i] * (xv * r);
            else
              accq[i] += y[i] * (xv * r);
          }
          y[i] = r * (y[i] * weight_at(a, which, d) - xv * m);
        }
      }
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i < D) out[lane + 32 * i] = __float2bfloat16_rn(y[i]);
    }
  }
  if constexpr (kDw) {
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) red[warp * kMaxDim + lane + 32 * i] = which ? acck[i] : accq[i];
      __syncthreads();
      for (int d = threadIdx.x; d < D; d += kThreads) {
        float sum = 0.f;
        for (int w = 0; w < kWarps; ++w) sum += red[w * kMaxDim + d];
        a.dw_part[(static_cast<int64_t>(blockIdx.x) * 2 + which) * D + d] = sum;
      }
    }
  }
}

// Sums the blocks' weight gradients in block order: 32 columns to a block, 32
// row groups, then the groups in order.
__global__ void dw_kernel(const float* __restrict__ part, int blocks, int D, float* __restrict__ dqw,
                          float* __restrict__ dkw) {
  __shared__ float red[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.f;
  if (col < 2 * D)
    for (int b = threadIdx.y; b < blocks; b += 32) sum += part[static_cast<int64_t>(b) * 2 * D + col];
  red[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && col < 2 * D) {
    sum = 0.f;
    for (int g = 0; g < 32; ++g) sum += red[g][threadIdx.x];
    float* out = col < D ? dqw : dkw;
    if (out) out[col < D ? col : col - D] = sum;
  }
}

using Kernel = void (*)(const Args);

template <bool kNorm, bool kBwd, bool kDw>
Kernel pick(bool vec, bool inter) {
  if (vec) return inter ? vec_kernel<kNorm, true, kBwd, kDw> : vec_kernel<kNorm, false, kBwd, kDw>;
  return inter ? scalar_kernel<kNorm, true, kBwd, kDw> : scalar_kernel<kNorm, false, kBwd, kDw>;
}

// 16-byte rows, offsets within a block in 32 bits.
bool rows_fit(const void* p, int64_t tok, int64_t head, int heads) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && tok % 8 == 0 && head % 8 == 0 && tok >= 0 && head >= 0 &&
         tok * kMaxTokens + head * heads < (int64_t(1) << 31);
}

int launch(Args& a, bool norm, bool inter, bool bwd, float* dqw, float* dkw, cudaStream_t stream) {
  int dev = 0;
  const int sms = device_sms(cudaGetDevice(&dev) == cudaSuccess ? dev : -1);
  bool vec = a.D % 16 == 0 && a.rot % 16 == 0 && a.heads <= 4096;
  for (int i = 0; i < (a.heads > a.heads_q ? 2 : 1); ++i) {
    const Side& s = a.side[i];
    vec = vec && (reinterpret_cast<uintptr_t>(s.out) & 15u) == 0;
    if (!bwd || norm) vec = vec && rows_fit(s.x, s.x_tok, s.x_head, a.heads);
    if (bwd) vec = vec && rows_fit(s.dy, s.dy_tok, s.dy_head, a.heads);
  }
  const bool dw = dqw || dkw;
  const Kernel kernel = !bwd ? (norm ? pick<true, false, false>(vec, inter) : pick<false, false, false>(vec, inter))
                        : !norm ? pick<false, true, false>(vec, inter)
                        : dw    ? pick<true, true, true>(vec, inter)
                                : pick<true, true, false>(vec, inter);
  int64_t grid;
  if (vec) {
    a.lanes_log2 = 0;
    while ((16 << a.lanes_log2) < a.D) ++a.lanes_log2;
    // Tokens of a block: up to two loads' worth of rows, the count that leaves
    // the fewest of a pass's rows idle (36 heads of 128: 4 tokens in 160 rows
    // measured 41 us where 128 + 32 of 256 took 54); fewer while the blocks
    // would not cover the GPU twice.
    const int64_t pass = kThreads >> a.lanes_log2;
    int64_t tokens = 1;
    auto use = [&](int64_t n) { return static_cast<double>(n * a.heads) / ((n * a.heads + pass - 1) / pass * pass); };
    for (int64_t n = 2; n <= kMaxTokens && n * a.heads <= 2 * kChunk * pass; ++n)
      if (use(n) > use(tokens) + 0.01) tokens = n;
    while (tokens > 1 && (a.T + tokens - 1) / tokens < 2 * sms) --tokens;
    a.tokens = static_cast<int>(tokens);
    // exact while row * heads < 2^32
    a.heads_magic = static_cast<unsigned>(((uint64_t(1) << 32) + a.heads - 1) / a.heads);
    grid = (a.T + tokens - 1) / tokens;
  } else {
    // Two rows to a warp at least, so that a block's angles serve them.
    int64_t tokens = (2 * (kThreads / 32) + a.heads - 1) / a.heads;
    if (tokens > kMaxTokens) tokens = kMaxTokens;
    while (tokens > 1 && (a.T + tokens - 1) / tokens < 2 * sms) --tokens;
    a.tokens = static_cast<int>(tokens);
    grid = (a.T + tokens - 1) / tokens;
  }
  if (dw && grid > kGradBlocks) grid = kGradBlocks;
  if (grid > 0x7fffffff) grid = 0x7fffffff;
  kernel<<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
  if (dw) dw_kernel<<<(2 * a.D + 31) / 32, dim3(32, 32), 0, stream>>>(a.dw_part, static_cast<int>(grid), a.D, dqw, dkw);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FL_ERR_CUDA, "rotary launch: %s", cudaGetErrorString(e));
  return FL_OK;
}

int check(const char* who, int64_t T, int Hq, int Hk, int D, const void* pos, int pos_bytes, const float* inv, int rot,
          const void* qw, const void* kw, int w_bytes, float eps) {
  if (T < 0 || Hq < 1 || Hk < 0 || T > (int64_t(1) << 31) || Hq > 65536 || Hk > 65536)
    return set_error(FL_ERR_ARG, "%s: bad token or head count", who);
  if (D < 2 || D > kMaxDim) return set_error(FL_ERR_ARG, "%s: head size must be in [2, %d]", who, kMaxDim);
  if (rot < 2 || rot > D || rot % 2) return set_error(FL_ERR_ARG, "%s: rotated columns must be even and in [2, head size]", who);
  if (pos_bytes != 4 && pos_bytes != 8) return set_error(FL_ERR_ARG, "%s: positions must be 32- or 64-bit integers", who);
  if (w_bytes != 0 && w_bytes != 2 && w_bytes != 4)
    return set_error(FL_ERR_ARG, "%s: norm weights must be bf16 (2 bytes) or fp32 (4 bytes)", who);
  if (w_bytes && !(eps >= 0.f)) return set_error(FL_ERR_ARG, "%s: eps must be >= 0", who);
  if (T && (!pos || !inv)) return set_error(FL_ERR_ARG, "%s: null pointer", who);
  if (T && w_bytes && (!qw || (Hk && !kw))) return set_error(FL_ERR_ARG, "%s: null norm weight", who);
  return FL_OK;
}

}  // namespace rot
}  // namespace fl

using namespace fl;

extern "C" {

int fl_rotary_fwd(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, int Hq, const uint16_t* k,
                  int64_t k_token_stride, int64_t k_head_stride, int Hk, int64_t T, int D, const void* positions,
                  int position_bytes, const float* inv_freq, int rot, int interleaved, float factor,
                  const void* q_weight, const void* k_weight, int weight_bytes, float eps, uint16_t* q_out,
                  uint16_t* k_out, void* stream) {
  int rc = rot::check("fl_rotary_fwd", T, Hq, Hk, D, positions, position_bytes, inv_freq, rot, q_weight, k_weight,
                      weight_bytes, eps);
  if (rc || T == 0) return rc;
  if (!q || !q_out || (Hk && (!k || !k_out))) return set_error(FL_ERR_ARG, "fl_rotary_fwd: null pointer");
  rot::Args a{};
  a.side[0] = {reinterpret_cast<const __nv_bfloat16*>(q), nullptr, reinterpret_cast<__nv_bfloat16*>(q_out),
               q_token_stride, q_head_stride, 0, 0, q_weight};
  a.side[1] = {reinterpret_cast<const __nv_bfloat16*>(k), nullptr, reinterpret_cast<__nv_bfloat16*>(k_out),
               k_token_stride, k_head_stride, 0, 0, k_weight};
  a.heads_q = Hq;
  a.heads = Hq + Hk;
  a.T = T;
  a.D = D;
  a.rot = rot;
  a.pos = positions;
  a.pos64 = position_bytes == 8;
  a.w16 = weight_bytes == 2;
  a.inv = inv_freq;
  a.factor = factor;
  a.eps = eps;
  return rot::launch(a, weight_bytes != 0, interleaved != 0, false, nullptr, nullptr,
                     static_cast<cudaStream_t>(stream));
}

size_t fl_rotary_bwd_workspace_bytes(int D) {
  return D > 0 ? static_cast<size_t>(rot::kGradBlocks) * 2 * D * sizeof(float) : 0;
}

int fl_rotary_bwd(const uint16_t* dq, int64_t dq_token_stride, int64_t dq_head_stride, const uint16_t* dk,
                  int64_t dk_token_stride, int64_t dk_head_stride, const uint16_t* q, int64_t q_token_stride,
                  int64_t q_head_stride, int Hq, const uint16_t* k, int64_t k_token_stride, int64_t k_head_stride,
                  int Hk, int64_t T, int D, const void* positions, int position_bytes, const float* inv_freq, int rot,
                  int interleaved, float factor, const void* q_weight, const void* k_weight, int weight_bytes,
                  float eps, uint16_t* dq_out, uint16_t* dk_out, float* dq_weight, float* dk_weight, void* workspace,
                  size_t workspace_bytes, void* stream) {
  int rc = rot::check("fl_rotary_bwd", T, Hq, Hk, D, positions, position_bytes, inv_freq, rot, q_weight, k_weight,
                      weight_bytes, eps);
  if (rc) return rc;
  const bool norm = weight_bytes != 0, dw = dq_weight || dk_weight;
  if (dw && !norm) return set_error(FL_ERR_ARG, "fl_rotary_bwd: weight gradients without norm weights");
  if (dw && (!workspace || workspace_bytes < fl_rotary_bwd_workspace_bytes(D) ||
             (reinterpret_cast<uintptr_t>(workspace) & 3u)))
    return set_error(FL_ERR_ARG, "fl_rotary_bwd: workspace missing, short or misaligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    for (float* w : {dq_weight, dk_weight})
      if (w && cudaMemsetAsync(w, 0, static_cast<size_t>(D) * sizeof(float), st) != cudaSuccess)
        return set_error(FL_ERR_CUDA, "fl_rotary_bwd: clearing the weight gradients failed");
    return FL_OK;
  }
  if (!dq || !dq_out || (Hk && (!dk || !dk_out)) || (norm && (!q || (Hk && !k))))
    return set_error(FL_ERR_ARG, "fl_rotary_bwd: null pointer");
  rot::Args a{};
  a.side[0] = {reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<const __nv_bfloat16*>(dq),
               reinterpret_cast<__nv_bfloat16*>(dq_out), q_token_stride, q_head_stride, dq_token_stride,
               dq_head_stride, q_weight};
  a.side[1] = {reinterpret_cast<const __nv_bfloat16*>(k), reinterpret_cast<const __nv_bfloat16*>(dk),
               reinterpret_cast<__nv_bfloat16*>(dk_out), k_token_stride, k_head_stride, dk_token_stride,
               dk_head_stride, k_weight};
  a.heads_q = Hq;
  a.heads = Hq + Hk;
  a.T = T;
  a.D = D;
  a.rot = rot;
  a.pos = positions;
  a.pos64 = position_bytes == 8;
  a.w16 = weight_bytes == 2;
  a.inv = inv_freq;
  a.factor = factor;
  a.eps = eps;
  a.dw_part = static_cast<float*>(workspace);
  return rot::launch(a, norm, interleaved != 0, true, dq_weight, dk_weight, st);
}

}  // extern "C"
