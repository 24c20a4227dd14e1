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
// over head_dim/16 neighbouring lanes.  Other shapes take the scalar form, a
// warp per head, which loads each column's partner as well.
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

__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}

// Streamed once: keep the lines out of L1.
__device__ __forceinline__ uint4 load_stream(const __nv_bfloat16* p) {
  return __ldcs(reinterpret_cast<const uint4*>(p));
}

template <bool kNorm, bool kInter, bool kBwd, bool kDw>
__global__ void __launch_bounds__(kThreads) vec_kernel(const Args a) {
  __shared__ float4 cs4[kMaxTokens * kMaxDim / 4];   // (cos, sin) of [token][rot / 2]
  __shared__ float ws[kNorm ? 2 * kMaxDim : 1];
  float2* cs = reinterpret_cast<float2*>(cs4);
  const int L = 1 << a.lanes_log2, D = a.D, half = a.rot >> 1;
  const int slots = D >> 4, turned = a.rot >> 4;
  const int slot = threadIdx.x & (L - 1);
  const bool live_slot = slot < slots;
  // Columns of the thread's two vectors.
  const int c0 = kInter ? 16 * slot : (slot < turned ? 8 * slot : a.rot + 16 * (slot - turned));
  const int c1 = kInter ? c0 + 8 : (slot < turned ? c0 + half : c0 + 8);
  float accq[kDw ? 16 : 1], acck[kDw ? 16 : 1];
  if constexpr (kDw) {
#pragma unroll
    for (int i = 0; i < 16; ++i) accq[i] = acck[i] = 0.f;
  }
  if constexpr (kNorm) {
    for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
      const int which = i >= D;
      if (which == 0 || a.heads > a.heads_q) ws[i] = weight_at(a, which, i - which * D);
    }
  }
  const int n_rows = a.tokens * a.heads;           // (token, head) rows of a full block
  const int step = kThreads >> a.lanes_log2;       // rows a pass of the block covers
  const int row0 = threadIdx.x >> a.lanes_log2;
  const float inv_d = 1.0f / static_cast<float>(D);

  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens; t0 < a.T;
       t0 += static_cast<int64_t>(gridDim.x) * a.tokens) {
    bool first = true;
    // Uniform trip count: every lane takes part in the shuffles of each row.
    for (int rb = 0; rb < n_rows; rb += kChunk * step) {
      uint4 xa[kChunk], xb[kChunk], da[kBwd ? kChunk : 1], db[kBwd ? kChunk : 1];
#pragma unroll
      for (int u = 0; u < kChunk; ++u) {
        const int row = rb + u * step + row0;
        const int tl = row / a.heads;
        int h = row - tl * a.heads;
        const int64_t t = t0 + tl;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        xa[u] = xb[u] = zero;
        if constexpr (kBwd) da[u] = db[u] = zero;
        if (live_slot && row < n_rows && t < a.T) {
          const Side& s = a.side[h >= a.heads_q];
          if (h >= a.heads_q) h -= a.heads_q;
          if constexpr (!kBwd || kNorm) {
            const __nv_bfloat16* p = s.x + t * s.x_tok + h * s.x_head;
            xa[u] = load_stream(p + c0);
            xb[u] = load_stream(p + c1);
          }
          if constexpr (kBwd) {
            const __nv_bfloat16* p = s.dy + t * s.dy_tok + h * s.dy_head;
            da[u] = load_stream(p + c0);
            db[u] = load_stream(p + c1);
          }
        }
      }
      if (first) {  // the block's angles, formed while the first loads are in flight
        first = false;
        __syncthreads();
        for (int i = threadIdx.x; i < a.tokens * half; i += kThreads) {
          const int tl = i / half;
          if (t0 + tl < a.T) cs[i] = cos_sin(a, t0 + tl, i - tl * half);
        }
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < kChunk; ++u) {
        const int row = rb + u * step + row0;
        const int tl = row / a.heads;
        int h = row - tl * a.heads;
        const int64_t t = t0 + tl;
        const bool live = live_slot && row < n_rows && t < a.T;
        const int which = h >= a.heads_q;
        float x0[8], x1[8], y0[8], y1[8], c[8], sn[8];
        unpack8(xa[u], x0);
        unpack8(xb[u], x1);
        if (live && slot < turned) {
          const float4* q = cs4 + ((tl * half) >> 1) + slot * 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 v = q[i];
            c[2 * i] = v.x;
            sn[2 * i] = v.y;
            c[2 * i + 1] = v.z;
            sn[2 * i + 1] = v.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i] = 1.f, sn[i] = 0.f;
        }
        const float* w = ws + which * D;
        if constexpr (!kBwd) {
          if constexpr (kNorm) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += x0[i] * x0[i] + x1[i] * x1[i];
            for (int o = L >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = rsqrtf(ss * inv_d + a.eps);
            if (live) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                x0[i] *= r * w[c0 + i];
                x1[i] *= r * w[c1 + i];
              }
            }
          }
          if constexpr (kInter) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              y0[2 * i] = c[i] * x0[2 * i] - sn[i] * x0[2 * i + 1];
              y0[2 * i + 1] = c[i] * x0[2 * i + 1] + sn[i] * x0[2 * i];
              y1[2 * i] = c[4 + i] * x1[2 * i] - sn[4 + i] * x1[2 * i + 1];
              y1[2 * i + 1] = c[4 + i] * x1[2 * i + 1] + sn[4 + i] * x1[2 * i];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              y0[i] = c[i] * x0[i] - sn[i] * x1[i];
              y1[i] = c[i] * x1[i] + sn[i] * x0[i];
            }
          }
        } else {
          float d0[8], d1[8];
          unpack8(da[u], d0);
          unpack8(db[u], d1);
          if constexpr (kInter) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              y0[2 * i] = c[i] * d0[2 * i] + sn[i] * d0[2 * i + 1];
              y0[2 * i + 1] = c[i] * d0[2 * i + 1] - sn[i] * d0[2 * i];
              y1[2 * i] = c[4 + i] * d1[2 * i] + sn[4 + i] * d1[2 * i + 1];
              y1[2 * i + 1] = c[4 + i] * d1[2 * i + 1] - sn[4 + i] * d1[2 * i];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              y0[i] = c[i] * d0[i] + sn[i] * d1[i];
              y1[i] = c[i] * d1[i] - sn[i] * d0[i];
            }
          }
          if constexpr (kNorm) {
            float ss = 0.f, gx = 0.f, g0[8], g1[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              ss += x0[i] * x0[i] + x1[i] * x1[i];
              g0[i] = live ? y0[i] * w[c0 + i] : 0.f;
              g1[i] = live ? y1[i] * w[c1 + i] : 0.f;
              gx += g0[i] * x0[i] + g1[i] * x1[i];
            }
            for (int o = L >> 1; o; o >>= 1) {
              ss += __shfl_xor_sync(0xffffffffu, ss, o);
              gx += __shfl_xor_sync(0xffffffffu, gx, o);
            }
            const float r = rsqrtf(ss * inv_d + a.eps);
            const float m = gx * r * r * inv_d;   // mean(g w xh) r
            if constexpr (kDw) {
              if (live) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float e0 = y0[i] * (x0[i] * r), e1 = y1[i] * (x1[i] * r);
                  if (which) {
                    acck[i] += e0;
                    acck[8 + i] += e1;
                  } else {
                    accq[i] += e0;
                    accq[8 + i] += e1;
                  }
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              y0[i] = r * (g0[i] - x0[i] * m);
              y1[i] = r * (g1[i] - x1[i] * m);
            }
          }
        }
        if (live) {
          const int heads = which ? a.heads - a.heads_q : a.heads_q;
          if (which) h -= a.heads_q;
          __nv_bfloat16* o = a.side[which].out + (t * heads + h) * D;
          __stcs(reinterpret_cast<uint4*>(o + c0), pack8(y0));
          __stcs(reinterpret_cast<uint4*>(o + c1), pack8(y1));
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
      for (int i = 0; i < 16; ++i) red[threadIdx.x * 16 + i] = which ? acck[i] : accq[i];
      __syncthreads();
      for (int i = threadIdx.x; i < slots * 16; i += kThreads) {
        const int sl = i >> 4, e = i & 15;
        float sum = 0.f;
        for (int r = 0; r < step; ++r) sum += red[((r << a.lanes_log2) + sl) * 16 + e];
        const int b0 = kInter ? 16 * sl : (sl < turned ? 8 * sl : a.rot + 16 * (sl - turned));
        const int b1 = kInter ? b0 + 8 : (sl < turned ? b0 + half : b0 + 8);
        a.dw_part[(static_cast<int64_t>(blockIdx.x) * 2 + which) * D + (e < 8 ? b0 + e : b1 + e - 8)] = sum;
      }
    }
  }
}

// Scalar form: a warp per (token, head) row, lane l holding columns l, l + 32, ...
template <bool kNorm, bool kInter, bool kBwd, bool kDw>
__global__ void __launch_bounds__(kThreads) scalar_kernel(const Args a) {
  constexpr int kPer = kMaxDim / 32;
  __shared__ float red[kDw ? (kThreads / 32) * kMaxDim : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = a.D, half = a.rot >> 1;
  const int64_t rows = a.T * a.heads;
  float accq[kDw ? kPer : 1], acck[kDw ? kPer : 1];
  if constexpr (kDw) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) accq[i] = acck[i] = 0.f;
  }
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + warp; row < rows;
       row += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
    const int64_t t = row / a.heads;
    int h = static_cast<int>(row - t * a.heads);
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
        const float2 cs = cos_sin(a, t, kInter ? d >> 1 : (left ? d : mate));
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
  if constexpr (kDw) {
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) red[warp * kMaxDim + lane + 32 * i] = which ? acck[i] : accq[i];
      __syncthreads();
      for (int d = threadIdx.x; d < D; d += kThreads) {
        float sum = 0.f;
        for (int w = 0; w < kThreads / 32; ++w) sum += red[w * kMaxDim + d];
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

bool rows_aligned(const void* p, int64_t tok, int64_t head) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && tok % 8 == 0 && head % 8 == 0;
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n;
}

int launch(Args& a, bool norm, bool inter, bool bwd, float* dqw, float* dkw, cudaStream_t stream) {
  bool vec = a.D % 16 == 0 && a.rot % 16 == 0;
  for (int i = 0; i < (a.heads > a.heads_q ? 2 : 1); ++i) {
    const Side& s = a.side[i];
    vec = vec && (reinterpret_cast<uintptr_t>(s.out) & 15u) == 0;
    if (!bwd || norm) vec = vec && rows_aligned(s.x, s.x_tok, s.x_head);
    if (bwd) vec = vec && rows_aligned(s.dy, s.dy_tok, s.dy_head);
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
    // About kChunk rows to a thread, so that a block's angles serve many rows;
    // fewer tokens to a block while the blocks would not cover the GPU twice.
    int64_t tokens = (static_cast<int64_t>(kChunk) * (kThreads >> a.lanes_log2) + a.heads / 2) / a.heads;
    tokens = tokens < 1 ? 1 : tokens > kMaxTokens ? kMaxTokens : tokens;
    while (tokens > 1 && (a.T + tokens - 1) / tokens < 2 * sm_count()) --tokens;
    a.tokens = static_cast<int>(tokens);
    grid = (a.T + tokens - 1) / tokens;
  } else {
    grid = (a.T * a.heads + kThreads / 32 - 1) / (kThreads / 32);
    if (grid > (1 << 20)) grid = 1 << 20;
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
