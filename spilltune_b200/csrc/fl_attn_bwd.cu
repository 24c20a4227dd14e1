// Attention backward over row ranges (see fl_attn.cuh for the formulas).
//
//   delta_i = do_i . o_i,  p = 2^(x - lse),  ds = p (do v^T - delta) [(1 - tanh^2)]
//   dv = p^T do,  dk = scale ds^T q,  dq = scale ds k
//
// Three launches: delta with the row tiles' key ranges; dk and dv, a CTA per
// 128 keys of a key/value head, walking the query tiles of its whole head
// group (so the group's sum stays in one accumulator); dq, a CTA per 128
// (packed) query rows, walking the key tiles.  S and do v^T are formed in both:
// seven products instead of five, but no sum crosses CTAs, so nothing is added
// by atomics and equal inputs give equal bits.
//
// Both product kernels are one template.  Two tiles of 128 rows stay in shared
// memory (k and v, or q and do); tiles of 64 rows of the other two stream
// through a ring.  Per streamed tile:
//   S = A1 B1^T, P' = A2 B2^T  (128 x 64 each, TMEM, two buffers)
//   p and ds in registers -> bf16 over S and P' in TMEM
//   acc += p B2 and ds B1 (dk, dv: rows are keys), or ds B1 (dq: rows are queries)
// Eight warps own the elements, four to a buffer, so one buffer's exponentials
// run under the other's products.  bf16 p and ds are the products' operands:
// half a step of each term, of the same size as rounding the result.
#include <cuda_bf16.h>
#include <cstdint>

#include "fl_attn.cuh"

namespace fl {
namespace attn {

constexpr int kBwdThreads = 320;
constexpr int kTmemCols = 512;
constexpr int kColP = 128, kColAcc = 256;   // TMEM: S buffers, P' buffers, accumulators

template <int HD>
struct Bwd {
  static constexpr int kStages = 3;
  static constexpr int kRes = HD / 64 * kTile * 128;       // a resident tile
  static constexpr int kStr = HD / 64 * kBwdTile * 128;    // a streamed tile
  static constexpr int kSmem = 1024 + 2 * kRes + kStages * 2 * kStr + 4 * 4 * kBwdTile * 4 + 256;
};

struct BwdArgs {
  Shape s;
  const float* lse;      // [B, Sq, Hq]
  const float* delta;    // [B, Sq, Hq]
  const Range* ranges;   // [B, q_tiles], tiles of kBwdTile packed rows
  __nv_bfloat16* dq;     // [B, Sq, Hq, D]
  __nv_bfloat16* dk;     // [B, Sk, Hkv, D]
  __nv_bfloat16* dv;
  uint32_t* status;
  int q_tiles;           // of kBwdTile packed rows
  int tiles;             // resident tiles per head
};

struct __align__(16) BwdBars {
  uint64_t a_full;
  uint64_t b_full[3], b_empty[3];
  uint64_t sp_full[2], ds_full[2], acc_done[2];
  uint64_t all_done;
  uint32_t tmem, abort_word;
  int first, last;
};

// delta, and the ranges of the streamed query tiles (the first range_blocks blocks).
__global__ void __launch_bounds__(256) prep_kernel(const Shape s, const __nv_bfloat16* __restrict__ dout,
                                                   int64_t db, int64_t dt, int64_t dh,
                                                   const __nv_bfloat16* __restrict__ out, float* __restrict__ delta,
                                                   Range* __restrict__ ranges, int q_tiles, int range_blocks) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (static_cast<int>(blockIdx.x) < range_blocks) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + warp;
    if (i >= static_cast<int64_t>(q_tiles) * s.B) return;
    const int b = static_cast<int>(i / q_tiles), t = static_cast<int>(i % q_tiles);
    const Range r = tile_range(s, b, t * (kBwdTile >> s.lgp), kBwdTile >> s.lgp);
    if (lane == 0) ranges[i] = r;
    return;
  }
  // 16 lanes to a row, 8 columns to a lane.
  const int64_t row = (static_cast<int64_t>(blockIdx.x - range_blocks) * 256 + threadIdx.x) >> 4;
  const int64_t rows = static_cast<int64_t>(s.B) * s.Sq * s.Hq;
  const int d = (lane & 15) * 8;
  float sum = 0.f;
  if (row < rows && d < s.D) {
    const int h = static_cast<int>(row % s.Hq);
    const int64_t bt = row / s.Hq;
    const int64_t t = bt % s.Sq, b = bt / s.Sq;
    const uint4 x = *reinterpret_cast<const uint4*>(dout + b * db + t * dt + h * dh + d);
    const uint4 y = *reinterpret_cast<const uint4*>(out + row * s.D + d);
    const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum = fmaf(__uint_as_float(xw[i] << 16), __uint_as_float(yw[i] << 16), sum);
      sum = fmaf(__uint_as_float(xw[i] & 0xFFFF0000u), __uint_as_float(yw[i] & 0xFFFF0000u), sum);
    }
  }
#pragma unroll
  for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (row < rows && (lane & 15) == 0) delta[row] = sum;
}

// kDq: rows are packed queries (A1 = q, A2 = do; B1 = k, B2 = v).
// Otherwise rows are keys (A1 = k, A2 = v; B1 = q, B2 = do).
template <int HD, bool kDq, bool kBias>
__global__ void __launch_bounds__(kBwdThreads, 1)
    bwd_kernel(const __grid_constant__ CUtensorMap tm_a1, const __grid_constant__ CUtensorMap tm_a2,
               const __grid_constant__ CUtensorMap tm_b1, const __grid_constant__ CUtensorMap tm_b2,
               const BwdArgs a) {
  using C = Bwd<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* a1 = smem;
  uint8_t* a2 = a1 + C::kRes;
  uint8_t* bs = a2 + C::kRes;                              // kStages x (B1, B2)
  float* info = reinterpret_cast<float*>(bs + C::kStages * 2 * C::kStr);  // [2 groups][2][4][64]
  BwdBars* bars = reinterpret_cast<BwdBars*>(info + 4 * 4 * kBwdTile);
  volatile uint32_t* abort_word = &bars->abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Shape& s = a.s;
  const int G = s.Hq / s.Hkv, pg = 1 << s.lgp;

  // The heaviest tiles of a causal mask first: early keys, late queries.
  const int heads = kDq ? s.Hkv * s.groups : s.Hkv;
  const int per = heads * s.B;
  const int order = static_cast<int>(blockIdx.x) / per;
  const int tile = kDq ? a.tiles - 1 - order : order;
  const int hg = static_cast<int>(blockIdx.x) % per % heads;
  const int b = static_cast<int>(blockIdx.x) % per / heads;
  const int kvh = kDq ? hg / s.groups : hg;
  const int q_step = kBwdTile >> s.lgp;                    // tokens of a streamed query tile
  const int row0 = kDq ? tile * (kTile >> s.lgp) : tile * kTile;

  if (threadIdx.x == 0) {
    mbar_init(&bars->a_full, 1);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&bars->b_full[i], 1);
      mbar_init(&bars->b_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->sp_full[i], 1);
      mbar_init(&bars->ds_full[i], 4);
      mbar_init(&bars->acc_done[i], 1);
    }
    mbar_init(&bars->all_done, 1);
    bars->abort_word = 0;
    bars->first = kNone;
    bars->last = -1;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;

  // What to walk: `n` steps; dq: key tiles from `first`; else the head groups'
  // query tiles `first` .. `first + per_group - 1` (those between that see none
  // of the keys add nothing).
  Range mine{};
  int first = 0, n = 0, per_group = 0;
  if constexpr (kDq) {
    mine = tile_range(s, b, row0, kTile >> s.lgp);
    if (mine.min_lo < mine.max_hi) {
      first = mine.min_lo / kBwdTile;
      n = (mine.max_hi + kBwdTile - 1) / kBwdTile - first;
    }
  } else {
    int lo = kNone, hi = -1;
    for (int i = threadIdx.x; i < a.q_tiles; i += kBwdThreads) {
      const Range r = a.ranges[static_cast<int64_t>(b) * a.q_tiles + i];
      if (r.min_lo < row0 + kTile && r.max_hi > row0) {
        lo = min(lo, i);
        hi = i;
      }
    }
    if (hi >= 0) {
      atomicMin(&bars->first, lo);
      atomicMax(&bars->last, hi);
    }
    __syncthreads();
    first = bars->first;
    per_group = bars->last >= 0 ? bars->last - first + 1 : 0;
    n = per_group * s.groups;
  }

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      tma_prefetch_desc(&tm_a1);
      tma_prefetch_desc(&tm_a2);
      tma_prefetch_desc(&tm_b1);
      tma_prefetch_desc(&tm_b2);
      const int ah = kDq ? hg << s.lgp : kvh;
      mbar_arrive_expect_tx(&bars->a_full, 2 * C::kRes);
      for (int c = 0; c < HD / 64; ++c) {
        tma_load_4d(a1 + c * kTile * 128, &tm_a1, 64 * c, ah, row0, b, &bars->a_full);
        tma_load_4d(a2 + c * kTile * 128, &tm_a2, 64 * c, ah, row0, b, &bars->a_full);
      }
      int i = 0;
      for (; i < n; ++i) {
        const int st = i % C::kStages;
        if (i >= C::kStages && !mbar_wait(&bars->b_empty[st], (i / C::kStages - 1) & 1, abort_word, a.status,
                                          kStatusTimeoutEmpty))
          break;
        int bh, br;
        if constexpr (kDq) {
          bh = kvh;
          br = (first + i) * kBwdTile;
        } else {
          bh = kvh * G + (i / per_group) * pg;
          br = (first + i % per_group) * q_step;
        }
        uint8_t* b1 = bs + st * 2 * C::kStr;
        mbar_arrive_expect_tx(&bars->b_full[st], 2 * C::kStr);
        for (int c = 0; c < HD / 64; ++c) {
          tma_load_4d(b1 + c * kBwdTile * 128, &tm_b1, 64 * c, bh, br, b, &bars->b_full[st]);
          tma_load_4d(b1 + C::kStr + c * kBwdTile * 128, &tm_b2, 64 * c, bh, br, b, &bars->b_full[st]);
        }
      }
      // No copy may be in flight when the CTA leaves.
      uint32_t none = 0;
      mbar_wait(&bars->a_full, 0, &none, a.status, kStatusTimeoutDrain);
      for (int j = max(i - C::kStages, 0); j < i; ++j)
        mbar_wait(&bars->b_full[j % C::kStages], (j / C::kStages) & 1, &none, a.status, kStatusTimeoutDrain);
    }
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      const uint32_t id_s = idesc_bf16_f32(kTile, kBwdTile), id_acc = idesc_bf16_f32_bmn(kTile, HD);
      bool ok = mbar_wait(&bars->a_full, 0, abort_word, a.status, kStatusTimeoutFull);
      // S and P' of step i into buffer i & 1, once the products that read the
      // buffer's p and ds are done.
      auto scores = [&](int i) -> bool {
        const int st = i % C::kStages;
        if (i >= 2 && !mbar_wait(&bars->acc_done[i & 1], ((i >> 1) - 1) & 1, abort_word, a.status, kStatusTimeoutAccum))
          return false;
        if (!mbar_wait(&bars->b_full[st], (i / C::kStages) & 1, abort_word, a.status, kStatusTimeoutFull)) return false;
        tc_fence_after();
        const uint32_t b1 = smem_u32(bs + st * 2 * C::kStr);
        mma_rows<HD>(tmem + kBwdTile * (i & 1), smem_u32(a1), b1, kBwdTile, id_s);
        mma_rows<HD>(tmem + kColP + kBwdTile * (i & 1), smem_u32(a2), b1 + C::kStr, kBwdTile, id_s);
        tc_commit(&bars->sp_full[i & 1]);
        return true;
      };
      ok = ok && scores(0);
      for (int i = 0; i < n && ok; ++i) {
        if (i + 1 < n && !scores(i + 1)) break;
        if (!mbar_wait(&bars->ds_full[i & 1], (i >> 1) & 1, abort_word, a.status, kStatusTimeoutFull)) break;
        tc_fence_after();
        const int st = i % C::kStages;
        const uint32_t b1 = smem_u32(bs + st * 2 * C::kStr);
        if constexpr (kDq) {
          mma_cols<HD, kBwdTile>(tmem + kColAcc, tmem + kColP + kBwdTile * (i & 1), b1, id_acc, i > 0);
        } else {
          mma_cols<HD, kBwdTile>(tmem + kColAcc, tmem + kBwdTile * (i & 1), b1 + C::kStr, id_acc, i > 0);
          mma_cols<HD, kBwdTile>(tmem + kColAcc + HD, tmem + kColP + kBwdTile * (i & 1), b1, id_acc, i > 0);
        }
        tc_commit(&bars->b_empty[st]);
        tc_commit(&bars->acc_done[i & 1]);
      }
      // Completes after every product issued above, also after a wait that gave up.
      tc_commit(&bars->all_done);
      uint32_t none = 0;
      mbar_wait(&bars->all_done, 0, &none, a.status, kStatusTimeoutDrain);
    }
  } else {
    const int group = (warp - 2) >> 2;             // the buffer (step parity) this warp serves
    const int quarter = warp & 3, tid = (threadIdx.x - 64) & 127;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int row = quarter * 32 + lane;           // TMEM lane: the element row this thread owns
    float* my_info = info + group * 2 * 4 * kBwdTile;
    // dq: the row's token, head, range and statistics; else the row's key.
    int tok = 0, head = 0, lo = 0, hi = 0;
    float lse2 = INFINITY, delta = 0.f;
    const int key = row0 + row;
    if constexpr (kDq) {
      tok = row0 + (row >> s.lgp);
      head = (hg << s.lgp) + (row & (pg - 1));
      if (tok < s.Sq) {
        row_range(s, b, tok, lo, hi);
        const int64_t at = (static_cast<int64_t>(b) * s.Sq + tok) * s.Hq + head;
        lse2 = a.lse[at] * kLog2e;
        delta = a.delta[at];
      }
    }
    const float row_slope2 = kDq && kBias && s.slopes ? s.slopes[head] * kLog2e : 0.f;
    bool ok = true;
    for (int i = group; i < n; i += 2) {
      float* buf = my_info + ((i >> 1) & 1) * 4 * kBwdTile;
      bool whole;
      int col0, h_first = 0;                       // dq: first key; else first token and head
      if constexpr (kDq) {
        col0 = (first + i) * kBwdTile;
        whole = mine.max_lo <= col0 && mine.min_hi >= col0 + kBwdTile;
      } else {
        const int t = first + i % per_group;
        col0 = t * q_step;
        h_first = kvh * G + (i / per_group) * pg;
        const Range r = a.ranges[static_cast<int64_t>(b) * a.q_tiles + t];
        whole = r.max_lo <= row0 && r.min_hi >= row0 + kTile;
        // The columns' statistics and ranges, for all rows, through shared memory.
        const int c = tid & (kBwdTile - 1), ct = col0 + (c >> s.lgp);
        if (tid < kBwdTile) {
          float x = INFINITY, y = 0.f;             // a column past the sequence: p = 0
          if (ct < s.Sq) {
            const int64_t at = (static_cast<int64_t>(b) * s.Sq + ct) * s.Hq + h_first + (c & (pg - 1));
            x = a.lse[at] * kLog2e;
            y = a.delta[at];
          }
          buf[c] = x;
          buf[kBwdTile + c] = y;
        } else {
          int l = 0, h = 0;
          if (ct < s.Sq) row_range(s, b, ct, l, h);
          buf[2 * kBwdTile + c] = __int_as_float(l);
          buf[3 * kBwdTile + c] = __int_as_float(h);
        }
        named_barrier_sync(1 + group, 128);
      }
      if (ok && !mbar_wait_warp(&bars->sp_full[group], (i >> 1) & 1, abort_word, a.status, kStatusTimeoutAccum))
        ok = false;
      if (!ok) {
        if constexpr (kDq) break;
        continue;                                  // the group's other warps count on the barrier
      }
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < kBwdTile; c += 32) {
        uint32_t sv[32], pv[32], w[16];
        tmem_ld_32x32b_x32(tmem + kBwdTile * group + lanes + c, sv);
        tmem_ld_32x32b_x32(tmem + kColP + kBwdTile * group + lanes + c, pv);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 32; q += 4) {
          float l4[4], d4[4];
          int lo4[4], hi4[4];
          if constexpr (kDq) {
#pragma unroll
            for (int e = 0; e < 4; ++e) l4[e] = lse2, d4[e] = delta, lo4[e] = lo, hi4[e] = hi;
          } else {
            const float4 x = *reinterpret_cast<const float4*>(buf + c + q);
            const float4 y = *reinterpret_cast<const float4*>(buf + kBwdTile + c + q);
            l4[0] = x.x, l4[1] = x.y, l4[2] = x.z, l4[3] = x.w;
            d4[0] = y.x, d4[1] = y.y, d4[2] = y.z, d4[3] = y.w;
            if (!whole) {
              const int4 u = *reinterpret_cast<const int4*>(buf + 2 * kBwdTile + c + q);
              const int4 v = *reinterpret_cast<const int4*>(buf + 3 * kBwdTile + c + q);
              lo4[0] = u.x, lo4[1] = u.y, lo4[2] = u.z, lo4[3] = u.w;
              hi4[0] = v.x, hi4[1] = v.y, hi4[2] = v.z, hi4[3] = v.w;
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int col = c + q + e;
            const int k_at = kDq ? col0 + col : key;
            float p, ds, th = 0.f;
            if constexpr (kBias) {
              const int at = kDq ? tok : col0 + (col >> s.lgp);
              const float slope2 =
                  kDq ? row_slope2 : (s.slopes ? s.slopes[h_first + (col & (pg - 1))] * kLog2e : 0.f);
              p = ex2(score2(s, __uint_as_float(sv[q + e]), slope2, at + s.Sk - s.Sq - k_at, th) - l4[e]);
            } else {
              p = ex2(fmaf(__uint_as_float(sv[q + e]), s.sl2, -l4[e]));
            }
            ds = p * (__uint_as_float(pv[q + e]) - d4[e]);
            if constexpr (kBias) ds *= 1.0f - th * th;
            if (!whole && (k_at < lo4[e] || k_at >= hi4[e])) p = ds = 0.f;
            sv[q + e] = __float_as_uint(p);
            pv[q + e] = __float_as_uint(ds);
          }
        }
        if constexpr (!kDq) {
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack_bf16x2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1]));
          tmem_st_32x32b_x16(tmem + kBwdTile * group + lanes + c / 2, w);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = pack_bf16x2(__uint_as_float(pv[2 * e]), __uint_as_float(pv[2 * e + 1]));
        tmem_st_32x32b_x16(tmem + kColP + kBwdTile * group + lanes + c / 2, w);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->ds_full[group]);
    }
    if (n > 0 && !mbar_wait_warp(&bars->all_done, 0, abort_word, a.status, kStatusTimeoutAccum)) ok = false;
    tc_fence_after();
    if (ok) {
      // dq: each group stores half of the columns; else one stores dv, one dk.
      const bool live = kDq ? tok < s.Sq : key < s.Sk;
      __nv_bfloat16* o;
      if constexpr (kDq)
        o = a.dq + ((static_cast<int64_t>(b) * s.Sq + tok) * s.Hq + head) * s.D;
      else
        o = (group ? a.dk : a.dv) + ((static_cast<int64_t>(b) * s.Sk + key) * s.Hkv + kvh) * s.D;
      const float by = kDq || group ? s.scale : 1.0f;
      const int c_from = kDq ? group * (HD / 2) : 0, c_to = kDq ? c_from + HD / 2 : HD;
#pragma unroll 1
      for (int c = c_from; c < c_to; c += 32) {
        uint32_t v[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(tmem + kColAcc + (kDq ? 0 : group * HD) + lanes + c, v);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0u;
        }
        if (!live) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + 8 * e < s.D) {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              w[q] = pack_bf16x2(__uint_as_float(v[8 * e + 2 * q]) * by, __uint_as_float(v[8 * e + 2 * q + 1]) * by);
            *reinterpret_cast<uint4*>(o + c + 8 * e) = make_uint4(w[0], w[1], w[2], w[3]);
          }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <int HD, bool kDq, bool kBias>
int launch_bwd(const CUtensorMap& a1, const CUtensorMap& a2, const CUtensorMap& b1, const CUtensorMap& b2,
               const BwdArgs& a, int64_t grid, cudaStream_t stream) {
  int rc = allow_smem(reinterpret_cast<const void*>(&bwd_kernel<HD, kDq, kBias>), Bwd<HD>::kSmem);
  if (rc) return rc;
  bwd_kernel<HD, kDq, kBias><<<static_cast<unsigned>(grid), kBwdThreads, Bwd<HD>::kSmem, stream>>>(a1, a2, b1, b2, a);
  return FL_OK;
}

size_t a256(size_t n) { return (n + 255) / 256 * 256; }

int64_t q_tiles_of(int64_t Sq, int lgp) { return (Sq + (kBwdTile >> lgp) - 1) / (kBwdTile >> lgp); }

}  // namespace attn
}  // namespace fl

using namespace fl;

extern "C" {

// delta [B, Sq, Hq] fp32, then the ranges of the query tiles.
size_t fl_attn_bwd_workspace_bytes(int64_t B, int64_t Sq, int Hq, int Hkv) {
  if (B <= 0 || Sq <= 0 || Hq < 1 || Hkv < 1 || Hq % Hkv) return 0;
  return attn::a256(static_cast<size_t>(B) * Sq * Hq * sizeof(float)) +
         static_cast<size_t>(B) * attn::q_tiles_of(Sq, attn::packed_log2(Hq, Hkv)) * sizeof(attn::Range);
}

int fl_attn_bwd(const uint16_t* dout, const uint16_t* q, const uint16_t* k, const uint16_t* v, const int64_t* strides,
                const uint16_t* out, const float* lse, int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int D,
                const int32_t* begin, const int32_t* end, float scale, float softcap, const float* slopes,
                uint16_t* dq, uint16_t* dk, uint16_t* dv, void* workspace, size_t workspace_bytes, void* stream) {
  const void* bases[4] = {q, k, v, dout};
  int rc = attn_check("fl_attn_bwd", B, Sq, Sk, Hq, Hkv, D, strides, 4, bases, begin, end, scale, softcap);
  if (rc || B == 0) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t kv_bytes = static_cast<size_t>(B) * Sk * Hkv * D * 2;
  if (Sq && (!dq || !out || !lse || (reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(out)) & 15u))
    return set_error(FL_ERR_ARG, "fl_attn_bwd: out, lse and dq must be given, 16-byte aligned");
  if (Sk && (!dk || !dv || (reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv)) & 15u))
    return set_error(FL_ERR_ARG, "fl_attn_bwd: dk and dv must be given, 16-byte aligned");
  if (Sq == 0) {
    if (kv_bytes && (cudaMemsetAsync(dk, 0, kv_bytes, st) != cudaSuccess || cudaMemsetAsync(dv, 0, kv_bytes, st) != cudaSuccess))
      return set_error(FL_ERR_CUDA, "fl_attn_bwd: clearing dk and dv failed");
    return FL_OK;
  }
  if (Sk == 0) {
    if (cudaMemsetAsync(dq, 0, static_cast<size_t>(B) * Sq * Hq * D * 2, st) != cudaSuccess)
      return set_error(FL_ERR_CUDA, "fl_attn_bwd: clearing dq failed");
    return FL_OK;
  }
  if (!workspace || workspace_bytes < fl_attn_bwd_workspace_bytes(B, Sq, Hq, Hkv) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15u))
    return set_error(FL_ERR_ARG, "fl_attn_bwd: workspace missing, short or not 16-byte aligned");
  attn::BwdArgs a{};
  attn::fill_shape(a.s, (int)B, (int)Sq, (int)Sk, Hq, Hkv, D, begin, end, scale, softcap, slopes);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || !(a.status = status_word(dev)))
    return set_error(FL_ERR_CUDA, "fl_attn_bwd: status word unavailable");
  const int64_t rows = B * Sq * Hq;
  float* delta = static_cast<float*>(workspace);
  auto* ranges = reinterpret_cast<attn::Range*>(static_cast<uint8_t*>(workspace) + attn::a256(rows * sizeof(float)));
  a.lse = lse;
  a.delta = delta;
  a.ranges = ranges;
  a.dq = reinterpret_cast<__nv_bfloat16*>(dq);
  a.dk = reinterpret_cast<__nv_bfloat16*>(dk);
  a.dv = reinterpret_cast<__nv_bfloat16*>(dv);
  a.q_tiles = static_cast<int>(attn::q_tiles_of(Sq, a.s.lgp));
  const int pg = 1 << a.s.lgp, q_rows = attn::kTile >> a.s.lgp, q_step = attn::kBwdTile >> a.s.lgp;
  const int64_t key_tiles = (Sk + attn::kTile - 1) / attn::kTile;
  if (key_tiles * B * Hkv > (int64_t(1) << 30)) return set_error(FL_ERR_ARG, "fl_attn_bwd: too many key tiles");

  const int64_t range_blocks = (static_cast<int64_t>(a.q_tiles) * B + 7) / 8, delta_blocks = (rows * 16 + 255) / 256;
  attn::prep_kernel<<<static_cast<unsigned>(range_blocks + delta_blocks), 256, 0, st>>>(
      a.s, reinterpret_cast<const __nv_bfloat16*>(dout), strides[9], strides[10], strides[11],
      reinterpret_cast<const __nv_bfloat16*>(out), delta, ranges, a.q_tiles, static_cast<int>(range_blocks));

  // Resident (128 rows) and streamed (64 rows) maps of each tensor.
  CUtensorMap q_res, do_res, k_res, v_res, q_str, do_str, k_str, v_str;
  const int b = (int)B, sq = (int)Sq, sk = (int)Sk;
  auto rows_map = [&](CUtensorMap* m, const void* p, const int64_t* s, int tokens) {
    return attn_map(m, p, s[0], s[1], s[2], b, sq, Hq, D, pg, tokens);
  };
  auto keys_map = [&](CUtensorMap* m, const void* p, const int64_t* s, int tokens) {
    return attn_map(m, p, s[0], s[1], s[2], b, sk, Hkv, D, 1, tokens);
  };
  if ((rc = rows_map(&q_res, q, strides, q_rows)) || (rc = rows_map(&do_res, dout, strides + 9, q_rows)) ||
      (rc = rows_map(&q_str, q, strides, q_step)) || (rc = rows_map(&do_str, dout, strides + 9, q_step)) ||
      (rc = keys_map(&k_res, k, strides + 3, attn::kTile)) || (rc = keys_map(&v_res, v, strides + 6, attn::kTile)) ||
      (rc = keys_map(&k_str, k, strides + 3, attn::kBwdTile)) || (rc = keys_map(&v_str, v, strides + 6, attn::kBwdTile)))
    return rc;
  const bool bias = softcap != 0.f || slopes;
  a.tiles = static_cast<int>(key_tiles);
  const int64_t kv_grid = key_tiles * B * Hkv;
  rc = D <= 64 ? (bias ? attn::launch_bwd<64, false, true>(k_res, v_res, q_str, do_str, a, kv_grid, st)
                       : attn::launch_bwd<64, false, false>(k_res, v_res, q_str, do_str, a, kv_grid, st))
               : (bias ? attn::launch_bwd<128, false, true>(k_res, v_res, q_str, do_str, a, kv_grid, st)
                       : attn::launch_bwd<128, false, false>(k_res, v_res, q_str, do_str, a, kv_grid, st));
  if (rc) return rc;
  const int64_t q_grid = attn::fwd_ctas(b, sq, Hq, Hkv);
  a.tiles = static_cast<int>(q_grid / B / (Hq >> a.s.lgp));
  rc = D <= 64 ? (bias ? attn::launch_bwd<64, true, true>(q_res, do_res, k_str, v_str, a, q_grid, st)
                       : attn::launch_bwd<64, true, false>(q_res, do_res, k_str, v_str, a, q_grid, st))
               : (bias ? attn::launch_bwd<128, true, true>(q_res, do_res, k_str, v_str, a, q_grid, st)
                       : attn::launch_bwd<128, true, false>(q_res, do_res, k_str, v_str, a, q_grid, st));
  if (rc) return rc;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FL_ERR_CUDA, "fl_attn_bwd: %s", cudaGetErrorString(e));
  return FL_OK;
}

}  // extern "C"
