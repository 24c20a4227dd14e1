// Attention backward over row ranges (see fl_attn.cuh for the formulas).
//
//   delta_i = sum_j p_ij dp_ij,  dp = do v^T,  p = 2^(x - lse),
//   ds = p f (dp - delta),  f = 1 - tanh^2 under a cap, else 1
//   dv = p^T do,  dk = scale ds^T q,  dq = scale ds k
//
// Two launches: dq, a CTA per 128 (packed) query rows, walking the key tiles;
// then dk and dv, a CTA per 128 keys of a key/value head, walking the query
// tiles of its whole head group (so the group's sum stays in one accumulator).
// S and dp are formed in both: more products than one kernel would need, but no
// sum crosses CTAs, so nothing is added by atomics and equal inputs give equal
// bits.
//
// delta is known only once a row's keys have been walked.  do . o is delta up
// to the rounding of o, which is too far off for rows with few keys: there p
// (dp - delta) is a small difference.  So the dq kernel works with d0 = do . o,
// sums delta in FP32 beside it, and corrects at the end:
//   dq = scale (sum p f (dp - d0) k - (delta - d0) sum p f k),
// the last sum being one more product over operands that are there already
// (delta - d0 is small, so its bf16 operands are exact enough).  The dk/dv
// kernel gets the summed delta.
//
// Both are one template.  Two tiles of 128 rows stay in shared memory (q and
// do, or k and v); tiles of 64 rows of the other two stream through a ring.
// Per streamed tile:
//   S = A1 B1^T, P' = A2 B2^T  (128 x 64 each, TMEM, two buffers)
//   p and ds in registers -> bf16 over S and P' in TMEM
//   acc += ds B1 and p f B1 (dq) or p B2 (dk, dv)
// Eight warps own the elements, four to a buffer, so one buffer's exponentials
// run under the other's products.  bf16 p and ds are the products' operands:
// half a step of each term, of the same size as rounding the result.
#include <cuda_bf16.h>
#include <cstdint>
#include <type_traits>

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
  const __nv_bfloat16* out;   // [B, Sq, Hq, D]
  const __nv_bfloat16* dout;  // strided
  int64_t do_batch, do_token, do_head;
  const float* lse;      // [B, Sq, Hq]
  float* delta;          // [B, Sq, Hq]: written by the dq kernel, read by the other
  Range* ranges;         // [B, q_tiles], tiles of kBwdTile packed rows: likewise
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

// Dot product of two rows of D bf16 values (D a multiple of 8, 16-byte aligned).
__device__ __forceinline__ float row_dot(const __nv_bfloat16* x, const __nv_bfloat16* y, int D) {
  float sum = 0.f;
  for (int d = 0; d < D; d += 8) {
    const uint4 a = *reinterpret_cast<const uint4*>(x + d), b = *reinterpret_cast<const uint4*>(y + d);
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum = fmaf(__uint_as_float(aw[i] << 16), __uint_as_float(bw[i] << 16), sum);
      sum = fmaf(__uint_as_float(aw[i] & 0xFFFF0000u), __uint_as_float(bw[i] & 0xFFFF0000u), sum);
    }
  }
  return sum;
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
        mma_cols<HD, kBwdTile>(tmem + kColAcc, tmem + kBwdTile * (i & 1), kDq ? b1 : b1 + C::kStr, id_acc, i > 0);
        mma_cols<HD, kBwdTile>(tmem + kColAcc + HD, tmem + kColP + kBwdTile * (i & 1), b1, id_acc, i > 0);
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
    float lse2 = INFINITY, d0 = 0.f;
    uint64_t dsum2 = 0;                            // (0, 0)
    const uint64_t sl2_2 = pair(s.sl2, s.sl2);
    const int key = row0 + row;
    if constexpr (kDq) {
      tok = row0 + (row >> s.lgp);
      head = (hg << s.lgp) + (row & (pg - 1));
      if (tok < s.Sq) {
        row_range(s, b, tok, lo, hi);
        const int64_t at = (static_cast<int64_t>(b) * s.Sq + tok) * s.Hq + head;
        lse2 = a.lse[at] * kLog2e;
        d0 = row_dot(a.dout + b * a.do_batch + tok * a.do_token + head * a.do_head, a.out + at * s.D, s.D);
      }
      // The ranges of this tile's two streamed tiles, for the dk/dv kernel.
      if (hg == 0 && quarter == 0) {
        const int t = 2 * tile + group;
        const Range r = tile_range(s, b, t * q_step, q_step);
        if (lane == 0 && t < a.q_tiles) a.ranges[static_cast<int64_t>(b) * a.q_tiles + t] = r;
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
          float x = -INFINITY, y = 0.f;            // a column past the sequence: p = 0
          if (ct < s.Sq) {
            const int64_t at = (static_cast<int64_t>(b) * s.Sq + ct) * s.Hq + h_first + (c & (pg - 1));
            x = -a.lse[at] * kLog2e;
            y = -a.delta[at];
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
      const uint32_t at_s = tmem + kBwdTile * group + lanes, at_p = at_s + kColP;
      uint32_t sv[kBwdTile], pv[kBwdTile];
#pragma unroll
      for (int c = 0; c < kBwdTile; c += 32) {
        tmem_ld_32x32b_x32(at_s + c, reinterpret_cast<uint32_t(&)[32]>(sv[c]));
        tmem_ld_32x32b_x32(at_p + c, reinterpret_cast<uint32_t(&)[32]>(pv[c]));
      }
      tmem_wait_ld();
      // Columns c .. c + 3 of the row: p (dq: p f) into sv, ds into pv.
      auto four = [&](int c, auto masked) {
        uint64_t nl[2], nd[2];                     // -lse2 and -delta of the columns
        if constexpr (kDq) {
          nl[0] = nl[1] = pair(-lse2, -lse2);
          nd[0] = nd[1] = pair(-d0, -d0);
        } else {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(buf + c);
          const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(buf + kBwdTile + c);
          nl[0] = x.x, nl[1] = x.y;
          nd[0] = y.x, nd[1] = y.y;
        }
        bool hide[4] = {};
        if constexpr (decltype(masked)::value) {
          if constexpr (kDq) {
#pragma unroll
            for (int e = 0; e < 4; ++e) hide[e] = c + e < lo - col0 || c + e >= hi - col0;
          } else {
            const int4 u = *reinterpret_cast<const int4*>(buf + 2 * kBwdTile + c);
            const int4 v = *reinterpret_cast<const int4*>(buf + 3 * kBwdTile + c);
            hide[0] = key < u.x || key >= v.x;
            hide[1] = key < u.y || key >= v.y;
            hide[2] = key < u.z || key >= v.z;
            hide[3] = key < u.w || key >= v.w;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = c + 2 * h;
          float p[2];
          [[maybe_unused]] float f[2];
          if constexpr (kBias) {
            float l[2];
            unpair(nl[h], l[0], l[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = i + e;
              const int at = kDq ? tok : col0 + (col >> s.lgp), k_at = kDq ? col0 + col : key;
              const float slope2 =
                  kDq ? row_slope2 : (s.slopes ? s.slopes[h_first + (col & (pg - 1))] * kLog2e : 0.f);
              float th;
              p[e] = ex2(score2(s, __uint_as_float(sv[col]), slope2, at + s.Sk - s.Sq - k_at, th) + l[e]);
              f[e] = 1.0f - th * th;
            }
          } else {
            unpair(fma2(pair(sv[i], sv[i + 1]), sl2_2, nl[h]), p[0], p[1]);
            p[0] = ex2(p[0]);
            p[1] = ex2(p[1]);
          }
          if constexpr (decltype(masked)::value) {
            if (hide[2 * h]) p[0] = 0.f;
            if (hide[2 * h + 1]) p[1] = 0.f;
          }
          const uint64_t dp = pair(pv[i], pv[i + 1]);
          uint64_t pp = pair(p[0], p[1]);
          if constexpr (kDq) {
            if constexpr (decltype(masked)::value) {
              // 0 times whatever a hidden key's value makes of dp
              float x, y;
              unpair(mul2(pp, dp), x, y);
              dsum2 = add2(dsum2, pair(hide[2 * h] ? 0.f : x, hide[2 * h + 1] ? 0.f : y));
            } else {
              dsum2 = fma2(pp, dp, dsum2);
            }
          }
          uint64_t pf = pp;
          if constexpr (kBias) pf = mul2(pp, pair(f[0], f[1]));
          float ds[2];
          unpair(mul2(pf, add2(dp, nd[h])), ds[0], ds[1]);
          if constexpr (decltype(masked)::value) {
            if (hide[2 * h]) ds[0] = 0.f;
            if (hide[2 * h + 1]) ds[1] = 0.f;
          }
          float a0, a1;
          unpair(kDq ? pf : pp, a0, a1);
          sv[i / 2] = pack_bf16x2(a0, a1);
          pv[i / 2] = pack_bf16x2(ds[0], ds[1]);
        }
      };
      if (whole) {
#pragma unroll
        for (int c = 0; c < kBwdTile; c += 4) four(c, std::false_type{});
      } else {
#pragma unroll
        for (int c = 0; c < kBwdTile; c += 4) four(c, std::true_type{});
      }
      tmem_st_32x32b_x32(at_s, reinterpret_cast<uint32_t(&)[32]>(sv[0]));
      tmem_st_32x32b_x32(at_p, reinterpret_cast<uint32_t(&)[32]>(pv[0]));
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->ds_full[group]);
    }
    float fix = 0.f;
    if constexpr (kDq) {
      // Each group summed delta over its half of the key tiles.
      float dsum, odd;
      unpair(dsum2, dsum, odd);
      info[group * kTile + row] = dsum + odd;
      named_barrier_sync(1, 256);
      dsum = info[row] + info[kTile + row];
      fix = d0 - dsum;
      if (group == 0 && tok < s.Sq) a.delta[(static_cast<int64_t>(b) * s.Sq + tok) * s.Hq + head] = dsum;
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
          tmem_ld_32x32b_x32(tmem + kColAcc + (kDq || group ? HD : 0) + lanes + c, v);
          if constexpr (kDq) {
            uint32_t u[32];
            tmem_ld_32x32b_x32(tmem + kColAcc + lanes + c, u);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              v[e] = __float_as_uint(fmaf(fix, __uint_as_float(u[e]), __uint_as_float(v[e])));
          } else {
            tmem_wait_ld();
          }
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
  a.out = reinterpret_cast<const __nv_bfloat16*>(out);
  a.dout = reinterpret_cast<const __nv_bfloat16*>(dout);
  a.do_batch = strides[9];
  a.do_token = strides[10];
  a.do_head = strides[11];
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
  const int64_t q_grid = attn::fwd_ctas(b, sq, Hq, Hkv);
  a.tiles = static_cast<int>(q_grid / B / (Hq >> a.s.lgp));
  rc = D <= 64 ? (bias ? attn::launch_bwd<64, true, true>(q_res, do_res, k_str, v_str, a, q_grid, st)
                       : attn::launch_bwd<64, true, false>(q_res, do_res, k_str, v_str, a, q_grid, st))
               : (bias ? attn::launch_bwd<128, true, true>(q_res, do_res, k_str, v_str, a, q_grid, st)
                       : attn::launch_bwd<128, true, false>(q_res, do_res, k_str, v_str, a, q_grid, st));
  if (rc) return rc;
  a.tiles = static_cast<int>(key_tiles);
  const int64_t kv_grid = key_tiles * B * Hkv;
  rc = D <= 64 ? (bias ? attn::launch_bwd<64, false, true>(k_res, v_res, q_str, do_str, a, kv_grid, st)
                       : attn::launch_bwd<64, false, false>(k_res, v_res, q_str, do_str, a, kv_grid, st))
               : (bias ? attn::launch_bwd<128, false, true>(k_res, v_res, q_str, do_str, a, kv_grid, st)
                       : attn::launch_bwd<128, false, false>(k_res, v_res, q_str, do_str, a, kv_grid, st));
  if (rc) return rc;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FL_ERR_CUDA, "fl_attn_bwd: %s", cudaGetErrorString(e));
  return FL_OK;
}

}  // extern "C"
