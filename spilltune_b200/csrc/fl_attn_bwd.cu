// Attention backward over row ranges (see fl_attn.cuh for the formulas).
//
//   delta_i = sum_j p_ij dp_ij,  dp = do v^T,  p = 2^(x - lse),
//   ds = p f (dp - delta),  f = 1 - tanh^2 under a cap, else 1
//   dv = p^T do,  dk = scale ds^T q,  dq = scale ds k
//
// Two launches: dq, an item per 128 (packed) query rows, walking the key tiles;
// then dk and dv, an item per 128 keys of a key/value head, walking the query
// tiles of its whole head group (so the group's sum stays in one accumulator).
// S and dp are formed in both: eight products where one kernel would form five,
// but no sum crosses CTAs, so nothing is added by atomics and equal inputs give
// equal bits.  Where the key tiles would leave half the SMs idle, several items
// share a walk and a third launch adds their FP32 sums in order.
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
// do, or k and v); tiles of 128 rows of the other two stream through a ring.
// Per streamed tile:
//   S = A1 B1^T, P' = A2 B2^T  (128 x 128 each, TMEM)
//   p and ds in registers -> bf16 over S and P' in TMEM
//   acc1 += p f B1 (dq) or p B2 (dv);  acc2 += ds B1 (dq, dk)
// S, P' and the accumulators fill TMEM, so nothing is double-buffered; the order
// acc1(i), S(i + 1), acc2(i), P'(i + 1) keeps the tensor cores on one pair while
// the sixteen element warps (four to each 32 columns) work on the other.  What
// bounds a step is that chain: over 4 x 2048 causal tokens, 32/8 heads of 128, a
// step takes 2.3 us in dq and 2.0 us in dk/dv, the ends of the walks included, where
// its four products take 2048 cycles (1.1 us).
// * Products are 128 columns wide: with 64, the fetch of the resident operand
//   makes a product take 48 cycles where 32 would do (measured back to back).
// * One elected lane of a warp that walks as one issues them: a divergent lane's
//   operands went through vector registers, 120 cycles from one product to the
//   next beside busy element warps (dq 391 -> 321 us).
// * A quarter of the exponentials (half under a cap, whose tanh takes two more
//   results) run on the FMA pipes.
// * The columns' statistics come with their tile by a bulk copy, left in that
//   form by the dq kernel; fetched by the element warps they cost 1000 cycles a
//   step.
// * CTAs are persistent: the next item's loads, scores and products start while
//   the last one's results are stored.
// * The second product of a pair starts when half of its operand is there (16 of
//   a group's 32 columns): dk/dv 296 -> 279 us, 262 -> 223 us where documents
//   make short walks; no gain for dq.
// * Shared memory is declared aligned, not aligned by hand: a pointer that went
//   through an integer is generic to the compiler (64-bit, and its accesses
//   slower), and 96 registers had no room for that: dk/dv 278 -> 235 us; the
//   128-wide forms without slopes no longer spill (others store up to 56 bytes,
//   with operands in two parts up to 96).  The slack saved lets dq keep a third key
//   tile (303 -> 280 us).
// Measured at 4 x 2048 causal tokens, 32/8 heads of 128, in short runs: dq 266 us,
// dk/dv 236 us (five products at 685 TFLOP/s; the eight that run at 1096, 66% of the
// burst rate of a bf16 GEMM); both together 594 us kept up for seconds, at the power cap.
// bf16 p and ds are the products' operands: half a step of each term, of the
// same size as rounding the result; in two parts in small calls (few_results).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

#include "fl_attn.cuh"

namespace fl {
namespace attn {

constexpr int kGroups = 4;                  // groups of four element warps
constexpr int kCols = kTile / kGroups;      // columns of a tile that one group owns
constexpr int kBwdThreads = 64 + 128 * kGroups;
constexpr int kTmemCols = 512;
constexpr int kColP = 128, kColAcc = 256;   // TMEM: S, P', the two accumulators

// What the dk/dv kernel needs of 128 packed query rows, left by the dq kernel
// and loaded with the tile: -lse log2(e), -delta (over kCapSlope under a cap,
// as dp there), begin and end of each row,
// then {max begin, min end} of each kCols rows inside the sequence.  Rows
// past the sequence get a first entry of -inf, which makes p 0, and the range
// (-1, -1); of no rows inside the sequence, max begin is kNone - 1.
struct __align__(16) RowInfo {
  float nlse2[kTile], ndelta[kTile];
  int lo[kTile], hi[kTile];
  float slope2[kTile];             // with slopes: of the row's head, times log2(e)
  int max_lo[kGroups], min_hi[kGroups];
};
constexpr int kInfoBytes = sizeof(RowInfo);

template <int HD, bool kDq>
struct Bwd {
  // Of B1 and B2.  dq has no row infos to keep (but sums, and dots of do and o),
  // which leaves room for a third tile of keys: all 227 KB of an SM.
  static constexpr int kStages[2] = {kDq ? 3 : 2, 2};
  static constexpr int kBytes = HD / 64 * kTile * 128;     // a tile of 128 rows
  static constexpr int kExtra = kDq ? (kGroups + 1) * kTile * static_cast<int>(sizeof(float)) : 2 * kInfoBytes;
  static constexpr int kSmem = (2 + kStages[0] + kStages[1]) * kBytes + kExtra + 512;
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

struct BwdArgs {
  Shape s;
  const __nv_bfloat16* out;   // [B, Sq, Hq, D]
  const __nv_bfloat16* dout;  // strided
  int64_t do_batch, do_token, do_head;
  const float* lse;      // [B, Sq, Hq]
  RowInfo* info;         // [B, Hkv * groups, q_tiles]: written by the dq kernel, read by the other
  Range* ranges;         // [B, q_tiles]: likewise
  __nv_bfloat16* dq;     // [B, Sq, Hq, D]
  __nv_bfloat16* dk;     // [B, Sk, Hkv, D]
  __nv_bfloat16* dv;
  uint32_t* status;
  int q_tiles;           // of kTile packed rows
  int tiles;             // resident tiles per head
  int64_t items;         // pieces of work: tiles, heads, sequences, parts
  int* taken;            // items of dk and dv beyond the CTAs' first: 0 again after the dq kernel
  int sms;               // of the device
  int parts;             // dk, dv: items that share a tile's walk
  float* part;           // their sums [parts][dv, dk][B, Sk, Hkv, D] (parts > 1)
};

// One piece of work: a resident tile and the steps to walk.
struct Item {
  int tile, hg, b, part;   // tile < 0: no more work
  int first;               // dq: first key tile; else first query tile of each head group
  int per_group, from, n;  // dk, dv: query tiles of a group, first step; steps
  Range seen;              // dq: of the tile's rows
};

struct __align__(16) BwdBars {
  uint64_t item_full[2], item_empty[2];
  uint64_t a_full, a_empty;
  uint64_t b_full[2][3], b_empty[2][3];   // [B1, B2][stage]
  uint64_t s_full, dp_full;               // S, P' written
  uint64_t p_full[2], ds_full[2];         // p, ds written over them: half of each group's columns, all
  uint64_t acc1_done, acc2_done;
  uint64_t acc_full, acc_empty;           // accumulators summed, read
  uint64_t met;                           // dq: the element warps among themselves
  uint64_t drained;
  Item item[2];
  uint32_t tmem, abort_word;
};

// Dot product of 8 bf16 columns.
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b) {
  const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum = fmaf(__uint_as_float(aw[i] << 16), __uint_as_float(bw[i] << 16), sum);
    sum = fmaf(__uint_as_float(aw[i] & 0xFFFF0000u), __uint_as_float(bw[i] & 0xFFFF0000u), sum);
  }
  return sum;
}

// kDq: rows are packed queries (A1 = q, A2 = do; B1 = k, B2 = v).
// Otherwise rows are keys (A1 = k, A2 = v; B1 = q, B2 = do).
// kFine: ds (and p of dv) in two bf16 parts.
template <int HD, bool kDq, int kMode, bool kFine>
__global__ void __launch_bounds__(kBwdThreads, 1)
    bwd_kernel(const __grid_constant__ CUtensorMap tm_a1, const __grid_constant__ CUtensorMap tm_a2,
               const __grid_constant__ CUtensorMap tm_b1, const __grid_constant__ CUtensorMap tm_b2,
               const BwdArgs a) {
  using C = Bwd<HD, kDq>;
  constexpr int kS1 = C::kStages[0], kS2 = C::kStages[1];
  constexpr bool kBias = kMode != kPlain, kCap = has_cap(kMode), kSlope = has_slopes(kMode);
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* a1 = smem;
  uint8_t* a2 = a1 + C::kBytes;
  uint8_t* bs = a2 + C::kBytes;                            // B1 [stage], B2 [stage]
  uint8_t* extra = bs + (kS1 + kS2) * C::kBytes;
  RowInfo* info = reinterpret_cast<RowInfo*>(extra);       // dk, dv: [stage of B1]
  BwdBars* bars = reinterpret_cast<BwdBars*>(extra + C::kExtra);
  volatile uint32_t* abort_word = &bars->abort_word;
  // Broadcast so that the compiler knows a warp to be of one mind.
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Shape& s = a.s;
  const int G = s.Hq / s.Hkv, pg = 1 << s.lgp;

  const int heads = kDq ? s.Hkv * s.groups : s.Hkv;
  const int q_step = kTile >> s.lgp;                       // tokens of a query tile
  static_assert(sizeof(BwdBars) <= 512, "the barriers' space");

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->item_full[i], 1);
      mbar_init(&bars->item_empty[i], 1 + 4 * kGroups);
    }
    mbar_init(&bars->a_full, 1);
    mbar_init(&bars->a_empty, 1);
    for (int o = 0; o < 2; ++o)
      for (int i = 0; i < (o ? kS2 : kS1); ++i) {
        mbar_init(&bars->b_full[o][i], 1);
        mbar_init(&bars->b_empty[o][i], 1);
      }
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->dp_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->p_full[i], 4 * kGroups);
      mbar_init(&bars->ds_full[i], 4 * kGroups);
    }
    mbar_init(&bars->acc1_done, 1);
    mbar_init(&bars->acc2_done, 1);
    mbar_init(&bars->acc_full, 1);
    mbar_init(&bars->acc_empty, 4 * kGroups);
    mbar_init(&bars->met, 4 * kGroups);
    mbar_init(&bars->drained, 1);
    bars->abort_word = 0;
    fence_barrier_init();
    if (kDq && blockIdx.x == 0) *a.taken = 0;
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  // The head group and query tile of an item's step (dk, dv).
  struct Walk {
    int group, tile;
    __device__ explicit Walk(const Item& it)
        : group(it.n ? it.from / it.per_group : 0), tile(it.n ? it.first + it.from % it.per_group : 0) {}
    __device__ void step(const Item& it) {
      if (++tile == it.first + it.per_group) {
        tile = it.first;
        ++group;
      }
    }
  };
  auto wait = [&](uint64_t* bar, int phase, uint32_t bit) {
    return mbar_wait_short_warp(bar, phase & 1, abort_word, a.status, bit);
  };

  if (warp == 0) {
    // ------------------------------------------------------ work and loads
    if (lane == 0) {
      tma_prefetch_desc(&tm_a1);
      tma_prefetch_desc(&tm_a2);
      tma_prefetch_desc(&tm_b1);
      tma_prefetch_desc(&tm_b2);
    }
    int loads_a = 0, loads_b[2] = {0, 0}, k = 0, g = 0;
    // Heaviest tiles of a causal mask first (early keys, late queries): dq's
    // many short items dealt out back and forth, so that every CTA gets as many
    // early as late; those of dk and dv to whichever CTA is free.
    auto dealt = [&](int turn) {
      int64_t deal = blockIdx.x;
      if constexpr (kDq) {
        deal = static_cast<int64_t>(turn) * gridDim.x + (turn & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      } else if (turn > 0) {
        int taken = 0;
        if (lane == 0) taken = atomicAdd(a.taken, 1);
        deal = static_cast<int64_t>(gridDim.x) + __shfl_sync(0xffffffffu, taken, 0);
      }
      Item it{};
      it.tile = -1;
      if (deal < a.items) {
        const int per = heads * s.B * a.parts, w = static_cast<int>(deal);
        it.tile = kDq ? a.tiles - 1 - w / per : w / per;
        it.hg = w % per % heads;
        it.b = w % per / heads % s.B;
        it.part = w % per / heads / s.B;
      }
      return it;
    };
    for (int turn = 0;; ++turn) {
      Item it = dealt(turn);
      if (it.tile >= 0) {
        if constexpr (kDq) {
          it.seen = tile_range(s, it.b, it.tile * q_step, q_step);
          if (it.seen.min_lo < it.seen.max_hi) {
            it.first = it.seen.min_lo / kTile;
            it.n = (it.seen.max_hi + kTile - 1) / kTile - it.first;
          }
        } else {
          // The query tiles from the first to the last that see any of the keys
          // (those between that see none add nothing).
          int lo = kNone, hi = -1;
          for (int i = lane; i < a.q_tiles; i += 32) {
            const Range r = a.ranges[static_cast<int64_t>(it.b) * a.q_tiles + i];
            if (r.min_lo < (it.tile + 1) * kTile && r.max_hi > it.tile * kTile) {
              lo = min(lo, i);
              hi = i;
            }
          }
          lo = __reduce_min_sync(0xffffffffu, lo);
          hi = __reduce_max_sync(0xffffffffu, hi);
          it.first = lo;
          it.per_group = hi >= 0 ? hi - lo + 1 : 0;
          const int n = it.per_group * s.groups;
          it.from = static_cast<int>(static_cast<int64_t>(n) * it.part / a.parts);
          it.n = static_cast<int>(static_cast<int64_t>(n) * (it.part + 1) / a.parts) - it.from;
        }
      }
      if (turn >= 2 && !wait(&bars->item_empty[turn & 1], (turn >> 1) - 1, kStatusTimeoutEmpty)) break;
      if (lane == 0) {
        bars->item[turn & 1] = it;
        mbar_arrive(&bars->item_full[turn & 1]);
      }
      __syncwarp();
      if (it.tile < 0) break;
      if (it.n == 0) continue;
      if (k > 0 && !wait(&bars->a_empty, k - 1, kStatusTimeoutEmpty)) break;
      const int kvh = kDq ? it.hg / s.groups : it.hg;
      const int ah = kDq ? it.hg << s.lgp : kvh, ar = it.tile * (kDq ? q_step : kTile);
      if (elected()) {
        mbar_arrive_expect_tx(&bars->a_full, 2 * C::kBytes);
        for (int c = 0; c < HD / 64; ++c) {
          tma_load_4d(a1 + c * kTile * 128, &tm_a1, 64 * c, ah, ar, it.b, &bars->a_full);
          tma_load_4d(a2 + c * kTile * 128, &tm_a2, 64 * c, ah, ar, it.b, &bars->a_full);
        }
      }
      __syncwarp();
      loads_a = ++k;
      bool ok = true;
      Walk at(it);
      for (int i = 0; i < it.n && ok; ++i, ++g, at.step(it)) {
        const int bh = kDq ? kvh : kvh * G + at.group * pg;
        const int br = kDq ? (it.first + i) * kTile : at.tile * q_step;
        for (int o = 0; o < 2 && ok; ++o) {
          const int stages = o ? kS2 : kS1, st = g % stages;
          if (g >= stages && !wait(&bars->b_empty[o][st], g / stages - 1, kStatusTimeoutEmpty)) {
            ok = false;
            break;
          }
          if (elected()) {
            uint8_t* dst = bs + (o * kS1 + st) * C::kBytes;
            mbar_arrive_expect_tx(&bars->b_full[o][st], C::kBytes + (!kDq && o == 0 ? kInfoBytes : 0));
            if (!kDq && o == 0)
              bulk_load(info + st,
                        a.info + (static_cast<int64_t>(it.b) * s.Hkv * s.groups + kvh * s.groups + at.group) *
                                     a.q_tiles + at.tile,
                        kInfoBytes, &bars->b_full[o][st]);
            for (int c = 0; c < HD / 64; ++c)
              tma_load_4d(dst + c * kTile * 128, o ? &tm_b2 : &tm_b1, 64 * c, bh, br, it.b, &bars->b_full[o][st]);
          }
          __syncwarp();
          ++loads_b[o];
        }
      }
      if (!ok) break;
    }
    // No copy may be in flight when the CTA leaves.
    uint32_t none = 0;
    if (loads_a) mbar_wait(&bars->a_full, (loads_a - 1) & 1, &none, a.status, kStatusTimeoutDrain);
    for (int o = 0; o < 2; ++o)
      for (int stages = o ? kS2 : kS1, i = max(loads_b[o] - stages, 0); i < loads_b[o]; ++i)
        mbar_wait(&bars->b_full[o][i % stages], (i / stages) & 1, &none, a.status, kStatusTimeoutDrain);
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------- products
    // The whole warp walks and one lane issues: operands stay uniform, and the
    // issue takes few slots of the scheduler that the element warps share.
    const uint32_t id_s = idesc_bf16_f32(kTile, kTile), id_acc = idesc_bf16_f32_bmn(kTile, HD);
    const uint32_t col_s = tmem, col_p = tmem + kColP;
    const uint64_t d_a[2] = {sdesc_kmajor_sw128(smem_u32(a1)), sdesc_kmajor_sw128(smem_u32(a2))};
    const uint64_t d_rows = sdesc_kmajor_sw128(smem_u32(bs)), d_cols = cols_desc<kTile>(smem_u32(bs));
    auto at = [&](int g, int o) {
      return static_cast<uint64_t>(o ? kS1 + g % kS2 : g % kS1) * (C::kBytes >> 4);
    };
    int g0 = 0, k = 0;       // steps and items with steps before this one
    bool issued = false;
    // S (o = 0) or P' (o = 1) of step g, once the products that read the p or
    // ds in its columns are done; the item's last P' frees the resident tiles.
    auto scores = [&](int g, int o, bool last) -> bool {
      if (g > 0 && !wait(o ? &bars->acc2_done : &bars->acc1_done, g - 1, kStatusTimeoutAccum)) return false;
      const int stages = o ? kS2 : kS1;
      if (!wait(&bars->b_full[o][g % stages], g / stages, kStatusTimeoutFull)) return false;
      tc_fence_after();
      if (elected()) {
        mma_rows<HD, kTile>(o ? col_p : col_s, d_a[o], d_rows + at(g, o), id_s);
        tc_commit(o ? &bars->dp_full : &bars->s_full);
        if (o && last) tc_commit(&bars->a_empty);
      }
      __syncwarp();
      issued = true;
      return true;
    };
    bool ok = true;
    for (int turn = 0; ok; ++turn) {
      if (!wait(&bars->item_full[turn & 1], turn >> 1, kStatusTimeoutFull)) break;
      const int n = bars->item[turn & 1].tile < 0 ? -1 : bars->item[turn & 1].n;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->item_empty[turn & 1]);
      if (n < 0) break;
      if (n == 0) continue;
      ok = wait(&bars->a_full, k, kStatusTimeoutFull) && scores(g0, 0, false) && scores(g0, 1, n == 1);
      for (int i = 0; i < n && ok; ++i) {
        const int g = g0 + i;
        // Each product in two parts: the first runs while the other half of its
        // operand is still computed.
        for (int half = 0; half < 2 && ok; ++half) {
          ok = wait(&bars->p_full[half], g, kStatusTimeoutFull) &&
               (half || i > 0 || k == 0 || wait(&bars->acc_empty, k - 1, kStatusTimeoutAccum));
          if (!ok) break;
          tc_fence_after();
          if (elected()) {
            mma_cols_half<HD, kTile>(tmem + kColAcc, col_s, d_cols + at(g, kDq ? 0 : 1), id_acc, half, i > 0);
            if constexpr (kFine && !kDq)
              mma_cols_half<HD, kTile>(tmem + kColAcc, col_s + kCols / 2, d_cols + at(g, 1), id_acc, half, true);
            if (half) {
              tc_commit(&bars->b_empty[1][g % kS2]);
              tc_commit(&bars->acc1_done);
            }
          }
          __syncwarp();
        }
        ok = ok && (i + 1 == n || scores(g + 1, 0, false));
        for (int half = 0; half < 2 && ok; ++half) {
          ok = wait(&bars->ds_full[half], g, kStatusTimeoutFull);
          if (!ok) break;
          tc_fence_after();
          if (elected()) {
            mma_cols_half<HD, kTile>(tmem + kColAcc + HD, col_p, d_cols + at(g, 0), id_acc, half, i > 0);
            if constexpr (kFine)
              mma_cols_half<HD, kTile>(tmem + kColAcc + HD, col_p + kCols / 2, d_cols + at(g, 0), id_acc, half, true);
            if (half) {
              tc_commit(&bars->b_empty[0][g % kS1]);
              tc_commit(&bars->acc2_done);
              if (i + 1 == n) tc_commit(&bars->acc_full);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        if (i + 1 < n && !scores(g + 1, 1, i + 2 == n)) ok = false;
      }
      g0 += n;
      ++k;
    }
    // Every product issued has to be done before the CTA leaves, also after a wait that gave up.
    if (issued) {
      if (elected()) tc_commit(&bars->drained);
      uint32_t none = 0;
      mbar_wait(&bars->drained, 0, &none, a.status, kStatusTimeoutDrain);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------- elements
    const int group = (warp - 2) >> 2;             // the columns this warp owns
    const int quarter = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int row = quarter * 32 + lane;           // TMEM lane: the element row this thread owns
    const uint64_t sl2_2 = pair(s.sl2, s.sl2);
    const int mine0 = group * kCols;               // the first of the group's columns
    int g0 = 0, k = 0, meetings = 0;
    // A barrier of the element warps that gives up as every other wait does.
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->met);
      return wait(&bars->met, meetings++, kStatusTimeoutAccum);
    };
    // dq: what the item's rows need from memory.  Every load at once, from the
    // last row where there is none.  Of do and o 16 lanes have a row, two rows to a
    // warp.  kAhead: for the next item before this one's results are stored (at
    // the end of the work the first tile's: always, so that the registers are
    // free in between; 280 -> 266 us, short walks of documents 203 -> 184).  Not
    // under a cap, whose registers it would spill (105 -> 110 us).
    constexpr bool kAhead = kDq && !kCap;
    constexpr int kRounds = kTile / (8 * kGroups);
    [[maybe_unused]] uint4 do_row[kDq ? kRounds : 1], o_row[kDq ? kRounds : 1];
    [[maybe_unused]] int row_begin = 0, row_end = 0;
    [[maybe_unused]] float row_lse = 0.f;
    const bool in_row = (lane & 15) * 8 < s.D;
    auto fetch = [&](const Item& it) {
      const int last = s.Sq - 1, row0 = max(it.tile, 0) * q_step, d = in_row ? (lane & 15) * 8 : 0;
      const int64_t tokens = static_cast<int64_t>(it.b) * s.Sq;
      const int64_t at = tokens + min(row0 + (row >> s.lgp), last);
      row_begin = s.begin[at], row_end = s.end[at];
      row_lse = a.lse[at * s.Hq + (it.hg << s.lgp) + (row & (pg - 1))];
#pragma unroll
      for (int i = 0; i < kRounds; ++i) {
        const int rr = ((warp - 2) * kRounds + i) * 2 + (lane >> 4);
        const int rt = min(row0 + (rr >> s.lgp), last), rh = (it.hg << s.lgp) + (rr & (pg - 1));
        do_row[i] = *reinterpret_cast<const uint4*>(a.dout + it.b * a.do_batch + rt * a.do_token + rh * a.do_head + d);
        o_row[i] = *reinterpret_cast<const uint4*>(a.out + ((tokens + rt) * s.Hq + rh) * s.D + d);
      }
    };
    auto take = [&](int turn, Item& it) -> bool {
      if (!wait(&bars->item_full[turn & 1], turn >> 1, kStatusTimeoutFull)) return false;
      it = bars->item[turn & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->item_empty[turn & 1]);
      return true;
    };
    Item it{-1};
    const bool begun = !kAhead || take(0, it);
    if constexpr (kAhead) fetch(it);
    for (int turn = 0; begun; ++turn) {
      if constexpr (!kAhead)
        if (!take(turn, it)) break;
      if (it.tile < 0) break;
      if constexpr (kDq && !kAhead) fetch(it);
      const int kvh = kDq ? it.hg / s.groups : it.hg, b = it.b;
      const int row0 = it.tile * (kDq ? q_step : kTile);
      // dq: the row's token, head, range and statistics; else the row's key.
      int tok = 0, head = 0, lo = 0, hi = 0;
      float lse2 = INFINITY, d0 = 0.f;
      uint64_t dsum2 = 0;                          // (0, 0)
      const int key = row0 + row;
      if constexpr (kDq) {
        tok = row0 + (row >> s.lgp);
        head = (it.hg << s.lgp) + (row & (pg - 1));
        // d0 = do . o, handed to the rows' owners through shared memory (read before
        // the item's second meeting, written after it).
        float* dots = reinterpret_cast<float*>(extra) + kGroups * kTile;
        if (tok < s.Sq) {
          lo = max(row_begin, 0);
          hi = min(row_end, s.Sk);
          if (lo >= hi) lo = hi = 0;
          lse2 = row_lse * kLog2e;
        }
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
          float sum = in_row ? dot8(do_row[i], o_row[i]) : 0.f;
#pragma unroll
          for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          if ((lane & 15) == 0) dots[((warp - 2) * kRounds + i) * 2 + (lane >> 4)] = sum;
        }
        if (!meet()) break;
        d0 = dots[row];
      }
      const float row_slope2 = kDq && kSlope ? s.slopes[head] * kLog2e : 0.f;
      bool ok = true;
      Walk at(it);
      for (int i = 0; i < it.n; ++i, at.step(it)) {
        const int g = g0 + i, st = g % kS1;
        const RowInfo& cols = info[kDq ? 0 : st];              // dk, dv: of the step's columns
        bool whole;
        int col0;                                    // dq: the group's first key; else its first token
        if (!kDq && !wait(&bars->b_full[0][st], g / kS1, kStatusTimeoutFull)) {
          ok = false;
          break;
        }
        if constexpr (kDq) {
          col0 = (it.first + i) * kTile + mine0;
          whole = it.seen.max_lo <= col0 && it.seen.min_hi >= col0 + kCols;
        } else {
          col0 = at.tile * q_step + (mine0 >> s.lgp);
          whole = cols.max_lo[group] <= row0 && cols.min_hi[group] >= row0 + kTile;
        }
        [[maybe_unused]] uint64_t nl_of[kDq ? 1 : kCols / 2];   // dk, dv: -lse2 of the columns
        if constexpr (!kDq && !kBias) {
#pragma unroll
          for (int c = 0; c < kCols; c += 4) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(cols.nlse2 + mine0 + c);
            nl_of[c / 2] = v.x, nl_of[c / 2 + 1] = v.y;
          }
        }
        if (!wait(&bars->s_full, g, kStatusTimeoutAccum)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // 0 times infinity is not 0: what no row of this tile (dq) or no key at all
        // (dk, dv) meets but shares a streamed tile with what is met is cleared.
        // S has been read by now, P' is waited for where its operand is cleared.
        if constexpr (kDq) {
          const int from = it.seen.min_lo - (col0 - mine0), to = it.seen.max_hi - (col0 - mine0);
          if (from > 0 || (to < kTile && it.seen.max_hi < s.Sk)) {
            uint4* tile = reinterpret_cast<uint4*>(bs + st * C::kBytes);   // chunks of kTile rows of 8
            for (int e = threadIdx.x - 64; e < C::kBytes / 16; e += 128 * kGroups) {
              const int at_row = (e >> 3) % kTile;
              if (at_row < from || at_row >= to) tile[e] = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        } else if (cols.max_lo[group] == kNone) {    // some row sees nothing
          // (past the sequence the loads brought zeros)
          const int first = cols.lo[mine0 + lane];
          const uint32_t none = __ballot_sync(0xffffffffu, first >= cols.hi[mine0 + lane] && first >= 0);
          if (none) {
            if (!wait(&bars->dp_full, g, kStatusTimeoutAccum)) {
              ok = false;
              break;
            }
            // Each of the group's warps clears its 8 of the 32 rows, in both operands.
            for (int o = 0; o < 2; ++o) {
              uint4* tile = reinterpret_cast<uint4*>(bs + (o ? kS1 + g % kS2 : st) * C::kBytes);
              for (int e = lane; e < HD; e += 32) {            // chunks of 64 columns, rows, pieces of 16 bytes
                const int at_row = quarter * 8 + ((e >> 3) & 7);
                if (none >> at_row & 1) tile[((e >> 6) * kTile + mine0 + at_row) * 8 + (e & 7)] = make_uint4(0, 0, 0, 0);
              }
            }
            fence_proxy_async_smem();
          }
        }
        // dq: from the row's token to the first key; else from the row's key to the first token.
        [[maybe_unused]] const float dist0 = static_cast<float>((kDq ? tok - col0 : col0 - key) + s.Sk - s.Sq);
        const uint32_t at_s = tmem + kCols * group + lanes, at_p = at_s + kColP;
        uint32_t x[kCols], w[kCols / 4];             // scores, then p; half the packed operands
        [[maybe_unused]] uint32_t u[kCols / 4];      // kFine: what their rounding left
        auto left = [](uint32_t hi, float a, float b) {
          return pack_bf16x2(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xFFFF0000u));
        };
        [[maybe_unused]] __half2 fac[kCap ? kCols / 2 : 1];
        tmem_ld_32x32b_x32(at_s, x);
        tmem_wait_ld();
        // Which of the columns c .. c + 3 the row does not see.
        auto hidden = [&](int c, bool (&hide)[4]) {
          if constexpr (kDq) {
#pragma unroll
            for (int e = 0; e < 4; ++e) hide[e] = c + e < lo - col0 || c + e >= hi - col0;
          } else {
            const int4 u = *reinterpret_cast<const int4*>(cols.lo + mine0 + c);
            const int4 v = *reinterpret_cast<const int4*>(cols.hi + mine0 + c);
            hide[0] = key < u.x || key >= v.x;
            hide[1] = key < u.y || key >= v.y;
            hide[2] = key < u.z || key >= v.z;
            hide[3] = key < u.w || key >= v.w;
          }
        };
        auto exponentials = [&](int c, auto masked) {
          uint64_t nl[2];                            // -lse2 of the columns
          if constexpr (kDq) {
            nl[0] = nl[1] = pair(-lse2, -lse2);
          } else if constexpr (kBias) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(cols.nlse2 + mine0 + c);
            nl[0] = v.x, nl[1] = v.y;
          } else {
            nl[0] = nl_of[c / 2], nl[1] = nl_of[c / 2 + 1];
          }
          float p[4];
          [[maybe_unused]] uint64_t f[2];
          if constexpr (kBias) {
            [[maybe_unused]] float slope2[4] = {row_slope2, row_slope2, row_slope2, row_slope2};
            if constexpr (!kDq && kSlope) {
              const float4 v = *reinterpret_cast<const float4*>(cols.slope2 + mine0 + c);
              slope2[0] = v.x, slope2[1] = v.y, slope2[2] = v.z, slope2[3] = v.w;
            }
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
              const int col = c + h;
              uint64_t e = pair(x[col], x[col + 1]);
              if constexpr (kCap) {
                const uint64_t u = cap_u2_finite(cap_arg2(s, e)), r = cap_r2(u);
                e = capped2(s, r, add2(nl[h / 2], pair(s.cap2, s.cap2)));
                f[h / 2] = cap_slope2(r, u);
              } else {
                e = fma2(e, sl2_2, nl[h / 2]);
              }
              if constexpr (kSlope) {
                // dq: columns are keys; else those of a token's packed heads share its distance
                const float d_0 = kDq ? dist0 - col : dist0 + small_float(col >> s.lgp);
                const float d_1 = kDq ? dist0 - (col + 1) : dist0 + small_float((col + 1) >> s.lgp);
                e = fma2(pair(-slope2[h], -slope2[h + 1]), pair(fabsf(d_0), fabsf(d_1)), e);
              }
              unpair(e, p[h], p[h + 1]);
            }
            if constexpr (kCap)                    // two of four: the tanh keeps the special units busy
              ex2_pair(p[0], p[1], p[0], p[1]);
            else
              p[0] = ex2(p[0]), p[1] = ex2(p[1]);
            p[2] = ex2(p[2]), p[3] = ex2(p[3]);
          } else {
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
              unpair(fma2(pair(x[c + h], x[c + h + 1]), sl2_2, nl[h / 2]), p[h], p[h + 1]);
              if (h == 0 && c % 8 == 0) {            // a quarter of the exponentials
                ex2_pair(p[h], p[h + 1], p[h], p[h + 1]);
              } else {
                p[h] = ex2(p[h]);
                p[h + 1] = ex2(p[h + 1]);
              }
            }
          }
          if constexpr (decltype(masked)::value) {
            bool hide[4];
            hidden(c, hide);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (hide[e]) p[e] = 0.f;
            if constexpr (kCap) {                  // f of a hidden score may not be finite
#pragma unroll
              for (int h = 0; h < 4; h += 2) {
                float f_0, f_1;
                unpair(f[h / 2], f_0, f_1);
                f[h / 2] = pair(hide[h] ? 0.f : f_0, hide[h + 1] ? 0.f : f_1);
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) x[c + e] = __float_as_uint(p[e]);
          if constexpr (kCap) {
            // f, 2^15 times the derivative, waits for dp in 16 bits: half a step, 2^-11 of a
            // factor of ds, an eighth of ds's own rounding, up to scores of 10.7 caps.
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
              float f_0, f_1;
              unpair(f[h / 2], f_0, f_1);
              fac[(c + h) / 2] = __floats2half2_rn(f_0, f_1);
              if constexpr (kDq) unpair(mul2(pair(p[h], p[h + 1]), f[h / 2]), p[h], p[h + 1]);
            }
          }
          w[c % 16 / 2] = pack_bf16x2(p[0], p[1]);
          w[c % 16 / 2 + 1] = pack_bf16x2(p[2], p[3]);
          if constexpr (kFine && !kDq) {
            u[c % 16 / 2] = left(w[c % 16 / 2], p[0], p[1]);
            u[c % 16 / 2 + 1] = left(w[c % 16 / 2 + 1], p[2], p[3]);
          }
        };
        // The operands' first or second half (of the group's columns) to TMEM; what
        // their rounding left into the second half of the group's columns there.
        auto hand_over = [&](uint32_t at_w, uint64_t* bar, auto two) {
          tmem_st_32x32b_x8(at_w, w);
          if constexpr (decltype(two)::value) tmem_st_32x32b_x8(at_w + kCols / 2, u);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar);
        };
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 16) {
          if (whole) {
#pragma unroll
            for (int c = 0; c < 16; c += 4) exponentials(c0 + c, std::false_type{});
          } else {
#pragma unroll
            for (int c = 0; c < 16; c += 4) exponentials(c0 + c, std::true_type{});
          }
          hand_over(at_s + c0 / 2, &bars->p_full[c0 / 16], std::bool_constant<kFine && !kDq>{});
        }

        if (!wait(&bars->dp_full, g, kStatusTimeoutAccum)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // dp of the columns c .. c + 3 in y; ds into w.
        auto gradients = [&](const uint32_t* y, int c, auto masked) {
          uint64_t nd[2];                            // -delta of the columns, times unit
          constexpr float unit = kCap ? 1.0f / kCapSlope : 1.0f;
          if constexpr (kDq) {
            nd[0] = nd[1] = pair(-d0 * unit, -d0 * unit);
          } else {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(cols.ndelta + mine0 + c);
            nd[0] = v.x, nd[1] = v.y;
          }
          [[maybe_unused]] bool hide[4];
          if constexpr (decltype(masked)::value) hidden(c, hide);
#pragma unroll
          for (int h = 0; h < 4; h += 2) {
            const int col = c + h;
            const uint64_t dp = pair(y[h], y[h + 1]), p = pair(x[col], x[col + 1]);
            if constexpr (kDq) {
              if constexpr (decltype(masked)::value) {
                // p is 0 at a hidden key, but whatever its value makes of dp may not be finite
                float d_0, d_1;
                unpair(mul2(p, dp), d_0, d_1);
                dsum2 = add2(dsum2, pair(hide[h] ? 0.f : d_0, hide[h + 1] ? 0.f : d_1));
              } else {
                dsum2 = fma2(p, dp, dsum2);
              }
            }
            float ds[2];
            if constexpr (kCap) {
              const float2 f = __half22float2(fac[col / 2]);
              unpair(mul2(mul2(p, pair(f.x, f.y)), fma2(dp, pair(unit, unit), nd[h / 2])), ds[0], ds[1]);
            } else {
              unpair(mul2(p, add2(dp, nd[h / 2])), ds[0], ds[1]);
            }
            if constexpr (decltype(masked)::value) {
              if (hide[h]) ds[0] = 0.f;
              if (hide[h + 1]) ds[1] = 0.f;
            }
            w[col % 16 / 2] = pack_bf16x2(ds[0], ds[1]);
            if constexpr (kFine) u[col % 16 / 2] = left(w[col % 16 / 2], ds[0], ds[1]);
          }
        };
        [[maybe_unused]] uint32_t y_next[kFine ? 16 : 1];
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 16) {
          uint32_t y[16];
          if constexpr (kFine) {
            if (c0 == 0) {
              tmem_ld_32x32b_x16(at_p, y);
              tmem_ld_32x32b_x16(at_p + 16, y_next);   // u goes over these columns
              tmem_wait_ld();
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] = y_next[e];
            }
          } else {
            tmem_ld_32x32b_x16(at_p + c0, y);
            tmem_wait_ld();
          }
          if (whole) {
#pragma unroll
            for (int c = 0; c < 16; c += 4) gradients(y + c, c0 + c, std::false_type{});
          } else {
#pragma unroll
            for (int c = 0; c < 16; c += 4) gradients(y + c, c0 + c, std::true_type{});
          }
          hand_over(at_p + c0 / 2, &bars->ds_full[c0 / 16], std::bool_constant<kFine>{});
        }
      }
      g0 += it.n;
      float fix = 0.f;
      if constexpr (kDq) {
        // Each group summed delta over its columns.
        float dsum, odd;
        unpair(dsum2, dsum, odd);
        float* sums = reinterpret_cast<float*>(extra);   // [kGroups][128]
        sums[group * kTile + row] = dsum + odd;
        if (!ok || !meet()) break;
        dsum = 0.f;
#pragma unroll
        for (int q = 0; q < kGroups; ++q) dsum += sums[q * kTile + row];
        fix = lo < hi ? d0 - dsum : 0.f;             // a row that sees nothing: whatever its dout
        if constexpr (kCap) fix *= 1.0f / kCapSlope; // the sum of p f k has it
        RowInfo* o = a.info + (static_cast<int64_t>(b) * heads + it.hg) * a.q_tiles + it.tile;
        if (group == 0) {
          o->nlse2[row] = tok < s.Sq ? -lse2 : -INFINITY;
          o->ndelta[row] = tok < s.Sq ? -dsum * (kCap ? 1.0f / kCapSlope : 1.0f) : 0.f;
        } else if (group == 1) {
          o->lo[row] = tok < s.Sq ? lo : -1;         // (-1, -1): past the sequence
          o->hi[row] = tok < s.Sq ? hi : -1;
        } else if (kSlope && group == 2) {
          o->slope2[row] = row_slope2;
        }
        if (group == 3) {
          // The rows of a quarter are a group's columns there.  None inside the
          // sequence: -inf + NaN is not masked, so not whole either.
          static_assert(kCols == 32 && kGroups == 4, "a quarter's rows");
          const bool in = tok < s.Sq;
          const int max_lo = __reduce_max_sync(0xffffffffu, !in ? -1 : lo < hi ? lo : kNone);
          const int min_hi = __reduce_min_sync(0xffffffffu, !in ? kNone : hi);
          if (lane == 0) {
            o->max_lo[quarter] = min_hi == kNone ? kNone - 1 : max_lo;
            o->min_hi[quarter] = min_hi;
            if (it.hg == 0 && quarter == 0) a.ranges[static_cast<int64_t>(b) * a.q_tiles + it.tile] = it.seen;
          }
        }
      }
      [[maybe_unused]] Item next;
      if constexpr (kAhead) {
        if (!take(turn + 1, next)) break;            // (after a wait that gave up, dq has left above)
        fetch(next);
      }
      if (it.n > 0) {
        ok = ok && wait(&bars->acc_full, k, kStatusTimeoutAccum);
        ++k;
      }
      tc_fence_after();
      if (ok) {
        // dq: each group stores a quarter of the columns; else two store the
        // halves of dv, two those of dk.
        const bool live = kDq ? tok < s.Sq : key < s.Sk;
        const bool second = kDq || group >= kGroups / 2;   // of the accumulators
        __nv_bfloat16* o;
        if constexpr (kDq)
          o = a.dq + ((static_cast<int64_t>(b) * s.Sq + tok) * s.Hq + head) * s.D;
        else
          o = (second ? a.dk : a.dv) + ((static_cast<int64_t>(b) * s.Sk + key) * s.Hkv + kvh) * s.D;
        const float by = second ? s.scale : 1.0f;
        constexpr int kWidth = kDq ? HD / kGroups : HD / (kGroups / 2);
        const int c_from = (kDq ? group : group & 1) * kWidth;
#pragma unroll 1
        for (int c = c_from; c < c_from + kWidth; c += 16) {
          uint32_t v[16];
          if (it.n > 0) {
            tmem_ld_32x32b_x16(tmem + kColAcc + (second ? HD : 0) + lanes + c, v);
            if constexpr (kDq) {
              uint32_t u[16];
              tmem_ld_32x32b_x16(tmem + kColAcc + lanes + c, u);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e)
                v[e] = __float_as_uint(fmaf(fix, __uint_as_float(u[e]), __uint_as_float(v[e])));
            } else {
              tmem_wait_ld();
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = 0u;
          }
          if (!live) continue;
          if (!kDq && a.parts > 1) {
            const int64_t rows = static_cast<int64_t>(s.B) * s.Sk * s.Hkv;
            float* f =
                a.part + ((it.part * 2 + second) * rows + (static_cast<int64_t>(b) * s.Sk + key) * s.Hkv + kvh) * s.D + c;
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              if (c + e < s.D)
                *reinterpret_cast<float4*>(f + e) =
                    make_float4(__uint_as_float(v[e]) * by, __uint_as_float(v[e + 1]) * by,
                                __uint_as_float(v[e + 2]) * by, __uint_as_float(v[e + 3]) * by);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (c + 8 * e < s.D) {
              uint32_t u[4];
#pragma unroll
              for (int q = 0; q < 4; ++q)
                u[q] = pack_bf16x2(__uint_as_float(v[8 * e + 2 * q]) * by, __uint_as_float(v[8 * e + 2 * q + 1]) * by);
              *reinterpret_cast<uint4*>(o + c + 8 * e) = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
      }
      if (!ok) break;
      if (it.n > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->acc_empty);
      }
      if constexpr (kAhead) it = next;
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

// dv and dk from the parts' sums, in the parts' order.  n4: groups of four
// columns of one of the two.
__global__ void __launch_bounds__(256) parts_kernel(const float4* __restrict__ part, int parts, int64_t n4,
                                                    uint2* __restrict__ dv, uint2* __restrict__ dk) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < 2 * n4;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    float4 sum = part[i];
    for (int p = 1; p < parts; ++p) {
      const float4 x = part[2 * n4 * p + i];
      sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
    }
    (i < n4 ? dv[i] : dk[i - n4]) = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
  }
}

// CTAs that share one key tile's walk: none where two to each would be more than
// the SMs; else towards one CTA per SM, each keeping four steps of the longest
// walk (a step is about 2 us, the reduction's launch another).  Backward without /
// with parts, 32/8 heads of 128 and, in brackets, every key seen instead of a causal
// mask:  32 key tiles (512 tokens) 66 / 49 us (64 / 48), 64 91 / 76 (103 / 88), 72
// 102 / 84 (112 / 95); two parts from 75 on, more CTAs than SMs:  80 117 / 95 (142 /
// 158), 128 187 / 155 (240 / 262), 144 224 / 192 (280 / 304).  Past half the SMs two
// parts gain 14 - 26% under a causal mask, whose walks differ, and lose 5 - 11% where
// all are equal; which of the two a call is only its ranges say.
int bwd_parts(int64_t key_ctas, int64_t steps) {
  if (key_ctas > 74) return 1;
  int64_t n = 148 / key_ctas;
  if (n > steps / 4) n = steps / 4;
  return n < 1 ? 1 : static_cast<int>(n);
}

template <int HD, bool kDq, int kMode, bool kFine>
int launch_bwd(const CUtensorMap& a1, const CUtensorMap& a2, const CUtensorMap& b1, const CUtensorMap& b2,
               const BwdArgs& a, cudaStream_t stream) {
  constexpr int kSmem = Bwd<HD, kDq>::kSmem;
  int rc = allow_smem(reinterpret_cast<const void*>(&bwd_kernel<HD, kDq, kMode, kFine>), kSmem);
  if (rc) return rc;
  const int64_t grid = a.items < a.sms ? a.items : a.sms;
  bwd_kernel<HD, kDq, kMode, kFine><<<static_cast<unsigned>(grid), kBwdThreads, kSmem, stream>>>(a1, a2, b1, b2, a);
  return FL_OK;
}

template <int HD, bool kDq, bool kFine>
int launch_bwd_mode(int mode, const CUtensorMap& a1, const CUtensorMap& a2, const CUtensorMap& b1,
                    const CUtensorMap& b2, const BwdArgs& a, cudaStream_t stream) {
  return mode == kCappedSlopes ? launch_bwd<HD, kDq, kCappedSlopes, kFine>(a1, a2, b1, b2, a, stream)
         : mode == kCapped     ? launch_bwd<HD, kDq, kCapped, kFine>(a1, a2, b1, b2, a, stream)
         : mode == kSlopes     ? launch_bwd<HD, kDq, kSlopes, kFine>(a1, a2, b1, b2, a, stream)
                               : launch_bwd<HD, kDq, kPlain, kFine>(a1, a2, b1, b2, a, stream);
}

template <bool kDq>
int launch_bwd_any(int D, int mode, bool fine, const CUtensorMap& a1, const CUtensorMap& a2, const CUtensorMap& b1,
                   const CUtensorMap& b2, const BwdArgs& a, cudaStream_t stream) {
  if (D <= 64)
    return fine ? launch_bwd_mode<64, kDq, true>(mode, a1, a2, b1, b2, a, stream)
                : launch_bwd_mode<64, kDq, false>(mode, a1, a2, b1, b2, a, stream);
  return fine ? launch_bwd_mode<128, kDq, true>(mode, a1, a2, b1, b2, a, stream)
              : launch_bwd_mode<128, kDq, false>(mode, a1, a2, b1, b2, a, stream);
}

int64_t q_tiles_of(int64_t Sq, int lgp) { return (Sq + (kTile >> lgp) - 1) / (kTile >> lgp); }

}  // namespace attn
}  // namespace fl

using namespace fl;

extern "C" {

// The query tiles' row statistics, then their ranges, the count of items taken,
// and the parts' sums.
static size_t attn_bwd_sizes(int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int D, int* parts, size_t* part_at) {
  const int lgp = attn::packed_log2(Hq, Hkv);
  const int64_t q_tiles = attn::q_tiles_of(Sq, lgp), key_tiles = (Sk + attn::kTile - 1) / attn::kTile;
  *parts = attn::bwd_parts(key_tiles * B * Hkv, q_tiles * ((Hq / Hkv) >> lgp));
  *part_at = static_cast<size_t>(B) * q_tiles * ((Hq >> lgp) * sizeof(attn::RowInfo) + sizeof(attn::Range)) + 16;
  return *part_at + (*parts > 1 ? static_cast<size_t>(*parts) * 2 * B * Sk * Hkv * D * sizeof(float) : 0);
}

size_t fl_attn_bwd_workspace_bytes(int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int D) {
  if (B <= 0 || Sq <= 0 || Sk <= 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 8 || B > (1 << 16) || Sq > (1 << 30) ||
      Sk > (1 << 30))
    return 0;
  int parts;
  size_t part_at;
  return attn_bwd_sizes(B, Sq, Sk, Hq, Hkv, D, &parts, &part_at);
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
    if (kv_bytes && (cudaMemsetAsync(dk, 0, kv_bytes, st) != cudaSuccess ||
                     cudaMemsetAsync(dv, 0, kv_bytes, st) != cudaSuccess))
      return set_error(FL_ERR_CUDA, "fl_attn_bwd: clearing dk and dv failed");
    return FL_OK;
  }
  if (Sk == 0) {
    if (cudaMemsetAsync(dq, 0, static_cast<size_t>(B) * Sq * Hq * D * 2, st) != cudaSuccess)
      return set_error(FL_ERR_CUDA, "fl_attn_bwd: clearing dq failed");
    return FL_OK;
  }
  int parts;
  size_t part_at;
  const size_t need = attn_bwd_sizes(B, Sq, Sk, Hq, Hkv, D, &parts, &part_at);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u))
    return set_error(FL_ERR_ARG, "fl_attn_bwd: workspace missing, short or not 16-byte aligned");
  attn::BwdArgs a{};
  attn::fill_shape(a.s, (int)B, (int)Sq, (int)Sk, Hq, Hkv, D, begin, end, scale, softcap, slopes);
  int dev = 0;
  if ((rc = current_context(&dev))) return rc;
  if (!(a.status = status_word(dev))) return set_error(FL_ERR_CUDA, "fl_attn_bwd: status word unavailable");
  a.sms = device_sms(dev);
  a.q_tiles = static_cast<int>(attn::q_tiles_of(Sq, a.s.lgp));
  a.info = static_cast<attn::RowInfo*>(workspace);
  a.ranges = reinterpret_cast<attn::Range*>(a.info + B * (Hq >> a.s.lgp) * a.q_tiles);
  a.taken = reinterpret_cast<int*>(a.ranges + B * a.q_tiles);
  a.out = reinterpret_cast<const __nv_bfloat16*>(out);
  a.dout = reinterpret_cast<const __nv_bfloat16*>(dout);
  a.do_batch = strides[9];
  a.do_token = strides[10];
  a.do_head = strides[11];
  a.lse = lse;
  a.dq = reinterpret_cast<__nv_bfloat16*>(dq);
  a.dk = reinterpret_cast<__nv_bfloat16*>(dk);
  a.dv = reinterpret_cast<__nv_bfloat16*>(dv);
  const int pg = 1 << a.s.lgp, q_step = attn::kTile >> a.s.lgp;
  const int64_t key_tiles = (Sk + attn::kTile - 1) / attn::kTile;
  if (key_tiles * B * Hkv > (int64_t(1) << 30)) return set_error(FL_ERR_ARG, "fl_attn_bwd: too many key tiles");

  CUtensorMap mq, mk, mv, mdo;
  const int b = (int)B, sq = (int)Sq, sk = (int)Sk;
  if ((rc = attn_map(&mq, q, strides[0], strides[1], strides[2], b, sq, Hq, D, pg, q_step)) ||
      (rc = attn_map(&mk, k, strides[3], strides[4], strides[5], b, sk, Hkv, D, 1, attn::kTile)) ||
      (rc = attn_map(&mv, v, strides[6], strides[7], strides[8], b, sk, Hkv, D, 1, attn::kTile)) ||
      (rc = attn_map(&mdo, dout, strides[9], strides[10], strides[11], b, sq, Hq, D, pg, q_step)))
    return rc;
  const int mode = (softcap != 0.f ? attn::kCapped : attn::kPlain) + (slopes ? attn::kSlopes : 0);
  a.items = attn::fwd_ctas(b, sq, Hq, Hkv);
  a.parts = 1;
  a.tiles = static_cast<int>(a.items / B / (Hq >> a.s.lgp));
  const bool fine = attn::few_results(B * Sq * Hq, Sk);
  rc = attn::launch_bwd_any<true>(D, mode, fine, mq, mdo, mk, mv, a, st);
  if (rc) return rc;
  a.tiles = static_cast<int>(key_tiles);
  a.parts = parts;
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + part_at);
  a.items = key_tiles * B * Hkv * parts;
  rc = attn::launch_bwd_any<false>(D, mode, fine, mk, mv, mq, mdo, a, st);
  if (rc) return rc;
  if (parts > 1) {
    const int64_t n4 = B * Sk * Hkv * D / 4;
    const int64_t blocks = (2 * n4 + 255) / 256;
    attn::parts_kernel<<<static_cast<unsigned>(blocks < 2368 ? blocks : 2368), 256, 0, st>>>(
        reinterpret_cast<const float4*>(a.part), parts, n4, reinterpret_cast<uint2*>(dv), reinterpret_cast<uint2*>(dk));
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FL_ERR_CUDA, "fl_attn_bwd: %s", cudaGetErrorString(e));
  return FL_OK;
}

}  // extern "C"
