// Attention forward over row ranges (see fl_attn.cuh for the formulas).
//
// A CTA takes a tile of 128 (packed) query rows and walks the 64-key tiles that
// its rows see, with the running maximum m and sum l of a softmax:
//   S = Q K^T (tcgen05, accumulator in TMEM, two buffers)
//   p = 2^(x - m) in FP32, l += sum p, P = bf16(p) over S's columns in TMEM
//   O += P V (tcgen05, A operand from TMEM)
// Roles: one warp issues TMA loads, one the MMAs, four own the rows (a thread
// per row, so row maxima and sums need no exchange).  Two CTAs share an SM: one's
// softmax runs under the other's products.
//
// What bounds it is the chain scores - softmax - values of a CTA.  8192 causal
// tokens, 32/8 heads of 128, take 550 us kept up for seconds (1000 TFLOP/s, 72% of
// the sustained rate of a bf16 GEMM, both at the power cap) and 472 to 487 in short
// runs (1130 to 1163, 70% of its burst rate).  With 128-key tiles and one S buffer
// (P lies over S) the next scores waited for the product that reads P: 530 in short
// runs.  With 64-key tiles S(j + 1) is there before the softmax of S(j) ends,
// although 64 columns leave the scores' product bound by its operands' fetches (48
// cycles where 32 would do).  Two threads to a row instead of one gained nothing
// (they meet once a tile).
//
// O is rescaled only when a row's maximum has grown by more than 2^8 over the
// one in use (the sums then stay far inside FP32's range); otherwise the old
// reference stays.  P is rounded to bf16 as the second product's operand: half a
// step of each probability, of the same size as rounding the result.
//
// Few rows over many keys (a decode step): the key tiles are split over several
// CTAs whose normalised FP32 results and log sums are joined by a second
// kernel.  There what P's rounding left follows as a second operand: the few
// results of such a call show every rounding, and the products are not what
// bounds it (one token over 8192 keys, 32/8 heads, 4 sequences: 28.8 us instead
// of 26.1, error against 64 bits 1.7e-3 instead of 2.3e-3).  Small calls without
// splits do so too (few_results).
#include <cuda_bf16.h>
#include <cstdint>
#include <map>
#include <mutex>

#include "fl_attn.cuh"

namespace fl {
namespace attn {

constexpr int kFwdThreads = 192;
constexpr int kKeys = 64;           // keys of a streamed tile
constexpr float kRescale = 8.0f;   // growth of the maximum (in powers of two) that rescales O

template <int HD>
struct Fwd {
  static constexpr int kStages = HD == 64 ? 4 : 2;       // K and V tiles in flight
  static constexpr int kQBytes = HD / 64 * kTile * 128;
  static constexpr int kTileBytes = HD / 64 * kKeys * 128;
  static constexpr int kSmem = kQBytes + 2 * kStages * kTileBytes + 256;
  static constexpr int kTmem = 256;                      // two S (P over each) + O
};

struct FwdArgs {
  Shape s;
  __nv_bfloat16* out;   // [B, Sq, Hq, D]
  float* lse;           // [B, Sq, Hq]
  float* part_o;        // [splits][B Sq Hq][D] (splits > 1)
  float* part_lse;      // [splits][B Sq Hq]
  uint32_t* status;
  int tiles, splits;
};

struct __align__(16) FwdBars {
  uint64_t q_full, pv_done, all_done;
  uint64_t s_full[2], p_full[2];       // of the two S buffers
  uint64_t k_full[4], v_full[4], k_empty[4], v_empty[4];
  uint64_t v_clear[2];                 // of the first and the last tile
  uint32_t tmem, abort_word;
};

// kFine: P in two bf16 parts.
template <int HD, int kMode, bool kFine>
__global__ void __launch_bounds__(kFwdThreads, 2)
    fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const FwdArgs a) {
  using C = Fwd<HD>;
  constexpr bool kBias = kMode != kPlain;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* qs = smem;
  uint8_t* ks = qs + C::kQBytes;
  uint8_t* vs = ks + C::kStages * C::kTileBytes;
  FwdBars* bars = reinterpret_cast<FwdBars*>(vs + C::kStages * C::kTileBytes);
  volatile uint32_t* abort_word = &bars->abort_word;
  // Broadcast so that the compiler knows a warp to be of one mind.
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Shape& s = a.s;

  // Late tiles first: under a causal mask they see the most keys.
  const int per = s.Hkv * s.groups * s.B * a.splits;
  const int tile = a.tiles - 1 - static_cast<int>(blockIdx.x) / per;
  int rest = static_cast<int>(blockIdx.x) % per;
  const int hg = rest % (s.Hkv * s.groups);
  rest /= s.Hkv * s.groups;
  const int b = rest % s.B, split = rest / s.B;
  const int kvh = hg / s.groups;
  const int h0 = hg << s.lgp;
  const int t0 = tile * (kTile >> s.lgp);

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->pv_done, 1);
    mbar_init(&bars->all_done, 1);
    mbar_init(&bars->v_clear[0], 1);
    mbar_init(&bars->v_clear[1], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], 4);
    }
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->v_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
      mbar_init(&bars->v_empty[i], 1);
    }
    bars->abort_word = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem, C::kTmem);
    tmem_relinquish();
  }
  // Every warp finds the tile's key range itself.
  const Range r = tile_range(s, b, t0, kTile >> s.lgp);
  int k_first = 0, n = 0;
  if (r.min_lo < r.max_hi) {
    k_first = r.min_lo / kKeys;
    n = (r.max_hi + kKeys - 1) / kKeys - k_first;
  }
  if (a.splits > 1) {
    const int from = static_cast<int>(static_cast<int64_t>(n) * split / a.splits);
    const int to = static_cast<int>(static_cast<int64_t>(n) * (split + 1) / a.splits);
    k_first += from;
    n = to - from;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_s = bars->tmem, tmem_o = bars->tmem + 2 * kKeys;

  auto wait = [&](uint64_t* bar, int phase, uint32_t bit) {
    return mbar_wait_short_warp(bar, phase & 1, abort_word, a.status, bit);
  };
  // Values that no row of the tile sees may be anything, and 0 times infinity is
  // not 0: where they share a key tile with seen ones (the walk's first and last
  // tile at most) they are cleared.  Past the last key the loads bring zeros.
  auto edge = [&](int j) {
    const int key0 = (k_first + j) * kKeys;
    return key0 < r.min_lo || (key0 + kKeys > r.max_hi && r.max_hi < s.Sk);
  };

  if (warp == 0) {
    if (n > 0) {
      if (elected()) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        mbar_arrive_expect_tx(&bars->q_full, C::kQBytes);
        for (int c = 0; c < HD / 64; ++c) tma_load_4d(qs + c * kTile * 128, &tm_q, 64 * c, h0, t0, b, &bars->q_full);
      }
      __syncwarp();
      int kn = 0, vn = 0;  // loads issued
      auto clear = [&](int j) -> bool {
        const int st = j % C::kStages, key0 = (k_first + j) * kKeys;
        if (!wait(&bars->v_full[st], j / C::kStages, kStatusTimeoutFull)) return false;
        uint4* tile = reinterpret_cast<uint4*>(vs + st * C::kTileBytes);   // chunks of kKeys rows of 8
        for (int i = lane; i < C::kTileBytes / 16; i += 32) {
          const int key = key0 + (i >> 3) % kKeys;
          if (key < r.min_lo || key >= r.max_hi) tile[i] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->v_clear[j ? 1 : 0]);
        return true;
      };
      for (int j = 0; j < n; ++j) {
        const int st = j % C::kStages;
        const int key = (k_first + j) * kKeys;
        // The first tile is cleared when the second's loads are under way.
        if (j == 2 && edge(0) && !clear(0)) break;
        if (j >= C::kStages && !wait(&bars->k_empty[st], j / C::kStages - 1, kStatusTimeoutEmpty)) break;
        if (elected()) {
          mbar_arrive_expect_tx(&bars->k_full[st], C::kTileBytes);
          for (int c = 0; c < HD / 64; ++c)
            tma_load_4d(ks + st * C::kTileBytes + c * kKeys * 128, &tm_k, 64 * c, kvh, key, b, &bars->k_full[st]);
        }
        __syncwarp();
        ++kn;
        if (j >= C::kStages && !wait(&bars->v_empty[st], j / C::kStages - 1, kStatusTimeoutEmpty)) break;
        if (elected()) {
          mbar_arrive_expect_tx(&bars->v_full[st], C::kTileBytes);
          for (int c = 0; c < HD / 64; ++c)
            tma_load_4d(vs + st * C::kTileBytes + c * kKeys * 128, &tm_v, 64 * c, kvh, key, b, &bars->v_full[st]);
        }
        __syncwarp();
        ++vn;
      }
      if (vn == n) {
        bool ok = n > 2 || !edge(0) || clear(0);
        if (ok && n > 1 && edge(n - 1)) clear(n - 1);
      }
      // No copy may be in flight when the CTA leaves.
      uint32_t none = 0;
      mbar_wait(&bars->q_full, 0, &none, a.status, kStatusTimeoutDrain);
      for (int i = max(kn - C::kStages, 0); i < kn; ++i)
        mbar_wait(&bars->k_full[i % C::kStages], (i / C::kStages) & 1, &none, a.status, kStatusTimeoutDrain);
      for (int i = max(vn - C::kStages, 0); i < vn; ++i)
        mbar_wait(&bars->v_full[i % C::kStages], (i / C::kStages) & 1, &none, a.status, kStatusTimeoutDrain);
      __syncwarp();
    }
  } else if (warp == 1) {
    // The whole warp walks and one lane issues: operands stay uniform, and the
    // issue takes few slots of the scheduler that the softmax warps share.
    if (n > 0) {
      const uint32_t id_s = idesc_bf16_f32(kTile, kKeys), id_o = idesc_bf16_f32_bmn(kTile, HD);
      const uint64_t dq = sdesc_kmajor_sw128(smem_u32(qs)), dk = sdesc_kmajor_sw128(smem_u32(ks));
      const uint64_t dv = cols_desc<kKeys>(smem_u32(vs));
      auto scores = [&](int j) -> bool {
        const int st = j % C::kStages;
        if (!wait(&bars->k_full[st], j / C::kStages, kStatusTimeoutFull)) return false;
        tc_fence_after();
        if (elected()) {
          mma_rows<HD, kKeys>(tmem_s + (j & 1) * kKeys, dq, dk + st * (C::kTileBytes >> 4), id_s);
          tc_commit(&bars->k_empty[st]);
          tc_commit(&bars->s_full[j & 1]);
        }
        __syncwarp();
        return true;
      };
      bool ok = wait(&bars->q_full, 0, kStatusTimeoutFull) && scores(0) && (n == 1 || scores(1));
      for (int j = 0; j < n && ok; ++j) {
        const int st = j % C::kStages;
        if (!wait(&bars->v_full[st], j / C::kStages, kStatusTimeoutFull) ||
            ((j == 0 || j + 1 == n) && edge(j) && !wait(&bars->v_clear[j ? 1 : 0], 0, kStatusTimeoutFull)) ||
            !wait(&bars->p_full[j & 1], j >> 1, kStatusTimeoutFull))
          break;
        tc_fence_after();
        if (elected()) {
          const uint32_t p = tmem_s + (j & 1) * kKeys;
          mma_cols<HD, kKeys>(tmem_o, p, dv + st * (C::kTileBytes >> 4), id_o, j > 0);
          if constexpr (kFine)
            mma_cols<HD, kKeys>(tmem_o, p + kKeys / 2, dv + st * (C::kTileBytes >> 4), id_o, true);
          tc_commit(&bars->v_empty[st]);
          tc_commit(&bars->pv_done);
        }
        __syncwarp();
        // P(j) lies in the columns of S(j + 2): the product that reads it has to
        // be done, which it is while the softmax of S(j + 1) goes on.
        if (j + 2 < n) ok = wait(&bars->pv_done, j, kStatusTimeoutAccum) && scores(j + 2);
      }
      // The products still under way read shared memory and TMEM.
      if (elected()) tc_commit(&bars->all_done);
      uint32_t none = 0;
      mbar_wait(&bars->all_done, 0, &none, a.status, kStatusTimeoutDrain);
      __syncwarp();
    }
  } else {
    const int quarter = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int row = quarter * 32 + lane;
    const int tok = t0 + (row >> s.lgp), head = h0 + (row & ((1 << s.lgp) - 1));
    int lo = 0, hi = 0;
    if (tok < s.Sq) row_range(s, b, tok, lo, hi);
    const float slope2 = has_slopes(kMode) ? s.slopes[head] * kLog2e : 0.f;
    const int qpos = tok + s.Sk - s.Sq;
    const float mult = kBias ? 1.0f : s.sl2;   // from what TMEM holds to powers of two
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int key0 = (k_first + j) * kKeys;
      const uint32_t at_s = tmem_s + (j & 1) * kKeys + lanes;
      const bool whole = r.max_lo <= key0 && r.min_hi >= key0 + kKeys;
      if (!mbar_wait_short_warp(&bars->s_full[j & 1], (j >> 1) & 1, abort_word, a.status, kStatusTimeoutAccum)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // The row's scores, in registers from here on.
      uint32_t v[kKeys];
#pragma unroll
      for (int c = 0; c < kKeys; c += 32) tmem_ld_32x32b_x32(at_s + c, reinterpret_cast<uint32_t(&)[32]>(v[c]));
      tmem_wait_ld();
      if constexpr (kBias) {
        [[maybe_unused]] const float from_key0 = static_cast<float>(qpos - key0);
        const uint64_t sl2_2 = pair(s.sl2, s.sl2), cap2_2 = pair(s.cap2, s.cap2);
#pragma unroll
        for (int i = 0; i < kKeys; i += 2) {
          uint64_t x = pair(v[i], v[i + 1]);
          x = has_cap(kMode) ? capped2(s, cap_r2(cap_u2(cap_arg2(s, x))), cap2_2) : mul2(x, sl2_2);
          if constexpr (has_slopes(kMode))
            x = fma2(pair(-slope2, -slope2), pair(fabsf(from_key0 - i), fabsf(from_key0 - (i + 1))), x);
          float x0, x1;
          unpair(x, x0, x1);
          v[i] = __float_as_uint(x0);
          v[i + 1] = __float_as_uint(x1);
        }
      }
      if (!whole) {
        const int lo_c = lo - key0, hi_c = hi - key0;
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
          if (i < lo_c || i >= hi_c) v[i] = 0xff800000u;
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kKeys; i += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          m4[e] = fmaxf(m4[e], fmaxf(__uint_as_float(v[i + e]), __uint_as_float(v[i + 4 + e])));
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * mult;
      if (j == 0) {
        m = mx;
      } else {
        const bool grow = mx > m + kRescale;
        if (__any_sync(0xffffffffu, grow)) {
          // O is at rest once P(j - 1) V is done (P(j - 2) V is, or S(j) would not be).
          if (!mbar_wait_short_warp(&bars->pv_done, (j - 1) & 1, abort_word, a.status, kStatusTimeoutAccum)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float by = grow ? ex2(m - mx) : 1.0f;
          if (grow) m = mx;
          l *= by;
#pragma unroll 1
          for (int c = 0; c < HD; c += 16) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(tmem_o + lanes + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
            tmem_st_32x32b_x16(tmem_o + lanes + c, o);
          }
          tmem_wait_st();
        }
      }
      const float neg = m == -INFINITY ? 0.f : -m;
      const uint64_t mult_2 = pair(mult, mult), neg_2 = pair(neg, neg);
      uint64_t sum0 = 0, sum1 = 0;   // (0, 0)
#pragma unroll
      for (int c = 0; c < kKeys; c += 32) {
        uint32_t w[16];
        [[maybe_unused]] uint32_t u[16];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float x0, x1, x2, x3;
          unpair(fma2(pair(v[c + 2 * i], v[c + 2 * i + 1]), mult_2, neg_2), x0, x1);
          unpair(fma2(pair(v[c + 2 * i + 2], v[c + 2 * i + 3]), mult_2, neg_2), x2, x3);
          if constexpr (has_cap(kMode))            // two of four: the tanh keeps the special units busy
            ex2_pair(x0, x1, x0, x1);
          else
            x0 = ex2(x0), x1 = ex2(x1);
          x2 = ex2(x2), x3 = ex2(x3);
          sum0 = add2(sum0, pair(x0, x1));
          sum1 = add2(sum1, pair(x2, x3));
          w[i] = pack_bf16x2(x0, x1);
          w[i + 1] = pack_bf16x2(x2, x3);
          if constexpr (kFine) {                            // what the rounding left, to be added as a second part
            u[i] = pack_bf16x2(x0 - __uint_as_float(w[i] << 16), x1 - __uint_as_float(w[i] & 0xFFFF0000u));
            u[i + 1] = pack_bf16x2(x2 - __uint_as_float(w[i + 1] << 16), x3 - __uint_as_float(w[i + 1] & 0xFFFF0000u));
          }
        }
        if constexpr (kFine) tmem_st_32x32b_x16(at_s + kKeys / 2 + c / 2, u);
        tmem_st_32x32b_x16(at_s + c / 2, w);
      }
      float l0, l1;
      unpair(add2(sum0, sum1), l0, l1);
      l += l0 + l1;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full[j & 1]);
    }
    // A barrier of its own: of pv_done's last two phases either may be the current one here.
    if (n > 0 && ok) ok = mbar_wait_short_warp(&bars->all_done, 0, abort_word, a.status, kStatusTimeoutAccum);
    tc_fence_after();
    if (n == 0 || ok) {
      const int64_t at = (static_cast<int64_t>(b) * s.Sq + tok) * s.Hq + head;
      const int64_t rows = static_cast<int64_t>(s.B) * s.Sq * s.Hq;
      const bool live = tok < s.Sq, seen = n > 0 && l != 0.f;
      const float inv = seen ? 1.0f / l : 0.f;
      if (live) {
        const float lse = seen ? (m + log2f(l)) * kLn2 : -INFINITY;
        if (a.splits > 1)
          a.part_lse[split * rows + at] = lse;
        else
          a.lse[at] = lse;
      }
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t v[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(tmem_o + lanes + c, v);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = seen ? __float_as_uint(__uint_as_float(v[i]) * inv) : 0u;
        if (!live) continue;
        if (a.splits > 1) {
          float4* o = reinterpret_cast<float4*>(a.part_o + (split * rows + at) * s.D + c);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + 4 * i < s.D)
              o[i] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                 __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
        } else {
          uint4* o = reinterpret_cast<uint4*>(a.out + at * s.D + c);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + 8 * i < s.D) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack_bf16x2(__uint_as_float(v[8 * i + 2 * e]), __uint_as_float(v[8 * i + 2 * e + 1]));
              o[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(bars->tmem, C::kTmem);
  }
}

// Joins the splits of a row: weights 2^(lse_s - max) over their sum, splits in
// order.  16 lanes to a row, 8 columns to a lane; the lanes share the log sums.
__global__ void __launch_bounds__(128) join_kernel(const float* __restrict__ part_o,
                                                   const float* __restrict__ part_lse, int splits, int64_t rows, int D,
                                                   __nv_bfloat16* __restrict__ out, float* __restrict__ lse) {
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 4;
  const int sub = threadIdx.x & 15, d = sub * 8;
  griddep_wait();
  const int64_t at = row < rows ? row : rows - 1;
  float top = -INFINITY, sum = 0.f;
  for (int i = sub; i < splits; i += 16) top = fmaxf(top, part_lse[i * rows + at]);
#pragma unroll
  for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float base = top == -INFINITY ? 0.f : top;
  for (int i = sub; i < splits; i += 16) sum += ex2((part_lse[i * rows + at] - base) * kLog2e);
#pragma unroll
  for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (row >= rows) return;
  float o[8] = {};
  if (d < D) {
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
      const float4* p = reinterpret_cast<const float4*>(part_o + (i * rows + row) * D + d);
      const float4 x = p[0], y = p[1];
      const float w = ex2((part_lse[i * rows + row] - base) * kLog2e);
      o[0] += w * x.x, o[1] += w * x.y, o[2] += w * x.z, o[3] += w * x.w;
      o[4] += w * y.x, o[5] += w * y.y, o[6] += w * y.z, o[7] += w * y.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    *reinterpret_cast<uint4*>(out + row * D + d) =
        make_uint4(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv),
                   pack_bf16x2(o[4] * inv, o[5] * inv), pack_bf16x2(o[6] * inv, o[7] * inv));
  }
  if (sub == 0) lse[row] = sum == 0.f ? -INFINITY : top + log2f(sum) * kLn2;
}

// Splits of the key tiles: none while the row tiles fill half the SMs of a B200
// (its 148 are constants here: the workspace's size depends on the arguments
// alone); else towards two CTAs per SM, each keeping two key tiles at least.
// Measured unsplit / split, 32/8 heads of 128, one token in each sequence:
//   8192 keys:  32 row tiles 117 / 35 us, 72 119 / 58, 80 119 / 69, 128 125 / 99, 144 130 / 104
//   2048 keys:  32 31 / 21, 72 31 / 21, 80 33 / 25, 128 37 / 34
// and causal tokens:  64 row tiles of 1024 keys 22 / 24, of 2048 33 / 24; 76 of 2432
// 38 / 28; 128 of 2048 35 / 34.  So the border at half the SMs costs calls of 75 to
// 148 row tiles up to 42% of their time with one token and 28% with more.
int fwd_splits(int64_t ctas, int Sk) {
  const int64_t key_tiles = (Sk + kTile - 1) / kTile;
  if (ctas > 74 || key_tiles < 4) return 1;
  int64_t n = 296 / ctas;
  if (n > key_tiles / 2) n = key_tiles / 2;
  return n < 1 ? 1 : static_cast<int>(n);
}

int packed_log2(int Hq, int Hkv) {
  const int g = Hq / Hkv;
  if (g & (g - 1)) return 0;
  int l = 0;
  while ((1 << l) < g && l < 6) ++l;
  return l;
}

void fill_shape(Shape& s, int B, int Sq, int Sk, int Hq, int Hkv, int D, const int* begin, const int* end, float scale,
                float cap, const float* slopes) {
  s.B = B;
  s.Sq = Sq;
  s.Sk = Sk;
  s.Hq = Hq;
  s.Hkv = Hkv;
  s.D = D;
  s.lgp = packed_log2(Hq, Hkv);
  s.groups = (Hq / Hkv) >> s.lgp;
  s.scale = scale;
  s.sl2 = scale * kLog2e;
  s.cap2 = cap * kLog2e;
  s.icap2 = cap != 0.f ? 2.0f * kLog2e * scale / cap : 0.f;
  s.begin = begin;
  s.end = end;
  s.slopes = slopes;
}

int64_t fwd_ctas(int B, int Sq, int Hq, int Hkv) {
  const int lgp = packed_log2(Hq, Hkv);
  const int64_t tiles = (static_cast<int64_t>(Sq) + (kTile >> lgp) - 1) / (kTile >> lgp);
  return tiles * B * (Hq >> lgp);
}

template <int HD, int kMode, bool kFine>
int launch_fwd(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FwdArgs& a, int64_t grid,
               cudaStream_t stream) {
  int rc = allow_smem(reinterpret_cast<const void*>(&fwd_kernel<HD, kMode, kFine>), Fwd<HD>::kSmem);
  if (rc) return rc;
  fwd_kernel<HD, kMode, kFine><<<static_cast<unsigned>(grid), kFwdThreads, Fwd<HD>::kSmem, stream>>>(q, k, v, a);
  return FL_OK;
}

template <int HD, bool kFine>
int launch_fwd_mode(int mode, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FwdArgs& a,
                    int64_t grid, cudaStream_t stream) {
  return mode == kCappedSlopes ? launch_fwd<HD, kCappedSlopes, kFine>(q, k, v, a, grid, stream)
         : mode == kCapped     ? launch_fwd<HD, kCapped, kFine>(q, k, v, a, grid, stream)
         : mode == kSlopes     ? launch_fwd<HD, kSlopes, kFine>(q, k, v, a, grid, stream)
                               : launch_fwd<HD, kPlain, kFine>(q, k, v, a, grid, stream);
}

}  // namespace attn

// Raises `kernel`'s dynamic shared-memory limit once per device.
int allow_smem(const void* kernel, int bytes) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, bool> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return set_error(FL_ERR_CUDA, "cudaGetDevice: %s", cudaGetErrorString(e));
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({kernel, dev})) return FL_OK;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return set_error(FL_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  done[{kernel, dev}] = true;
  return FL_OK;
}

int attn_map(CUtensorMap* map, const void* base, int64_t batch_stride, int64_t token_stride, int64_t head_stride, int B,
             int S, int H, int D, int heads, int tokens) {
  // A dimension of one element may have any stride: give it one that the map accepts.
  const uint64_t row = static_cast<uint64_t>(D) * 2;
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(H), static_cast<uint64_t>(S),
                            static_cast<uint64_t>(B)};
  const uint64_t strides[3] = {H > 1 ? static_cast<uint64_t>(head_stride) * 2 : row,
                               S > 1 ? static_cast<uint64_t>(token_stride) * 2 : row,
                               B > 1 ? static_cast<uint64_t>(batch_stride) * 2 : row};
  const uint32_t box[4] = {64, static_cast<uint32_t>(heads), static_cast<uint32_t>(tokens), 1};
  return make_tensor_map(map, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, dims, strides, box,
                         CU_TENSOR_MAP_SWIZZLE_128B);
}

int attn_check(const char* who, int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int D, const int64_t* strides,
               int tensors, const void* const* bases, const int* begin, const int* end, float scale, float cap) {
  if (B < 0 || Sq < 0 || Sk < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv)
    return set_error(FL_ERR_ARG, "%s: bad batch, length or head counts", who);
  if (B > (1 << 16) || Sq > (1 << 30) || Sk > (1 << 30) || Hq > (1 << 12))
    return set_error(FL_ERR_ARG, "%s: batch, length or head count too large", who);
  if (D < 8 || D > 128 || D % 8) return set_error(FL_ERR_ARG, "%s: head size must be a multiple of 8 in [8, 128]", who);
  // scale log2(e) has to be finite.
  if (!(scale > 0.f) || scale > 2.3e38f) return set_error(FL_ERR_ARG, "%s: scale must be in (0, 2.3e38]", who);
  // The tanh's error, a few 1e-7, times the cap stays under a quarter of P's half step.
  if (!(cap >= 0.f) || cap > 1024.f || (cap > 0.f && scale / cap > 1.0e30f))
    return set_error(FL_ERR_ARG, "%s: the cap must be 0, or at most 1024 and not too small for the scale", who);
  if (B == 0 || Sq == 0) return FL_OK;
  if (!begin || !end) return set_error(FL_ERR_ARG, "%s: null pointer", who);
  if (attn::fwd_ctas(static_cast<int>(B), static_cast<int>(Sq), Hq, Hkv) > (int64_t(1) << 30))
    return set_error(FL_ERR_ARG, "%s: too many row tiles", who);
  if (!strides) return set_error(FL_ERR_ARG, "%s: null strides", who);
  const int64_t S[4] = {Sq, Sk, Sk, Sq};
  const int H[4] = {Hq, Hkv, Hkv, Hq};
  for (int i = 0; i < tensors; ++i) {
    if (S[i] == 0) continue;
    if (!bases[i] || (reinterpret_cast<uintptr_t>(bases[i]) & 15u))
      return set_error(FL_ERR_ARG, "%s: tensors must be non-null and 16-byte aligned", who);
    const int64_t n[3] = {B, S[i], H[i]};
    for (int d = 0; d < 3; ++d) {
      const int64_t st = strides[3 * i + d];
      if (n[d] > 1 && (st <= 0 || st % 8 || st >= (int64_t(1) << 38)))
        return set_error(FL_ERR_ARG, "%s: strides must be positive multiples of 8 elements", who);
    }
  }
  return FL_OK;
}

}  // namespace fl

using namespace fl;

extern "C" {

size_t fl_attn_fwd_workspace_bytes(int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int D) {
  if (B <= 0 || Sq <= 0 || Sk <= 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 8 || B > (1 << 16) || Sq > (1 << 30) ||
      Sk > (1 << 30))
    return 0;
  const int splits = attn::fwd_splits(attn::fwd_ctas((int)B, (int)Sq, Hq, Hkv), (int)Sk);
  if (splits == 1) return 0;
  return static_cast<size_t>(splits) * B * Sq * Hq * (D + 1) * sizeof(float);
}

int fl_attn_fwd(const uint16_t* q, const uint16_t* k, const uint16_t* v, const int64_t* strides, int64_t B, int64_t Sq,
                int64_t Sk, int Hq, int Hkv, int D, const int32_t* begin, const int32_t* end, float scale,
                float softcap, const float* slopes, uint16_t* out, float* lse, void* workspace,
                size_t workspace_bytes, void* stream) {
  const void* bases[3] = {q, k, v};
  int rc = attn_check("fl_attn_fwd", B, Sq, Sk, Hq, Hkv, D, strides, 3, bases, begin, end, scale, softcap);
  if (rc || B == 0 || Sq == 0) return rc;
  if (!out || !lse || (reinterpret_cast<uintptr_t>(out) & 15u))
    return set_error(FL_ERR_ARG, "fl_attn_fwd: out and lse must be given, out 16-byte aligned");
  const size_t need = fl_attn_fwd_workspace_bytes(B, Sq, Sk, Hq, Hkv, D);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return set_error(FL_ERR_ARG, "fl_attn_fwd: workspace missing, short or not 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  attn::FwdArgs a{};
  attn::fill_shape(a.s, (int)B, (int)Sq, (int)Sk, Hq, Hkv, D, begin, end, scale, softcap, slopes);
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  int dev = 0;
  if ((rc = current_context(&dev))) return rc;
  if (!(a.status = status_word(dev))) return set_error(FL_ERR_CUDA, "fl_attn_fwd: status word unavailable");
  const int pg = 1 << a.s.lgp;
  const int64_t ctas = attn::fwd_ctas((int)B, (int)Sq, Hq, Hkv);
  a.tiles = static_cast<int>(ctas / B / (Hq >> a.s.lgp));
  a.splits = Sk ? attn::fwd_splits(ctas, (int)Sk) : 1;
  const int64_t rows = B * Sq * Hq;
  if (a.splits > 1) {
    a.part_o = static_cast<float*>(workspace);
    a.part_lse = a.part_o + a.splits * rows * D;
  }
  CUtensorMap mq{}, mk{}, mv{};
  if ((rc = attn_map(&mq, q, strides[0], strides[1], strides[2], (int)B, (int)Sq, Hq, D, pg, attn::kTile >> a.s.lgp)))
    return rc;
  if (Sk && ((rc = attn_map(&mk, k, strides[3], strides[4], strides[5], (int)B, (int)Sk, Hkv, D, 1, attn::kKeys)) ||
             (rc = attn_map(&mv, v, strides[6], strides[7], strides[8], (int)B, (int)Sk, Hkv, D, 1, attn::kKeys))))
    return rc;
  const int mode = (softcap != 0.f ? attn::kCapped : attn::kPlain) + (slopes ? attn::kSlopes : 0);
  const int64_t grid = ctas * a.splits;
  if (a.splits > 1 || attn::few_results(rows, Sk))
    rc = D <= 64 ? attn::launch_fwd_mode<64, true>(mode, mq, mk, mv, a, grid, st)
                 : attn::launch_fwd_mode<128, true>(mode, mq, mk, mv, a, grid, st);
  else
    rc = D <= 64 ? attn::launch_fwd_mode<64, false>(mode, mq, mk, mv, a, grid, st)
                 : attn::launch_fwd_mode<128, false>(mode, mq, mk, mv, a, grid, st);
  if (rc) return rc;
  if (a.splits > 1) {
    // A programmatic dependent: its launch overlaps the attention kernel, whose results it waits for.
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((rows * 16 + 127) / 128));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t le = cudaLaunchKernelEx(&cfg, attn::join_kernel, static_cast<const float*>(a.part_o),
                                              static_cast<const float*>(a.part_lse), a.splits, rows, D, a.out, lse);
    if (le != cudaSuccess) return set_error(FL_ERR_CUDA, "fl_attn_fwd: %s", cudaGetErrorString(le));
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FL_ERR_CUDA, "fl_attn_fwd: %s", cudaGetErrorString(e));
  return FL_OK;
}

}  // extern "C"
