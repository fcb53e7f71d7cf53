// Forward pass: o_i = sum_j p_ij v_j with p the softmax over the visible keys, on the tensor cores.
//
// An SM has two groups of four softmax warps, each with a tile of 128 queries by 128 keys under way, so that one group's
// exponentials run under the other group's products:
//   * pairs (PAIR): the groups have two neighbouring query tiles and walk the same keys. With heads of up to 64 (ALONE) they are CTAs of
//     their own, each with half of the SM's tensor memory, so that one's start and end (6 us of setting up, first loads and writing) run
//     under the other's work: 16 x 2048 tokens, 6 heads 131 -> 117 us, 8 x 512 26.6 -> 18.4; walks over 16384 keys lose 7 % (203 -> 218);
//   * halves: both have the same query tile, one the even and one the odd key tiles, and are added up at the end. Taken where
//     pairs would leave SMs idle; the keys may then also be split over CTAs (`splits`), whose parts a second kernel adds up.
// Bound by the softmax warps' arithmetic and exponentials: a tile of 128 x 128 takes 1430 (heads of 64) and 1910 clocks (of 128) of an SM
// in a long walk, of which its products need 700 and 1400 at the rate that a large product reaches here, and its exponentials 770.
// Whole calls with a cold L2: 8192 tokens, 16 heads on 4 of 128, causal: 240 to 267 us from card to card (1150 to 1030 TFLOP/s); 1024 queries after
// 15360: 137 to 141 us.
// Warp roles:
//   warp 0      TMA producer: query tiles once, then two-stage rings of key and value tiles
//   warp 1      tcgen05.mma: S_w = Q_w K^T into TMEM, O_w += P_w V with P_w read from TMEM
//   warps 2-3   pass the value tiles on; in those where not all keys are visible to all queries, values that are no numbers, and
//               those of keys past the sequence's length, are set to zero first, since zero weights would not take them out
//   warps 4-7, 8-11   softmax, one query per thread (TMEM lane = query)
// Heads of up to 64 have columns for scores and weights apart, so that the scores of a group's next tile are ready when it is done
// with one; with wider heads, whose sums take the room, weights lie over the scores, and the next scores wait for the product.
// P is bf16 (every weight is off by 2^-8 of itself at most, which averages out over the keys); fp32 sums take the weights before
// rounding. The running maximum is lazy: sums are rescaled only when it has grown by more than 2^8.
// TMEM: S_0 0-127, S_1 128-255, O_0 and O_1 from 256 on, P_0 384-447, P_1 448-511 or over the scores; ALONE: S 0-127, O 128-191, P 192-255.
#include <algorithm>
#include <type_traits>

#include "attention_tiles.cuh"

namespace tb {
namespace {

// PAIR with heads of up to 64: one group and one query tile, two CTAs per SM
constexpr bool alone(int db, bool pair) { return pair && db == 1; }
constexpr int fwd_threads(int db, bool pair) { return alone(db, pair) ? 256 : 384; }
// registers of a thread of the first four warps and of the others; 128 + 200 is twice the 128 that 256 threads are launched with, and
// 88 + 2 * 208 three times the 168 of 384
constexpr int fwd_few(int db, bool pair) { return alone(db, pair) ? 56 : 88; }
constexpr int fwd_many(int db, bool pair) { return alone(db, pair) ? 200 : 208; }
constexpr float FW_LAZY = 8.f;
constexpr int FW_POLY = 4;  // of so many pairs of exponentials one is a polynomial (2: 5 to 10 % slower, 3: the same)

struct FwdParams {
  AttentionShape a;
  __nv_bfloat16 *out, *rest;
  float* lse;
  float* part;  // [splits, B, H, T, 64 * DB] sums, then [splits, B, H, T, 2] maxima and weights
  const __nv_bfloat16* v;
  long long vr, vh, vb;
  const float *k_scales, *v_scales;  // [B, G, blocks]
  int blocks, splits;
  float scale2;  // scale * log2(e)
  int* status;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int DB, bool PAIR, bool SCALED>
__global__ void __launch_bounds__(fwd_threads(DB, PAIR), alone(DB, PAIR) ? 2 : 1) attention_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                                                                      const __grid_constant__ CUtensorMap tmV, const FwdParams p) {
  constexpr bool ALONE = alone(DB, PAIR);
  constexpr int QT = PAIR && !ALONE ? 2 : 1, TILE = DB * AT_BOX;
  // TMEM columns of the groups' scores, weights and sums. APART: weights do not lie over the scores
  constexpr bool APART = DB == 1;
  constexpr int S_AT[2] = {0, 128}, P_AT[2] = {ALONE ? 192 : APART ? 384 : 0, APART ? 448 : 128}, O_AT[2] = {ALONE ? 128 : 256, 256 + 64 * DB};
  constexpr uint32_t COLUMNS = ALONE ? 256 : 512;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sK = sQ + QT * TILE, *sV = sK + 2 * TILE;
  __shared__ __align__(8) uint64_t bars[21];
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 7, *v_clean = bars + 9, *s_full = bars + 11,
           *s_read = bars + 13, *p_half = bars + 15, *p_ready = bars + 17, *o_done = bars + 19;
  __shared__ uint32_t tmem_slot;
  __shared__ int special;  // a value that is no number was set to zero
  __shared__ float2 other[AT_M];
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int h = blockIdx.x % p.a.H, b = blockIdx.x / p.a.H, kvh = h / (p.a.H / p.a.G), kv_head = b * p.a.G + kvh;
  const int q0 = (gridDim.y - 1 - blockIdx.y) * QT * AT_M;  // the rows with the most keys start first
  const Visible vis(p.a, b);
  // key tiles of the two groups: group w takes tiles x, x + step, ... below y
  constexpr int step = PAIR ? 1 : 2;
  int2 range[2];
  int j0, j1;
  if constexpr (PAIR) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int t0 = q0 + w * AT_M;
      range[w] = t0 < p.a.T && w < QT ? vis.tiles(t0, min(p.a.T, t0 + AT_M) - 1) : make_int2(0, 0);
    }
    const bool e0 = range[0].x == range[0].y, e1 = range[1].x == range[1].y;
    j0 = e0 ? range[1].x : e1 ? range[0].x : min(range[0].x, range[1].x);
    j1 = e0 ? range[1].y : e1 ? range[0].y : max(range[0].y, range[1].y);
  } else {
    const int2 all = vis.tiles(q0, min(p.a.T, q0 + AT_M) - 1);
    const int n = all.y - all.x, per = (n + p.splits - 1) / p.splits;
    j0 = min(all.y, all.x + (int)blockIdx.z * per);
    j1 = min(all.y, j0 + per);
    range[0] = make_int2(j0, j1);
    range[1] = make_int2(min(j0 + 1, j1), j1);
  }
  auto count = [&](int w) { return (range[w].y - range[w].x + step - 1) / step; };
  auto takes = [&](int w, int j) { return PAIR ? j >= range[w].x && j < range[w].y : ((j - j0) & 1) == w; };
  // tiles whose values are looked through; the queries past T take part, so this holds for whole query tiles
  auto partial = [&](int j) {
    bool some = false;
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if (takes(w, j)) some = some || !vis.whole(q0 + (PAIR ? w : 0) * AT_M, q0 + (PAIR ? w : 0) * AT_M + AT_M - 1, j * AT_M);
    return some;
  };

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 1);
      mbar_init(v_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_ready + i, 128);
      mbar_init(p_half + i, 128);
      mbar_init(s_read + i, 128);
      mbar_init(o_done + i, 1);
      mbar_init(v_clean + i, 64);
    }
    mbar_fence_init();
    special = 0;
  }
  if (warp == 2) {
    tmem_alloc(&tmem_slot, COLUMNS);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = uniform(tmem_slot);
  if (warp < 4) {
  registers_down<fwd_few(DB, PAIR)>();
  if (warp == 0) {
    if (lane == 0 && j1 > j0) {
      prefetch_tmap(&tmQ);
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
      mbar_expect_tx(q_full, QT * TILE);
      for (int w = 0; w < QT; ++w)
        for (int d = 0; d < DB; ++d) tma_load_4d(sQ + w * TILE + d * AT_BOX, &tmQ, q_full, d * 64, q0 + w * AT_M, h, b);
      bool ok = true;
      // keys run one tile ahead of values: the scores of the next tile are issued before the use of these values ends
      for (int u = 0; u <= j1 - j0 && ok; ++u) {
        if (u < j1 - j0) {
          const int s = u & 1;
          if (u >= 2) ok = mbar_wait(k_empty + s, ((u >> 1) & 1) ^ 1);
          if (!ok) break;
          mbar_expect_tx(k_full + s, TILE);
          for (int d = 0; d < DB; ++d) tma_load_4d(sK + s * TILE + d * AT_BOX, &tmK, k_full + s, d * 64, (j0 + u) * AT_M, kvh, b);
        }
        if (u > 0) {
          const int i = u - 1, s = i & 1;
          if (i >= 2) ok = mbar_wait(v_empty + s, ((i >> 1) & 1) ^ 1);
          if (!ok) break;
          mbar_expect_tx(v_full + s, TILE);
          for (int d = 0; d < DB; ++d) tma_load_4d(sV + s * TILE + d * AT_BOX, &tmV, v_full + s, d * 64, (j0 + i) * AT_M, kvh, b);
        }
      }
      // nothing may arrive at the barriers once the block is gone
      for (int u = max(0, j1 - j0 - 2); u < j1 - j0 && ok; ++u) ok = mbar_wait(k_empty + (u & 1), (u >> 1) & 1) && mbar_wait(v_empty + (u & 1), (u >> 1) & 1);
      if (!ok && p.status) *p.status = ST_TIMEOUT_EMPTY;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (j1 > j0) {
      const int ks = (p.a.D + 15) / 16;
      const uint32_t qa = smem_u32(sQ), ka = smem_u32(sK), va = smem_u32(sV);
      int issued[2] = {0, 0}, done[2] = {0, 0};
      // Scores of tile j for group w, behind its read of the last ones (APART), or behind the product that read the weights over them
      auto scores = [&](auto group, int j) {
        constexpr int w = decltype(group)::value;
        if (APART && issued[w] > 0 && !warp_wait(s_read + w, (issued[w] - 1) & 1)) return false;
        tc_fence_after_sync();
        issue([&] {
          scores_product<DB>(tmem + S_AT[w], qa + (PAIR ? w : 0) * TILE, ka + ((j - j0) & 1) * TILE, ks);
          umma_commit(s_full + w);
        });
        ++issued[w];
        return true;
      };
      auto values = [&](auto group, int j) {
        constexpr int w = decltype(group)::value;
        const uint32_t v = va + ((j - j0) & 1) * TILE;
        const bool add = done[w] > 0;
        if (!warp_wait(p_half + w, done[w] & 1)) return false;
        tc_fence_after_sync();
        issue([&] { rows_product<DB, 0, 4>(tmem + O_AT[w], tmem + P_AT[w], v, add, [](int k) { return k * 8; }); });
        if (!warp_wait(p_ready + w, done[w] & 1)) return false;
        tc_fence_after_sync();
        issue([&] {
          rows_product<DB, 4, 4>(tmem + O_AT[w], tmem + P_AT[w], v, true, [](int k) { return k * 8; });
          umma_commit(o_done + w);
        });
        ++done[w];
        return true;
      };
      auto commit = [&](uint64_t* bar) { issue([&] { umma_commit(bar); }); };
      auto k_arrived = [&](int j) { return warp_wait(k_full + ((j - j0) & 1), ((j - j0) >> 1) & 1); };
      constexpr std::integral_constant<int, 0> g0{};
      constexpr std::integral_constant<int, 1> g1{};
      bool ok = warp_wait(q_full, 0) && k_arrived(j0);
      if constexpr (PAIR) {
        if (takes(0, j0)) ok = ok && scores(g0, j0);
        if (!ALONE && takes(1, j0)) ok = ok && scores(g1, j0);
        commit(k_empty);
      } else {
        ok = ok && scores(g0, j0);
        commit(k_empty);
        if (j1 - j0 > 1) {
          ok = ok && k_arrived(j0 + 1) && scores(g1, j0 + 1);
          commit(k_empty + 1);
        }
      }
      auto turn = [&](auto group, int j, int jn) {
        constexpr int w = decltype(group)::value;
        const int s = (j - j0) & 1;
        const bool next = jn < j1 && takes(w, jn);
        if (APART && next && !scores(group, jn)) return false;
        if (takes(w, j) && !(warp_wait(v_clean + s, ((j - j0) >> 1) & 1) && values(group, j))) return false;
        return APART || !next || scores(group, jn);
      };
      for (int j = j0; j < j1 && ok; ++j) {
        const int s = (j - j0) & 1, jn = j + step;
        const bool next = jn < j1;
        if (next) ok = k_arrived(jn);
        if (PAIR || s == 0) ok = ok && turn(g0, j, jn);
        if (!ALONE && (PAIR || s == 1)) ok = ok && turn(g1, j, jn);
        if (next) commit(k_empty + ((jn - j0) & 1));
        commit(v_empty + s);
      }
      if (!ok && p.status) *p.status = ST_TIMEOUT_FULL;
    }
  } else {
    const int tid = threadIdx.x - 64;
    bool ok = true;
    for (int j = j0; j < j1 && ok; ++j) {
      const bool look = partial(j);
      const int s = (j - j0) & 1, keep = vis.length - j * AT_M;
      ok = mbar_wait(v_full + s, ((j - j0) >> 1) & 1);
      if (!ok) break;
      bool found = false;
      for (int i = look ? tid : TILE; i < TILE / 16; i += 64) {
        uint4* x = reinterpret_cast<uint4*>(sV + s * TILE) + i;
        const int row = (i >> 3) & (AT_M - 1);  // 128-byte rows; the swizzle stays within them
        if (row >= keep) {
          *x = make_uint4(0, 0, 0, 0);
          continue;
        }
        uint4 y = *x;
        uint32_t* w = &y.x;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (bf16x2_special(w[e])) {
            bad = true;
            if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
            if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0x0000ffffu;
          }
        if (bad) *x = y;
        found = found || bad;
      }
      if (found) special = 1;
      fence_proxy_async_smem();
      mbar_arrive(v_clean + s);
    }
    if (!ok && p.status) *p.status = ST_TIMEOUT_FULL;
  }
  } else {
    registers_up<fwd_many(DB, PAIR)>();
    const int w = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const int first = q0 + (PAIR ? w : 0) * AT_M, t = first + row;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_base + (w == 0 ? S_AT[0] : S_AT[1]), tP = tmem + lane_base + (w == 0 ? P_AT[0] : P_AT[1]),
                   tO = tmem + lane_base + (w == 0 ? O_AT[0] : O_AT[1]);
    const float c2 = p.scale2;
    const int n = count(w), lo = vis.low(t), hi = vis.high(t);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    // One tile: maximum, then weights, their sums and their bf16 form. MASKED: not all of the tile's keys are visible to all queries.
    auto softmax = [&](auto some, int it, int key) {
      constexpr bool MASKED = decltype(some)::value;
      const int c_lo = lo - key, c_hi = hi - key;  // visible columns
      uint32_t x[4][32];
      float top[4];
      auto chunk_max = [&](uint32_t (&r)[32], int c) {
        if constexpr (MASKED) {
          const uint32_t see = visible_bits(c_lo - 32 * c, c_hi - 32 * c);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(see >> i & 1)) r[i] = 0xff800000u;  // -inf
        }
        float a = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])), e = fmaxf(__uint_as_float(r[2]), __uint_as_float(r[3]));
#pragma unroll
        for (int i = 4; i < 32; i += 4) {
          a = max3(a, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
          e = max3(e, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
        }
        top[c] = fmaxf(a, e);
      };
      tmem_load(tS, x[0], x[1]);
      tmem_load(tS + 64, x[2], x[3]);
      tc_fence_before_sync();
      if (APART) mbar_arrive(s_read + w);
#pragma unroll
      for (int c = 0; c < 4; ++c) chunk_max(x[c], c);
      float f0 = c2, f1 = c2;  // what the scores of the two blocks of 64 keys are multiplied by
      [[maybe_unused]] uint64_t v0 = 0, v1 = 0;
      if constexpr (SCALED) {
        f0 *= p.k_scales[(long long)kv_head * p.blocks + key / 64];
        f1 *= key / 64 + 1 < p.blocks ? p.k_scales[(long long)kv_head * p.blocks + key / 64 + 1] : 0.f;
        const float a = p.v_scales[(long long)kv_head * p.blocks + key / 64];
        const float e = key / 64 + 1 < p.blocks ? p.v_scales[(long long)kv_head * p.blocks + key / 64 + 1] : 0.f;
        v0 = pack_f2(a, a), v1 = pack_f2(e, e);
      }
      const float t0 = fmaxf(top[0], top[1]), t1 = fmaxf(top[2], top[3]);
      // a scale of zero takes no score (minus infinity, of a block without visible keys) to NaN: fmaxf passes over those
      const float mn = SCALED ? max3(m, t0 * f0, t1 * f1) : fmaxf(m, fmaxf(t0, t1) * c2);
      const bool grow = mn > m && (m == -INFINITY || mn - m > FW_LAZY);
      float f = 1.f;
      if (grow) {
        f = m == -INFINITY ? 0.f : ex2(m - mn);  // sums over invisible keys so far are zero
        m = mn;
        l *= f;
      }
      const bool any = __any_sync(0xffffffffu, grow);  // also brings the warp together again
      if (APART && it > 0) {  // the weights' columns and the sums are free again
        if (!warp_wait(o_done + w, (it - 1) & 1)) return false;
        tc_fence_after_sync();
      }
      if (it > 0 && any) {
        for (int c = 0; c < 64 * DB; c += 16) {
          uint32_t o[16];
          tmem_load(tO + c, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
          tmem_st_32x32b_x16(tO + c, o);
        }
      }
      const float ms = m == -INFINITY ? 0.f : m;  // no visible key yet
      const uint64_t mm = pack_f2(-ms, -ms);
      uint64_t sum2 = pack_f2(0.f, 0.f);
      auto weights = [&](uint32_t (&r)[32], int c) {
        const float fc = c < 2 ? f0 : f1;
        [[maybe_unused]] const uint32_t see = MASKED && SCALED ? visible_bits(c_lo - 32 * c, c_hi - 32 * c) : 0u;
        const uint64_t cc = pack_f2(fc, fc);
        uint32_t q[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint64_t y = fma2(pack_f2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), cc, mm);
          uint64_t e;
          if (i % FW_POLY == FW_POLY - 1 && !MASKED) {
            e = exp2_pair(y);
          } else {
            float a, z;
            unpack_f2(y, a, z);
            a = ex2(a);
            z = ex2(z);
            if constexpr (MASKED && SCALED) {  // where a block's scale, zero or no number, was multiplied by minus infinity
              a = see >> (2 * i) & 1 ? a : 0.f;
              z = see >> (2 * i + 1) & 1 ? z : 0.f;
            }
            e = pack_f2(a, z);
          }
          sum2 = add2(sum2, e);
          if constexpr (SCALED) e = mul2(e, c < 2 ? v0 : v1);
          if constexpr (MASKED && SCALED) {  // and a value scale that is no number must not reach queries that do not see its block
            float a, z;
            unpack_f2(e, a, z);
            e = pack_f2(see >> (2 * i) & 1 ? a : 0.f, see >> (2 * i + 1) & 1 ? z : 0.f);
          }
          q[i] = f2_to_bf16x2(e);
        }
        tmem_st_32x32b_x16(tP + 16 * c, q);
        if (c & 1) {  // the product starts on the first half of the keys
          tmem_st_wait();
          tc_fence_before_sync();
          mbar_arrive(c == 1 ? p_half + w : p_ready + w);
        }
      };
#pragma unroll
      for (int c = 0; c < 4; ++c) weights(x[c], c);
      float s0, s1;
      unpack_f2(sum2, s0, s1);
      l += s0 + s1;
      return true;
    };
    for (int it = 0; it < n; ++it) {
      const int key = (range[w].x + it * step) * AT_M;
      ok = warp_wait(s_full + w, it & 1);
      if (!ok) break;
      tc_fence_after_sync();
      if (vis.whole(first, first + AT_M - 1, key)) ok = softmax(std::false_type{}, it, key);
      else ok = softmax(std::true_type{}, it, key);
      if (!ok) break;
    }
    if (ok && n > 0) ok = warp_wait(o_done + w, (n - 1) & 1);
    if (!ok) l = __int_as_float(0x7fc00000);  // a wait has expired: what is handed on is no number
    tc_fence_after_sync();
    float share = 1.f;  // of this group's sums in the row
    float* half = reinterpret_cast<float*>(sK);
    if constexpr (!PAIR) {
      // the second group hands its sums over through the key tiles, which no product reads any more
      const bool both = count(1) > 0;
      if (w == 1 && both) {
        other[row] = make_float2(m, l);
        for (int c = 0; c < 64 * DB; c += 16) {
          uint32_t o[16];
          __syncwarp();
          tmem_load(tO + c, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) half[(c + i) * AT_M + row] = __uint_as_float(o[i]);
        }
      }
      if (both) named_barrier<256>(1);
    }
    if (PAIR || w == 0) {
      float r1 = 0.f;
      const bool both = !PAIR && count(1) > 0;
      if (both) {
        const float2 o = other[row];
        const float mn = fmaxf(m, o.x);
        share = m == -INFINITY ? 0.f : ex2(m - mn);
        r1 = o.x == -INFINITY ? 0.f : ex2(o.x - mn);
        // a row whose scores were no numbers has a sum that is none, whatever its maximum
        l = (m == -INFINITY && l == l ? 0.f : l * (m == -INFINITY ? 1.f : share)) + (o.x == -INFINITY && o.y == o.y ? 0.f : o.y * (o.x == -INFINITY ? 1.f : r1));
        m = mn;
      }
      const bool split = !PAIR && p.splits > 1;
      const float r = split ? 1.f : l == 0.f ? 0.f : 1.f / l;
      const bool inside = t < p.a.T;
      const long long row_at = ((long long)b * p.a.H + h) * p.a.T + t;
      const int padded = (p.a.T + AT_M - 1) / AT_M * AT_M;
      if (p.lse != nullptr && !split && t < padded) p.lse[((long long)b * p.a.H + h) * padded + t] = inside && l != 0.f ? -m - log2f(l) : -INFINITY;
      if (split && inside) {
        const long long rows = (long long)p.a.B * p.a.H * p.a.T;
        float2* ml = reinterpret_cast<float2*>(p.part + p.splits * rows * 64 * DB);
        ml[blockIdx.z * rows + row_at] = make_float2(m, l);
      }
      __nv_bfloat16* o = p.out + (((long long)b * p.a.T + t) * p.a.H + h) * p.a.D;
      float* po = p.part + ((long long)blockIdx.z * p.a.B * p.a.H * p.a.T + row_at) * 64 * DB;
      const bool any = n > 0;
      for (int c = 0; c < 64 * DB; c += 16) {
        uint32_t x[16];
        __syncwarp();
        if (any) {
          tmem_load(tO + c, x);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float y = any ? __uint_as_float(x[i]) : 0.f;
          if (both) y = y * share + half[(c + i) * AT_M + row] * r1;
          x[i] = __float_as_uint(y);
        }
        if (special != 0 && inside) {
          // values that are no numbers were left out of the products of the tiles that are not whole: for the rows that see them
          // they are added here, whatever their (positive) weight
          for (int j = j0; j < j1; ++j) {
            if (!partial(j)) continue;
            const int k0 = max(lo, j * AT_M), k1 = min(hi, j * AT_M + AT_M - 1);
            for (int k = k0; k <= k1; ++k)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (c + i < p.a.D) {
                  const float y = __bfloat162float(p.v[b * p.vb + k * p.vr + kvh * p.vh + c + i]);
                  if (!isfinite(y)) x[i] = __float_as_uint(__uint_as_float(x[i]) + y);
                }
          }
        }
        if (!inside) continue;
        if (split) {
#pragma unroll
          for (int g = 0; g < 4; ++g) reinterpret_cast<uint4*>(po + c)[g] = make_uint4(x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]);
        } else {
          store_row16(o, c, p.a.D, x, r);
          if (p.rest != nullptr) store_rest16(p.rest + (o - p.out), c, p.a.D, x, r);
        }
      }
    }
    if (!ok && p.status) *p.status = ST_TIMEOUT_TMEM;
  }
  __syncwarp();  // the block's barrier counts warps: one whose threads came one by one would count more than once
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 2) tmem_dealloc(tmem, COLUMNS);
}

// Parts of rows whose keys were split over CTAs: a warp per row.
template <int DB>
__global__ void __launch_bounds__(256) attention_join_kernel(const FwdParams p) {
  const long long rows = (long long)p.a.B * p.a.H * p.a.T, row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const float2* ml = reinterpret_cast<const float2*>(p.part + p.splits * rows * 64 * DB);
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[s * rows + row].x);
  float l = 0.f, acc[2 * DB] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float2 x = ml[s * rows + row];
    if (x.x == -INFINITY && x.y == x.y) continue;  // nothing visible there: its sums may not have been formed
    const float f = x.x == -INFINITY ? 1.f : ex2(x.x - m);  // zero times sums that are no numbers is none
    l += x.y * f;
#pragma unroll
    for (int i = 0; i < 2 * DB; ++i) acc[i] += p.part[(s * rows + row) * 64 * DB + lane + 32 * i] * f;
  }
  const int t = row % p.a.T, h = row / p.a.T % p.a.H;
  const long long b = row / ((long long)p.a.T * p.a.H);
  const float r = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < 2 * DB; ++i)
    if (lane + 32 * i < p.a.D) {
      const long long at = ((b * p.a.T + t) * p.a.H + h) * p.a.D + lane + 32 * i;
      const __nv_bfloat16 y = __float2bfloat16(acc[i] * r);
      p.out[at] = y;
      if (p.rest != nullptr) p.rest[at] = __float2bfloat16(acc[i] * r - __bfloat162float(y));
    }
  if (p.lse != nullptr && lane == 0) {
    const int padded = (p.a.T + AT_M - 1) / AT_M * AT_M;
    float* at = p.lse + row / p.a.T * padded;
    at[t] = l != 0.f ? -m - log2f(l) : -INFINITY;
    if (t == p.a.T - 1)
      for (int i = p.a.T; i < padded; ++i) at[i] = -INFINITY;
  }
}

// Pairs where they give every SM a CTA (ALONE: where there are more tiles than SMs: 150 tiles of 640 keys 22.5 us as halves, 16.4 as
// pairs; 192 causal ones of up to 3000 keys 37 and 39); else halves, with the keys split so far that the CTAs fill the SMs once, each with two key
// tiles at least.
int fwd_splits(const AttentionShape& a, bool& pair) {
  const int sms = multiprocessors();
  const long long heads = (long long)a.B * a.H, tiles = (a.T + AT_M - 1) / AT_M;
  pair = a.D <= 64 ? heads * tiles > sms : heads * ((tiles + 1) / 2) >= sms;
  if (pair) return 1;
  const long long most = std::max(1, (a.S + AT_M - 1) / AT_M / 2);
  return (int)std::max<long long>(1, std::min({sms / (heads * tiles), most, 32ll}));
}

template <int DB, bool PAIR, bool SCALED>
void run(const FwdParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t s) {
  constexpr int QT = PAIR && !alone(DB, PAIR) ? 2 : 1, smem = (QT + 4) * DB * AT_BOX + 1024, threads = fwd_threads(DB, PAIR);
  static PerDeviceOnce once;
  auto kern = attention_fwd_kernel<DB, PAIR, SCALED>;
  if (once.first_use()) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    cudaFuncAttributes f{};
    if (cudaFuncGetAttributes(&f, kern) != cudaSuccess || f.numRegs * threads < 128 * fwd_few(DB, PAIR) + (threads - 128) * fwd_many(DB, PAIR))
      throw std::runtime_error("attention_fwd: built with too few registers for its warps' shares");
  }
  kern<<<dim3(p.a.B * p.a.H, (p.a.T + QT * AT_M - 1) / (QT * AT_M), p.splits), threads, smem, s>>>(tq, tk, tv, p);
  attention_check_launch("attention_fwd");
}

template <int DB, bool SCALED>
void run_width(const AttentionFwd& f, cudaStream_t s) {
  const AttentionShape& a = f.a;
  const CUtensorMap tq = attention_map(f.q, a.D, a.T, a.H, a.B), tk = attention_map(f.k, a.D, a.S, a.G, a.B), tv = attention_map(f.v, a.D, a.S, a.G, a.B);
  bool pair;
  FwdParams p{a, f.out, f.rest, f.lse, f.part, (const __nv_bfloat16*)f.v.p, f.v.sr, f.v.sh, f.v.sb, f.k_scales, f.v_scales, f.blocks, fwd_splits(a, pair), a.scale * LOG2E, f.status};
  if (pair) return run<DB, true, SCALED>(p, tq, tk, tv, s);
  run<DB, false, SCALED>(p, tq, tk, tv, s);
  if (p.splits > 1) {
    const long long rows = (long long)a.B * a.H * a.T;
    attention_join_kernel<DB><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(p);
    attention_check_launch("attention_join");
  }
}

}  // namespace

long long attention_fwd_scratch(const AttentionShape& a) {
  bool pair;
  const int splits = fwd_splits(a, pair);
  return splits > 1 ? (long long)splits * a.B * a.H * a.T * ((a.D <= 64 ? 64 : 128) + 2) * 4 : 0;
}

void launch_attention_fwd(const AttentionFwd& f, cudaStream_t s) {
  if (f.k_scales != nullptr) f.a.D <= 64 ? run_width<1, true>(f, s) : run_width<2, true>(f, s);
  else f.a.D <= 64 ? run_width<1, false>(f, s) : run_width<2, false>(f, s);
}

}  // namespace tb
