// Backward pass: the probabilities are computed again from the scores and the saved logarithms of their sums. With
//   P = exp(S - lse),  dP = dO V^T,  delta_i = dO_i . O_i,  dS = P (dP - delta):
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO     (dK, dV summed over the query heads of a shared head).
//
// Two kernels, each of which keeps its sums in TMEM and writes every gradient once: one per 128 queries (dQ; it also forms delta),
// one per 128 keys (dK, dV). S and dP are formed in both, so there are seven tile products instead of the five of a kernel that
// adds dQ up in global memory: no atomics, the same bits every time, no fp32 copy of dQ.
// Both: warp 0 TMA producer, warp 1 tcgen05.mma, the warps from 4 on softmax; a thread has 64 columns of one row, and keeps
// the fp32 probabilities in registers between S and dP. P and dS are rounded to bf16 for the products (2^-8 of each term at
// most, which averages out over the sums); dS is formed from the unrounded P.
// For dQ the next tile's scores are formed as soon as these are in registers, and there are two sets of columns for dP (dS over it), so that
// a tile's dP need not wait for the product with the last one's dS. For dK and dV, P lies over S, and the next scores come behind
// the product with P unless P has columns of its own (P through shared memory, to have them earlier, left no room for a third stage of
// query tiles with heads of 128: 2911 clocks a tile instead of 2500, waiting for these).
// Bound by the chain from scores to slopes and, with heads of 128, by the products (1.26 and 1.37 PFLOP/s). With a cold L2, dQ and dK, dV:
// 8192 tokens, 16 heads on 4 of 128, causal: 332 and 407 us, of which the last 50 have SMs without work (the first keys' tile of a shared
// head is seen by 256 query tiles, the mean of an SM is 225).
#include <algorithm>
#include <type_traits>

#include "attention_tiles.cuh"

namespace tb {
namespace {

// TWO: tiles have 64 rows along the axis that is walked (keys for dQ, queries for dK and dV) instead of 128, four softmax warps instead of eight,
// and two CTAs share an SM, each with half of the tensor memory: one's exponentials run under the other's products, loads and stores.
// Wider heads' tiles and sums do not fit twice.
__host__ __device__ constexpr int bwd_tile(bool two) { return two ? 64 : 128; }
__host__ __device__ constexpr int bwd_threads(bool two) { return 128 + 2 * bwd_tile(two); }
constexpr int BW_FEW = 56, BW_MANY = 200;  // registers of a thread of the first four warps and of the others, of 128 each at launch

struct BwdParams {
  AttentionShape a;
  AttentionView out, rest, dout;
  const float* lse;
  float* delta;
  __nv_bfloat16 *dq, *dk, *dv;
  float scale2;
  int* status;
};

// TMEM column of step k of a 128 x 128 (or 64) bf16 operand: halves of 64 values, each in the first 32 columns of its 64
__device__ __forceinline__ int half_column(int k) { return (k >> 2) * 64 + (k & 3) * 8; }

// ---------------------------------------------------------------------------------------------------------------- queries
template <int DB, bool TWO>
__global__ void __launch_bounds__(bwd_threads(TWO), TWO ? 2 : 1) attention_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG,
                                                                     const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                                                     const BwdParams p) {
  // K is held until the product with dS, V only until dP is there: longer and shorter rings
  constexpr int BN = bwd_tile(TWO), HALVES = BN / 64, BOX = BN * 128, TILE = DB * AT_BOX, KTILE = DB * BOX, NK = DB == 1 ? 4 : 3, NV = DB == 1 ? 3 : 2;
  constexpr uint32_t P_AT = BN, Q_AT = 3 * BN, COLUMNS = 4 * BN;  // TMEM columns: S 0 .., dP (dS over it) twice, the sums
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sG = sQ + TILE, *sK = sG + TILE, *sV = sK + NK * KTILE;  // G: dO
  __shared__ __align__(8) uint64_t bars[11 + 2 * NK + 2 * NV];
  uint64_t *q_full = bars, *s_full = bars + 1, *s_read = bars + 2, *dp_full = bars + 3, *dp_next = bars + 4, *ds_ready = bars + 5, *done = bars + 6,
           *k_clean = bars + 7, *end_full = bars + 8, *ds_next = bars + 9, *k_full = bars + 11, *k_empty = k_full + NK, *v_full = k_empty + NK, *v_empty = v_full + NV;
  __shared__ uint32_t tmem_slot;
  __shared__ float part[AT_M];
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int h = blockIdx.x % p.a.H, b = blockIdx.x / p.a.H, kvh = h / (p.a.H / p.a.G);
  const int q0 = (gridDim.y - 1 - blockIdx.y) * AT_M;
  const Visible vis(p.a, b);
  const int2 range = vis.tiles(q0, min(p.a.T, q0 + AT_M) - 1, BN);
  const int n = range.y - range.x;
  // the tile, if any, in which the sequence ends before the tile does: its other keys may hold anything and are set to zero. It is
  // the last of all and has barriers of its own, whose only phase the warps that wait for nothing else cannot miss.
  const int ragged = vis.length % BN != 0 && vis.length < p.a.S ? vis.length / BN - range.x : -1;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < NK; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(v_full + i, 1);
      mbar_init(v_empty + i, 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_read, 128 * HALVES);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 128 * HALVES);
    mbar_init(ds_next, 128 * HALVES);
    mbar_init(done, 1);
    mbar_init(k_clean, 64);
    mbar_init(end_full, 1);
    mbar_init(dp_next, 1);
    mbar_fence_init();
  }
  if (warp == 2) {
    tmem_alloc(&tmem_slot, COLUMNS);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = uniform(tmem_slot);

  if (warp < 4) {
  if (warp == 0) {
    if (lane == 0 && n > 0) {
      prefetch_tmap(&tmQ);
      prefetch_tmap(&tmG);
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
      mbar_expect_tx(q_full, 2 * TILE);
      for (int d = 0; d < DB; ++d) {
        tma_load_4d(sQ + d * AT_BOX, &tmQ, q_full, d * 64, q0, h, b);
        tma_load_4d(sG + d * AT_BOX, &tmG, q_full, d * 64, q0, h, b);
      }
      bool ok = true;
      for (int u = 0; u < n && ok; ++u) {
        const int ks = u % NK, vs = u % NV;
        uint64_t *kf = u == ragged ? end_full : k_full + ks, *vf = u == ragged ? end_full : v_full + vs;
        if (u >= NK) ok = mbar_wait(k_empty + ks, ((u / NK) & 1) ^ 1);
        if (u >= NV) ok = ok && mbar_wait(v_empty + vs, ((u / NV) & 1) ^ 1);
        if (!ok) break;
        mbar_expect_tx(kf, u == ragged ? 2 * KTILE : KTILE);
        if (u != ragged) mbar_expect_tx(vf, KTILE);
        for (int d = 0; d < DB; ++d) tma_load_4d(sK + ks * KTILE + d * BOX, &tmK, kf, d * 64, (range.x + u) * BN, kvh, b);
        for (int d = 0; d < DB; ++d) tma_load_4d(sV + vs * KTILE + d * BOX, &tmV, vf, d * 64, (range.x + u) * BN, kvh, b);
      }
      // nothing may arrive once the block is gone
      for (int u = max(0, n - NK); u < n && ok; ++u) ok = mbar_wait(k_empty + u % NK, (u / NK) & 1);
      for (int u = max(0, n - NV); u < n && ok; ++u) ok = mbar_wait(v_empty + u % NV, (u / NV) & 1);
      if (!ok && p.status) *p.status = ST_TIMEOUT_EMPTY;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (n > 0) {
      const int ks = (p.a.D + 15) / 16;
      const uint32_t q = smem_u32(sQ), g = smem_u32(sG), k = smem_u32(sK), v = smem_u32(sV);
      // scores and dP of a tile, as its keys and values arrive
      auto scores = [&](int u) {
        const int ks_at = u % NK, vs_at = u % NV;
        if (!(u == ragged ? warp_wait(end_full, 0) && warp_wait(k_clean, 0) : warp_wait(k_full + ks_at, (u / NK) & 1))) return false;
        tc_fence_after_sync();
        issue([&] {
          scores_product<DB, BN>(tmem, q, k + ks_at * KTILE, ks);
          umma_commit(s_full);
        });
        if (u != ragged && !warp_wait(v_full + vs_at, (u / NV) & 1)) return false;
        issue([&] {
          scores_product<DB, BN>(tmem + P_AT + (u & 1) * BN, g, v + vs_at * KTILE, ks);
          umma_commit(u & 1 ? dp_next : dp_full);  // one for each set of columns
          umma_commit(v_empty + vs_at);
        });
        return true;
      };
      bool ok = warp_wait(q_full, 0) && scores(0);
      if (ok) {
        for (int u = 0; u < n && ok; ++u) {
          if (u + 1 < n) ok = warp_wait(s_read, u & 1) && scores(u + 1);  // the other dP columns were read by the product before
          ok = ok && warp_wait(u & 1 ? ds_next : ds_ready, (u >> 1) & 1);
          if (!ok) break;
          tc_fence_after_sync();
          issue([&] {
            rows_product<DB, 0, BN / 16>(tmem + Q_AT, tmem + P_AT + (u & 1) * BN, k + u % NK * KTILE, u > 0, half_column);
            umma_commit(k_empty + u % NK);
          });
        }
        if (ok) issue([&] { umma_commit(done); });
      }
      if (!ok && p.status) *p.status = ST_TIMEOUT_FULL;
    }
  } else {
    if (ragged >= 0 && ragged < n) {
      const int s = ragged % NK, keep = vis.length % BN;
      const bool ok = mbar_wait(end_full, 0);
      if (ok)
        for (int i = threadIdx.x - 64; i < KTILE / 16; i += 64)
          if (((i >> 3) & (BN - 1)) >= keep) reinterpret_cast<uint4*>(sK + s * KTILE)[i] = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      mbar_arrive(k_clean);
      if (!ok && p.status) *p.status = ST_TIMEOUT_FULL;
    }
  }
  } else {
    const int half = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane, t = q0 + row;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_base + half * 64;
    const int padded = (p.a.T + AT_M - 1) / AT_M * AT_M;
    const long long at = ((long long)b * p.a.H + h) * padded + t;
    const float lse = p.lse[at];
    // delta: its share of the row's columns by each of the row's threads
    float dot = 0.f;
    if (t < p.a.T) {
      const uint4* o = reinterpret_cast<const uint4*>((const __nv_bfloat16*)p.out.p + b * p.out.sb + t * p.out.sr + h * p.out.sh);
      const uint4* l = reinterpret_cast<const uint4*>((const __nv_bfloat16*)p.rest.p + b * p.rest.sb + t * p.rest.sr + h * p.rest.sh);
      const uint4* g = reinterpret_cast<const uint4*>((const __nv_bfloat16*)p.dout.p + b * p.dout.sb + t * p.dout.sr + h * p.dout.sh);
      const int pieces = p.a.D / 8, mid = (pieces + HALVES - 1) / HALVES;
      for (int i = half * mid; i < (half == 0 ? mid : pieces); ++i) {
        const uint4 x = o[i], y = g[i], z = l[i];
        const uint32_t *xp = &x.x, *yp = &y.x, *zp = &z.x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dot = fmaf(__uint_as_float(xp[e] << 16) + __uint_as_float(zp[e] << 16), __uint_as_float(yp[e] << 16), dot);
          dot = fmaf(__uint_as_float(xp[e] & 0xffff0000u) + __uint_as_float(zp[e] & 0xffff0000u), __uint_as_float(yp[e] & 0xffff0000u), dot);
        }
      }
    }
    if constexpr (HALVES == 2) {
      if (half == 1) part[row] = dot;
      named_barrier<256>(1);
      if (half == 0) part[row] += dot;
      named_barrier<256>(1);
      dot = part[row];
    }
    const float delta = -dot;
    if (half == 0) p.delta[at] = delta;
    const int lo = vis.low(t), hi = vis.high(t);
    bool ok = true;
    const uint64_t cc = pack_f2(p.scale2, p.scale2), mm = pack_f2(lse, lse), dd = pack_f2(delta, delta);
    // MASKED: not all keys of the tile are visible to all queries. Invisible ones have weight and slope zero, whatever they hold.
    auto tile = [&](auto some, int u, int c_lo, int c_hi) {
      constexpr bool MASKED = decltype(some)::value;
      const uint32_t tP = tS + P_AT + (u & 1) * BN;
      uint32_t x[32], y[32];
      tmem_load(tS, x, y);
      tc_fence_before_sync();
      mbar_arrive(s_read);
      auto weights = [&](uint32_t (&r)[32], int c0) {
        const uint32_t see = MASKED ? visible_bits(c_lo - c0, c_hi - c0) : 0u;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const uint64_t z = fma2(pack_f2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), cc, mm);
          float a, e;
          unpack_f2(z, a, e);
          a = ex2(a);
          e = ex2(e);
          if constexpr (MASKED) {
            a = see >> i & 1 ? a : 0.f;
            e = see >> (i + 1) & 1 ? e : 0.f;
          }
          r[i] = __float_as_uint(a);
          r[i + 1] = __float_as_uint(e);
        }
      };
      auto slopes = [&](uint32_t (&r)[32], int c0) {
        const uint32_t see = MASKED ? visible_bits(c_lo - c0, c_hi - c0) : 0u;
        uint32_t d[32], o[16];
        tmem_load(tP + c0, d);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const uint64_t z = mul2(add2(pack_f2(__uint_as_float(d[i]), __uint_as_float(d[i + 1])), dd), pack_f2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])));
          if constexpr (MASKED) {
            float a, e;
            unpack_f2(z, a, e);
            o[i / 2] = pack_bf16x2(see >> i & 1 ? a : 0.f, see >> (i + 1) & 1 ? e : 0.f);
          } else {
            o[i / 2] = f2_to_bf16x2(z);
          }
        }
        tmem_st_32x32b_x16(tP + c0 / 2, o);  // over columns that this thread has read
      };
      weights(x, 0);
      if (!warp_wait(u & 1 ? dp_next : dp_full, (u >> 1) & 1)) return false;
      tc_fence_after_sync();
      slopes(x, 0);
      weights(y, 32);
      slopes(y, 32);
      tmem_st_wait();
      tc_fence_before_sync();
      // a warp may be done with the next tile before another is with this one: each of the two sets has its barrier
      mbar_arrive(u & 1 ? ds_next : ds_ready);
      return true;
    };
    for (int u = 0; u < n; ++u) {
      const int key = (range.x + u) * BN;
      ok = warp_wait(s_full, u & 1);
      if (!ok) break;
      tc_fence_after_sync();
      if (vis.whole(q0, q0 + AT_M - 1, key, BN)) ok = tile(std::false_type{}, u, 0, 0);
      else ok = tile(std::true_type{}, u, lo - key - half * 64, hi - key - half * 64);
      if (!ok) break;
    }
    if (ok && n > 0) ok = warp_wait(done, 0);
    tc_fence_after_sync();
    __nv_bfloat16* o = p.dq + (((long long)b * p.a.T + t) * p.a.H + h) * p.a.D;
    for (int c = half * 32 * DB; c < (half + 1) * (64 / HALVES) * DB; c += 16) {
      uint32_t v[16] = {};
      if (n > 0) {
        __syncwarp();
        tmem_load(tmem + lane_base + Q_AT + c, v);
      }
      if (t < p.a.T) store_row16(o, c, p.a.D, v, !ok ? __int_as_float(0x7fc00000) : n > 0 ? p.a.scale : 0.f);  // no numbers where a wait expired
    }
    if (!ok && p.status) *p.status = ST_TIMEOUT_TMEM;
  }
  __syncwarp();  // the block's barrier counts warps, not threads
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 2) tmem_dealloc(tmem, COLUMNS);
}

// ---------------------------------------------------------------------------------------------------------------- keys, values
// Stages of query tiles: what shared memory holds
__host__ __device__ constexpr int key_stages(int db, bool two) { return two ? 4 : db == 1 ? 3 : 2; }

// SHARE: two neighbouring CTAs (a cluster) have the same keys and one half of their queries each; the second hands its sums to the first.
template <int DB, bool TWO, bool SHARE>
__global__ void __launch_bounds__(bwd_threads(TWO), TWO ? 2 : 1) attention_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG,
                                                                      const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                                                                      const BwdParams p) {
  constexpr int BN = bwd_tile(TWO), HALVES = BN / 64, BOX = BN * 128, TILE = DB * AT_BOX, QTILE = DB * BOX, NQ = key_stages(DB, TWO);
  constexpr int STATS = 2 * BN * 4;  // lse and delta of a query tile
  // TMEM columns: S 0 .., dP (dS over it), weights where they fit (APART, else over S), and the sums
  constexpr bool APART = DB == 1 && !TWO;
  constexpr uint32_t D_AT = BN, W_AT = APART ? 2 * BN : 0, V_AT = APART ? 3 * BN : 2 * BN, K_AT = V_AT + 64 * DB, COLUMNS = 4 * BN;
  extern __shared__ __align__(1024) uint8_t smem[];  // no other shared memory: it starts on a tile's boundary, which is looked at below
  uint8_t *sK = smem, *sV = sK + TILE, *sQ = sV + TILE, *sG = sQ + NQ * QTILE;
  float* sStat = reinterpret_cast<float*>(sG + NQ * QTILE);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sStat + NQ * 2 * BN);
  uint64_t *kv_full = bars, *s_full = bars + 1, *p_ready = bars + 2, *dp_full = bars + 3, *ds_ready = bars + 4, *done = bars + 5, *s_read = bars + 6,
           *p_free = bars + 7, *q_full = bars + 8, *q_empty = q_full + NQ;
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(q_empty + NQ);
  if ((smem_u32(smem) & 1023) != 0) {
    if (threadIdx.x == 0 && p.status) *p.status = ST_BAD_ARGUMENT;
    return;
  }
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int member = SHARE ? blockIdx.x & 1 : 0, head_at = SHARE ? blockIdx.x >> 1 : blockIdx.x;
  const int kvh = head_at % p.a.G, b = head_at / p.a.G, rep = p.a.H / p.a.G;
  const int k0 = blockIdx.y * AT_M;  // with a causal mask the first keys are seen by the most queries
  const Visible vis(p.a, b);
  const int first = vis.first(k0), last = vis.last(min(p.a.S, k0 + AT_M) - 1, p.a.T);
  const int i0 = first / BN, per = k0 < vis.length && last >= first ? last / BN + 1 - i0 : 0, all = per * rep;
  const int half_of_all = SHARE ? (all + 1) / 2 : all, n = member == 0 ? half_of_all : all - half_of_all;  // query tiles of all heads, head by head
  const int skip = member == 0 || n == 0 ? 0 : half_of_all;
  const int padded = (p.a.T + AT_M - 1) / AT_M * AT_M;
  bool finished = true;  // of the softmax warps: no wait expired

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < NQ; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
    }
    mbar_init(s_full, 1);
    mbar_init(p_ready, 128 * HALVES);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 128 * HALVES);
    mbar_init(done, 1);
    mbar_init(s_read, 128 * HALVES);
    mbar_init(p_free, 1);
    mbar_fence_init();
  }
  if (warp == 2) {
    tmem_alloc(&tmem_slot, COLUMNS);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = uniform(tmem_slot);

  if (warp < 4) {
  if constexpr (TWO) registers_down<BW_FEW>();
  if (warp == 0) {
    if (lane == 0 && n > 0) {
      prefetch_tmap(&tmQ);
      prefetch_tmap(&tmG);
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
      mbar_expect_tx(kv_full, 2 * TILE);
      for (int d = 0; d < DB; ++d) {
        tma_load_4d(sK + d * AT_BOX, &tmK, kv_full, d * 64, k0, kvh, b);
        tma_load_4d(sV + d * AT_BOX, &tmV, kv_full, d * 64, k0, kvh, b);
      }
      bool ok = true;
      int i = skip > 0 ? skip % per : 0, head = skip > 0 ? skip / per : 0;
      for (int u = 0; u < n && ok; ++u) {
        const int s = u % NQ, h = kvh * rep + head, t0 = (i0 + i) * BN;
        if (++i == per) i = 0, ++head;
        if (u >= NQ) ok = mbar_wait(q_empty + s, ((u / NQ) & 1) ^ 1);
        if (!ok) break;
        mbar_expect_tx(q_full + s, 2 * QTILE + STATS);
        for (int d = 0; d < DB; ++d) {
          tma_load_4d(sQ + s * QTILE + d * BOX, &tmQ, q_full + s, d * 64, t0, h, b);
          tma_load_4d(sG + s * QTILE + d * BOX, &tmG, q_full + s, d * 64, t0, h, b);
        }
        const long long at = ((long long)b * p.a.H + h) * padded + t0;
        bulk_load(sStat + s * 2 * BN, p.lse + at, BN * 4, q_full + s);
        bulk_load(sStat + s * 2 * BN + BN, p.delta + at, BN * 4, q_full + s);
      }
      for (int u = max(0, n - NQ); u < n && ok; ++u) ok = mbar_wait(q_empty + u % NQ, (u / NQ) & 1);
      if (!ok && p.status) *p.status = ST_TIMEOUT_EMPTY;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (n > 0) {
      const int ks = (p.a.D + 15) / 16;
      const uint32_t k = smem_u32(sK), v = smem_u32(sV), q = smem_u32(sQ), g = smem_u32(sG);
      auto arrived = [&](int u) { return warp_wait(q_full + u % NQ, (u / NQ) & 1); };
      bool ok = warp_wait(kv_full, 0) && arrived(0);
      if (ok) {
        tc_fence_after_sync();
        auto scores = [&](int u) {
          issue([&] {
            scores_product<DB, BN>(tmem, k, q + u % NQ * QTILE, ks);
            umma_commit(s_full);
          });
        };
        auto slopes = [&](int u) {
          issue([&] {
            scores_product<DB, BN>(tmem + D_AT, v, g + u % NQ * QTILE, ks);
            umma_commit(dp_full);
          });
        };
        scores(0);
        slopes(0);
        for (int u = 0; u < n && ok; ++u) {
          const int s = u % NQ;
          const bool next = u + 1 < n;
          if (APART && next) {  // the softmax warps have the scores in registers
            ok = warp_wait(s_read, u & 1) && arrived(u + 1);
            if (!ok) break;
            tc_fence_after_sync();
            scores(u + 1);
          }
          ok = warp_wait(p_ready, u & 1);
          if (!ok) break;
          tc_fence_after_sync();
          issue([&] {
            if constexpr (APART) rows_product<DB, 0, BN / 16>(tmem + V_AT, tmem + W_AT, g + s * QTILE, u > 0, [](int k) { return k * 8; });
            else rows_product<DB, 0, BN / 16>(tmem + V_AT, tmem, g + s * QTILE, u > 0, half_column);
            if (APART) umma_commit(p_free);
          });
          if (!APART && next) {  // behind the product that reads P from the same columns
            ok = arrived(u + 1);
            if (!ok) break;
            scores(u + 1);
          }
          ok = warp_wait(ds_ready, u & 1);
          if (!ok) break;
          tc_fence_after_sync();
          issue([&] {
            rows_product<DB, 0, BN / 16>(tmem + K_AT, tmem + D_AT, q + s * QTILE, u > 0, half_column);
            umma_commit(q_empty + s);
          });
          if (next) slopes(u + 1);  // behind the product that reads dS from the same columns
        }
        if (ok) issue([&] { umma_commit(done); });
      }
      if (!ok && p.status) *p.status = ST_TIMEOUT_FULL;
    }
  }
  } else {
    if constexpr (TWO) registers_up<BW_MANY>();
    const int half = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane, key = k0 + row;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_base + half * 64, tP = tS + D_AT;
    const bool inside = key < vis.length;
    const int lo = inside ? vis.first(key) : p.a.T, hi = inside ? vis.last(key, p.a.T) : -1;  // queries that see this key
    bool ok = true;
    const uint64_t cc = pack_f2(p.scale2, p.scale2);
    auto tile = [&](auto some, int u, int c_lo, int c_hi) {  // as for the queries
      constexpr bool MASKED = decltype(some)::value;
      const float4 *lse = reinterpret_cast<const float4*>(sStat + u % NQ * 2 * BN + half * 64), *delta = lse + BN / 4;
      uint32_t x[32], y[32];
      tmem_load(tS, x, y);
      tc_fence_before_sync();
      if (APART) mbar_arrive(s_read);
      if (APART && u > 0) {  // the product that read the last weights is done
        if (!warp_wait(p_free, (u - 1) & 1)) return false;
        tc_fence_after_sync();
      }
      auto weights = [&](uint32_t (&r)[32], int c0) {
        const uint32_t see = MASKED ? visible_bits(c_lo - c0, c_hi - c0) : 0u;
        uint32_t o[16];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 z = lse[(c0 + i) / 4];
          float a[4];
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            unpack_f2(fma2(pack_f2(__uint_as_float(r[i + k]), __uint_as_float(r[i + k + 1])), cc, k == 0 ? pack_f2(z.x, z.y) : pack_f2(z.z, z.w)), a[k], a[k + 1]);
            a[k] = ex2(a[k]);
            a[k + 1] = ex2(a[k + 1]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (MASKED) a[k] = see >> (i + k) & 1 ? a[k] : 0.f;
            r[i + k] = __float_as_uint(a[k]);
          }
          o[i / 2] = pack_bf16x2(a[0], a[1]);
          o[i / 2 + 1] = pack_bf16x2(a[2], a[3]);
        }
        tmem_st_32x32b_x16((APART ? tmem + lane_base + W_AT + half * 32 : tS) + c0 / 2, o);
      };
      weights(x, 0);
      weights(y, 32);
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(p_ready);
      if (!warp_wait(dp_full, u & 1)) return false;
      tc_fence_after_sync();
      auto slopes = [&](uint32_t (&r)[32], int c0) {
        const uint32_t see = MASKED ? visible_bits(c_lo - c0, c_hi - c0) : 0u;
        uint32_t d[32], o[16];
        tmem_load(tP + c0, d);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 z = delta[(c0 + i) / 4];
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            const uint64_t w = mul2(add2(pack_f2(__uint_as_float(d[i + k]), __uint_as_float(d[i + k + 1])), k == 0 ? pack_f2(z.x, z.y) : pack_f2(z.z, z.w)),
                                    pack_f2(__uint_as_float(r[i + k]), __uint_as_float(r[i + k + 1])));
            if constexpr (MASKED) {
              float a, e;
              unpack_f2(w, a, e);
              o[(i + k) / 2] = pack_bf16x2(see >> (i + k) & 1 ? a : 0.f, see >> (i + k + 1) & 1 ? e : 0.f);
            } else {
              o[(i + k) / 2] = f2_to_bf16x2(w);
            }
          }
        }
        tmem_st_32x32b_x16(tP + c0 / 2, o);
      };
      slopes(x, 0);
      slopes(y, 32);
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(ds_ready);
      return true;
    };
    for (int u = 0, i = skip > 0 ? skip % per : 0; u < n; ++u) {
      const int t0 = (i0 + i) * BN;
      if (++i == per) i = 0;
      ok = warp_wait(q_full + u % NQ, (u / NQ) & 1) && warp_wait(s_full, u & 1);
      if (!ok) break;
      tc_fence_after_sync();
      if (vis.whole(t0, t0 + BN - 1, k0)) ok = tile(std::false_type{}, u, 0, 0);
      else ok = tile(std::true_type{}, u, lo - t0 - half * 64, hi - t0 - half * 64);
      if (!ok) break;
    }
    if (ok && n > 0) ok = warp_wait(done, 0);
    tc_fence_after_sync();
    if (!ok && p.status) *p.status = ST_TIMEOUT_TMEM;
    finished = ok;
  }
  const int half = (warp - 4) >> 2, row = (warp & 3) * 32 + lane, key = k0 + row;
  const uint32_t sums = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  float* other = reinterpret_cast<float*>(smem);  // [2][64 DB][128]
  if constexpr (SHARE) {
    __syncwarp();
    cluster_sync_all();  // nothing reads or writes the tiles any more
    if (member == 1 && warp >= 4 && n > 0) {
      for (int which = half; which < 2; which += HALVES)
        for (int c = 0; c < 64 * DB; c += 16) {
          uint32_t v[16];
          __syncwarp();
          tmem_load(sums + (which == 0 ? V_AT : K_AT) + c, v);
          const uint32_t to = mapa_shared(smem_u32(other + (which * 64 * DB + c) * AT_M + row), 0);
#pragma unroll
          for (int i = 0; i < 16; ++i) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + i * AT_M * 4), "r"(finished ? v[i] : 0x7fc00000u) : "memory");
        }
    }
    __syncwarp();
    cluster_sync_all();
  }
  if (warp >= 4 && member == 0) {
    const bool inside = key < vis.length;
    // the first half of the warps writes dV, the second dK
    for (int which = half; which < 2; which += HALVES) {
      __nv_bfloat16* o = (which == 0 ? p.dv : p.dk) + (((long long)b * p.a.S + key) * p.a.G + kvh) * p.a.D;
      const float f = !finished ? __int_as_float(0x7fc00000) : n == 0 ? 0.f : which == 0 ? 1.f : p.a.scale;
      for (int c = 0; c < 64 * DB; c += 16) {
        uint32_t v[16] = {};
        if (n > 0) {
          __syncwarp();
          tmem_load(sums + (which == 0 ? V_AT : K_AT) + c, v);
        }
        if (SHARE && all > n) {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + other[(which * 64 * DB + c + i) * AT_M + row]);
        }
        if (!inside) {  // what keys past the length hold does not count
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = 0;
        }
        if (key < p.a.S) store_row16(o, c, p.a.D, v, f);
      }
    }
  }
  __syncwarp();  // the block's barrier counts warps, not threads
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 2) tmem_dealloc(tmem, COLUMNS);
}

template <int DB, bool TWO>
void run_queries(const AttentionBwd& f, const BwdParams& p, unsigned tiles, cudaStream_t s) {
  constexpr int BN = bwd_tile(TWO), NK = DB == 1 ? 4 : 3, NV = DB == 1 ? 3 : 2, smem = 2 * DB * AT_BOX + (NK + NV) * DB * BN * 128 + 1024;
  static_assert(smem + 1280 <= 227 * 1024 / (TWO ? 2 : 1), "shared memory of a block");
  const AttentionShape& a = f.a;
  static PerDeviceOnce once;
  if (once.first_use()) cudaFuncSetAttribute(attention_dq_kernel<DB, TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  attention_dq_kernel<DB, TWO><<<dim3(a.B * a.H, tiles), bwd_threads(TWO), smem, s>>>(
      attention_map(f.q, a.D, a.T, a.H, a.B), attention_map(f.dout, a.D, a.T, a.H, a.B), attention_map(f.k, a.D, a.S, a.G, a.B, BN),
      attention_map(f.v, a.D, a.S, a.G, a.B, BN), p);
  attention_check_launch("attention_dq");
}
template <int DB, bool TWO, bool SHARE>
void run_keys(const AttentionBwd& f, const BwdParams& p, unsigned tiles, cudaStream_t s) {
  constexpr int BN = bwd_tile(TWO), NQ = key_stages(DB, TWO), smem = 2 * DB * AT_BOX + NQ * (2 * DB * BN * 128 + 2 * BN * 4) + (9 + 2 * NQ) * 8;
  static_assert(smem + 1024 <= 227 * 1024 / (TWO ? 2 : 1), "shared memory of a block");
  const AttentionShape& a = f.a;
  static PerDeviceOnce once;
  if (once.first_use()) {
    cudaFuncSetAttribute(attention_dkv_kernel<DB, TWO, SHARE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    cudaFuncAttributes x{};
    if (TWO && (cudaFuncGetAttributes(&x, attention_dkv_kernel<DB, TWO, SHARE>) != cudaSuccess ||
                x.numRegs * bwd_threads(TWO) < 128 * BW_FEW + (bwd_threads(TWO) - 128) * BW_MANY))
      throw std::runtime_error("attention_dkv: built with too few registers for its warps' shares");
  }
  static_assert(!SHARE || 2 * 64 * DB * AT_M * 4 <= 2 * DB * AT_BOX + NQ * 2 * DB * BN * 128, "the sums take the tiles' place");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.B * a.G * (SHARE ? 2 : 1), tiles);
  cfg.blockDim = dim3(bwd_threads(TWO));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = SHARE ? 1 : 0;
  cudaLaunchKernelEx(&cfg, attention_dkv_kernel<DB, TWO, SHARE>, attention_map(f.q, a.D, a.T, a.H, a.B, BN), attention_map(f.dout, a.D, a.T, a.H, a.B, BN),
                     attention_map(f.k, a.D, a.S, a.G, a.B), attention_map(f.v, a.D, a.S, a.G, a.B), p);
  attention_check_launch("attention_dkv");
}

}  // namespace

// Heads of up to 64 with two CTAs per SM where all SMs get two: a CTA that is left by itself on an SM takes longer than one with tiles of
// 128. Both kernels, two per SM against one: 16 x 2048 tokens, 6 heads (1536 CTAs) 265 and 314 us, 8 x 1024 (384) 64 and 71; 3000 tokens,
// 8 heads (192) 93 and 68; 8192 tokens, 8 heads on 2 (512 and 128) 583 and 398.
// Keys shared by two CTAs where there are fewer of them than SMs and their walks over the queries of all heads are long. Both kernels, in tiles
// of 128 without and with it: 8192 tokens, 8 heads on 2 of 64 (128 CTAs, 256 tiles) 411 and 282 us; 4096, 12 on 4 of 128 (128, 96) 251 and 195; 600
// twice, 8 on 2 of 64 (20, 20) 46 and 38; 1024, 8 of 128 (64, 8) 48 and 46; but 2048, 8 of 128 (128, 16) 69 and 73; 1001, 12 of 80 (96, 8) 44 and
// 52; 4096, 4 of 128 with a window of 600 (128, 6) 46 and 62; 8192, 16 on 4 of 128 (256, 256) 759 and 753; 4 x 2048, 16 on 4 (256, 64) 286 and 310.
void launch_attention_bwd(const AttentionBwd& f, cudaStream_t s) {
  const AttentionShape& a = f.a;
  const BwdParams p{a, f.out, f.rest, f.dout, f.lse, f.delta, f.dq, f.dk, f.dv, a.scale * LOG2E, f.status};
  const unsigned tq = (a.T + AT_M - 1) / AT_M, tk = (a.S + AT_M - 1) / AT_M;
  const long long many = 2ll * multiprocessors();
  if (a.D > 64) run_queries<2, false>(f, p, tq, s);
  else if ((long long)a.B * a.H * tq >= many) run_queries<1, true>(f, p, tq, s);
  else run_queries<1, false>(f, p, tq, s);
  const long long ctas = (long long)a.B * a.G * tk, walk = (a.window > 0 ? std::min<long long>(tq, a.window / AT_M + 2) : tq) * (a.H / a.G);
  const bool few = ctas < multiprocessors() && walk >= (2 * ctas <= multiprocessors() ? 8 : 32);
  if (a.D > 64) few ? run_keys<2, false, true>(f, p, tk, s) : run_keys<2, false, false>(f, p, tk, s);
  else if ((long long)a.B * a.G * tk >= many) run_keys<1, true, false>(f, p, tk, s);
  else few ? run_keys<1, false, true>(f, p, tk, s) : run_keys<1, false, false>(f, p, tk, s);
}

}  // namespace tb
