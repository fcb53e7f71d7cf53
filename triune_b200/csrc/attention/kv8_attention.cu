// Attention of a few queries over the 8-bit cache (decoding steps, drafted tokens).
//
// Bound by the bytes of the cache, so codes go from memory straight into registers, 16 bytes a thread and load, and from there, as
// fp16 numbers (int8 and e4m3 codes are fp16 numbers exactly), into mma.sync.m16n8k16 with the queries as the eight columns: a tile
// of 16 keys times 8 queries takes D / 16 products for the scores and as many for the values. The tcgen05 unit has nothing to gain
// here: its smallest tile has 64 rows of queries where a step has H / G, and it reads codes from shared memory as they are.
//   scores^T = K Q^T: A = 16 keys. The head dimension is put in such an order that a thread's fragments are 16 consecutive bytes.
//   out^T = V^T P^T: A = 16 columns of V by 16 keys; columns are put in such an order that a thread's are 16 consecutive bytes;
//   neighbouring keys are paired by byte permutes, P^T comes from the scores by an 8x8 transpose (movmatrix).
// Scales: a block's key scale multiplies its scores; its value scale the weights, in units of a power of two of each query's own that is no
// less than its largest weight times value scale (but for the scale's fraction) so far. So it is by what they contribute that blocks are measured: a block of large values that
// a query hardly looks at takes no digits from the others. Queries are scaled by powers of two to fit fp16 (exact but for parts below 2^-24
// of a row's largest). Weights times scales lose 2^-11 of themselves to fp16 at most (2^-24 of the largest of them, where they are small); scores,
// statistics and sums are fp32.
// The open block is read from the ring in bf16, weights in two bf16 parts (2^-16).
//
// A CTA is one warp-group of four warps that take units of 32 keys in turn, each with statistics and sums of its own, joined at the
// end through shared memory. Keys of a head are split over `splits` CTAs; a second kernel joins their parts.
// Measured with a cold L2, with the append and the join: 32 sequences of 8191 tokens, 16 heads on 8 of 128 in int8 (537 MB of codes) 122 us, this
// kernel 100 to 105 (0.8 of a copy's rate, issue slots 49 % busy); one of 131000 tokens, 16 heads on 4 of 128 in e4m3 48 us. Fetching
// the next units into L2 ahead of their loads gains 2 to 4 % there and loses 2 % where L2 holds part of the cache; four CTAs per SM, at
// 128 registers a thread, take 135 us instead of 122.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "../common/dependent_launch.cuh"
#include "../common/per_device.h"
#include "../common/ptx.cuh"
#include "kv8.cuh"

namespace tb {
namespace {

constexpr int DW = 4, UNIT = 32;  // warps of a CTA, keys of a unit
constexpr int MOST_SPLITS = 512;
// CTAs of an SM, which registers are kept to. Columns of 64, up to 8 queries: with four CTAs (115 registers) instead of five, four drafted tokens on
// 8 x 2047, 30 heads take 24.6 us instead of 22.5, a step on 32 x 8191, 6 heads 58 (int8) and 61 (e4m3) instead of 62 and 69.
constexpr int resident(int P, int NT) { return P == 64 ? (NT == 1 ? 5 : 3) : (NT == 1 ? 3 : 2); }
constexpr int step_smem(int P, int NT) { return DW * NT * 8 * (P + 4) * 4; }

struct StepParams {
  Kv8Attention a;
  int rep, rows, tiles, splits;  // queries of a key/value head: rows = T * rep, in tiles of 8 * NT
  float scale2;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// four codes (bytes 0, 1 and 2, 3) as two pairs of fp16 numbers
template <bool E4M3>
__device__ __forceinline__ void numbers(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    lo = (uint32_t)a.x | (uint32_t)a.y << 16;
    hi = (uint32_t)b.x | (uint32_t)b.y << 16;
  } else {
    const uint32_t u = w ^ 0x80808080u;  // code + 128 in the last bits of 1024 + ..
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));  // 1152
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}
// A scale (>= 0, or NaN) as a fraction from 1 to 2 (0 and NaN: themselves) times a power of two, whose exponent is returned
__device__ __forceinline__ float exponent_of(float s, float& fraction) {
  const bool small = s < 0x1p-100f;  // subnormal numbers among them
  const uint32_t bits = __float_as_uint(small ? s * 0x1p64f : s);
  fraction = s > 0.f ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u) : s;
  return (float)((int)(bits >> 23) - (small ? 191 : 127));
}
template <int BYTES>
__device__ __forceinline__ void load_codes(const uint8_t* at, uint32_t* w) {
  if constexpr (BYTES == 16) {
    const uint4 x = *reinterpret_cast<const uint4*>(at);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(at);
    w[0] = x.x, w[1] = x.y;
  }
}

template <int P, bool E4M3, int NT>
__global__ void __launch_bounds__(DW * 32, resident(P, NT)) kv8_attention_kernel(const StepParams p) {
  constexpr int KS = P / 16, VW = P / 32;  // products of a tile; words of a thread's part of a value row
  __shared__ float2 stat[DW][NT * 8];
  extern __shared__ float sums[];  // [DW][NT * 8][P + 4]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const Kv8Cache& c = p.a.c;
  long long at = blockIdx.x;
  const int split = at % p.splits;
  at /= p.splits;
  const int tile = at % p.tiles;
  at /= p.tiles;
  const int kvh = at % c.G, b = at / c.G;
  const long long start = p.a.pos.at(b);
  const int row0 = tile * NT * 8, D = p.a.D;
  const bool idle = start < 0, outside = start >= c.C;
  const int pos = idle || outside ? 0 : (int)start, total = idle || outside ? 0 : (int)min((long long)c.C, start + p.a.T);
  const int full = total / KV8_BLOCK * KV8_BLOCK;
  const long long head = (long long)b * c.G + kvh;

  // queries as columns: scaled fp16 pairs of the dimensions 16 t + 4 w + {0, 1}, {2, 3} (and 64 more from w = 4 on)
  uint32_t qf[NT][KS][2];
  float back[NT][2];  // of the columns 2 t and 2 t + 1 of each tile: what undoes the scaling, times the softmax's scale
  auto query = [&](int n) {
    const int r = row0 + n * 8 + g;
    return (const __nv_bfloat16*)p.a.q.p + b * p.a.q.sb + (r / p.rep) * p.a.q.sr + (kvh * p.rep + r % p.rep) * p.a.q.sh;
  };
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    uint32_t x[P / 8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < P / 32; ++i) {
      const int d = (i >> 1) * 64 + 16 * t + 8 * (i & 1);
      const uint4 z = row0 + n * 8 + g < p.rows && d < D ? *reinterpret_cast<const uint4*>(query(n) + d) : make_uint4(0, 0, 0, 0);
      x[4 * i] = z.x, x[4 * i + 1] = z.y, x[4 * i + 2] = z.z, x[4 * i + 3] = z.w;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = max(top, max(x[4 * i + k] & 0x7fffu, (x[4 * i + k] >> 16) & 0x7fffu));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // exponent of the largest; rows of zeros, subnormal numbers or none stay as they are
    int e = (int)(top >> 7) - 127;
    if (e == -127 || e == 128) e = 0;
    const float down = __int_as_float((127 - max(-126, min(e, 126))) << 23), up = __int_as_float((127 + max(-126, min(e, 126))) << 23);
#pragma unroll
    for (int w = 0; w < KS; ++w)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        qf[n][w][k] = half2_bits(__uint_as_float(x[2 * w + k] << 16) * down, __uint_as_float(x[2 * w + k] & 0xffff0000u) * down);
    back[n][0] = __shfl_sync(0xffffffffu, up, 8 * t) * p.scale2;
    back[n][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4) * p.scale2;
  }
  int seen[NT][2];  // last visible position of the columns
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) seen[n][k] = pos + (row0 + n * 8 + 2 * t + k) / p.rep;

  float m[NT][2], l[NT][2], o[NT][KS][4];
  float unit[NT][2];  // the sums are in units of two to this power (of weights as they are now)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = unit[n][0] = unit[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }
  // statistics of so many tiles of 16 keys whose scores (base 2) are in s; s becomes the weights. -> the logarithms of the tiles' largest
  // weights, and of what weights so far have shrunk to
  auto softmax = [&](auto& s, int tiles, float (&top)[NT][2], float (&less)[NT][2]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (i < tiles) mx = fmaxf(mx, fmaxf(s[i][n][k], s[i][n][k + 2]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float here = mx;
        mx = fmaxf(mx, m[n][k]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        top[n][k] = here - ref;
        less[n][k] = m[n][k] == mx ? 0.f : m[n][k] - ref;
        m[n][k] = mx;
        l[n][k] *= ex2(less[n][k]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (i < tiles) {
            s[i][n][k] = ex2(s[i][n][k] - ref);
            s[i][n][k + 2] = ex2(s[i][n][k + 2] - ref);
            l[n][k] += s[i][n][k] + s[i][n][k + 2];
          }
      }
  };

  // ---- blocks of codes
  const int units = full / UNIT, per = (units + p.splits - 1) / p.splits, u1 = min(units, (split + 1) * per);
  int u = split * per + warp;
  uint32_t kw[2][2][P / 16], vw[2][4][VW];  // [tile][row g or g + 8], [tile][key 2 t, 2 t + 1, 2 t + 8, 2 t + 9]
  float ks = 0.f, vs = 0.f;
  const uint8_t *kbase = c.k8 + head * c.C * P, *vbase = c.v8 + head * c.C * P;
  const float *kscale = c.ks + head * (c.C / KV8_BLOCK), *vscale = c.vs + head * (c.C / KV8_BLOCK);
  auto load_keys = [&](int u) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint8_t* row = kbase + ((long long)u * UNIT + 16 * i + 8 * r + g) * P + 16 * t;
        load_codes<16>(row, kw[i][r]);
        if constexpr (P == 128) load_codes<16>(row + 64, kw[i][r] + 4);
      }
    ks = kscale[u * UNIT / KV8_BLOCK];
  };
  // Blocks that were full before this call's tokens came may be read while these are still being appended; the ring, and the block
  // that they fill, only after. What comes behind (the join) may take its place as soon as blocks leave.
  allow_dependents();
  const int settled = p.a.appended ? pos / KV8_BLOCK * (KV8_BLOCK / UNIT) : units;
  bool waited = !p.a.appended;
  auto wait_for = [&](int u) {
    if (!waited && u >= settled) {
      wait_predecessors();
      waited = true;
    }
  };
  if (u < u1) {
    wait_for(u);
    load_keys(u);
  }
  for (; u < u1; u += DW) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        load_codes<P / 8>(vbase + ((long long)u * UNIT + 16 * i + 2 * t + (r & 1) + 8 * (r >> 1)) * P + (P / 8) * g, vw[i][r]);
    vs = vscale[u * UNIT / KV8_BLOCK];
    float s[2][NT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        uint32_t a[4];
        numbers<E4M3>(kw[i][0][w], a[0], a[2]);
        numbers<E4M3>(kw[i][1][w], a[1], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(s[i][n], a, qf[n][w][0], qf[n][w][1]);
      }
    }
    const float here = ks;
    if (u + DW < u1) {
      wait_for(u + DW);
      load_keys(u + DW);
    }
    const int key = u * UNIT + g;
    const bool masked = u * UNIT + UNIT - 1 > pos;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          s[i][n][k] *= back[n][k & 1] * here;
          if (masked && key + 16 * i + 8 * (k >> 1) > seen[n][k & 1]) s[i][n][k] = -INFINITY;
        }
    float top[NT][2], less[NT][2], ratio[NT][2];
    softmax(s, 2, top, less);
    float fraction;
    const float power = exponent_of(vs, fraction);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float old = unit[n][k] + less[n][k], now = fmaxf(old, top[n][k] + power);
        f[k] = old == now ? 1.f : ex2(old - now);
        unit[n][k] = now;
        ratio[n][k] = fraction * ex2(fminf(power - now, 126.f));  // past 126 there are no weights, or none that fp32 holds
      }
      const float f0 = f[0], f1 = f[1];
      if (__any_sync(0xffffffffu, f0 != 1.f || f1 != 1.f))
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          o[n][i][0] *= f0;
          o[n][i][1] *= f1;
          o[n][i][2] *= f0;
          o[n][i][3] *= f1;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t w0[NT], w1[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        w0[n] = transpose8(half2_bits(s[i][n][0] * ratio[n][0], s[i][n][1] * ratio[n][1]));
        w1[n] = transpose8(half2_bits(s[i][n][2] * ratio[n][0], s[i][n][3] * ratio[n][1]));
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        uint32_t a[4], z[4];
        numbers<E4M3>(__byte_perm(vw[i][0][w], vw[i][1][w], 0x5140), a[0], a[1]);
        numbers<E4M3>(__byte_perm(vw[i][2][w], vw[i][3][w], 0x5140), a[2], a[3]);
        numbers<E4M3>(__byte_perm(vw[i][0][w], vw[i][1][w], 0x7362), z[0], z[1]);
        numbers<E4M3>(__byte_perm(vw[i][2][w], vw[i][3][w], 0x7362), z[2], z[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16(o[n][2 * w], a, w0[n], w1[n]);
          mma_f16(o[n][2 * w + 1], z, w0[n], w1[n]);
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float f[2] = {exp2f(unit[n][0]), exp2f(unit[n][1])};  // from here on in weights
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[n][i][k] *= f[k & 1];
  }

  // ---- the open block: a tile of 16 keys per warp, by the CTA of the last part
  const int k0 = full + 16 * warp;
  if (split == p.splits - 1 && k0 < total) {
    wait_for(units);
    const __nv_bfloat16 *kr = c.kt + (head * KV8_RING + (k0 & (KV8_RING - 1))) * P, *vr = c.vt + (head * KV8_RING + (k0 & (KV8_RING - 1))) * P;
    float s[1][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[0][n][0] = s[0][n][1] = s[0][n][2] = s[0][n][3] = 0.f;
    const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < P / 32; ++j) {
      const int d = 8 * (t + 4 * j);
      const uint4 x = k0 + g < total ? *reinterpret_cast<const uint4*>(kr + g * P + d) : none;
      const uint4 y = k0 + g + 8 < total ? *reinterpret_cast<const uint4*>(kr + (g + 8) * P + d) : none;
      const uint32_t a[4] = {x.x, y.x, x.y, y.y}, e[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 z = row0 + n * 8 + g < p.rows && d < D ? *reinterpret_cast<const uint4*>(query(n) + d) : none;
        mma_bf16(s[0][n], a, z.x, z.y);
        mma_bf16(s[0][n], e, z.z, z.w);
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int key = k0 + g + 8 * (k >> 1);
        s[0][n][k] = key <= seen[n][k & 1] && key < total ? s[0][n][k] * p.scale2 : -INFINITY;
      }
    float top[NT][2], less[NT][2];
    softmax(s, 1, top, less);
    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float f0 = ex2(less[n][0]), f1 = ex2(less[n][1]);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        o[n][i][0] *= f0;
        o[n][i][1] *= f1;
        o[n][i][2] *= f0;
        o[n][i][3] *= f1;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t x = pack_bf16x2(s[0][n][2 * k], s[0][n][2 * k + 1]);
        const uint32_t y = pack_bf16x2(s[0][n][2 * k] - __uint_as_float(x << 16), s[0][n][2 * k + 1] - __uint_as_float(x & 0xffff0000u));
        hi[n][k] = transpose8(x);
        lo[n][k] = transpose8(y);
      }
    }
    uint4 z[4][P / 64];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int key = 2 * t + (r & 1) + 8 * (r >> 1);
#pragma unroll
      for (int j = 0; j < P / 64; ++j)
        z[r][j] = k0 + key < total ? *reinterpret_cast<const uint4*>(vr + key * P + (P / 8) * g + 8 * j) : none;
    }
    if (p.a.T > 1) {
      // a zero weight would not take a value that is no number out of the product: such values of tokens that some queries do not
      // see are set to zero, and the sums of the queries that see the token are no numbers
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        bool bad = false;
#pragma unroll
        for (int j = 0; j < P / 64; ++j)
#pragma unroll
          for (int w = 0; w < 4; ++w) bad = bad || bf16x2_special((&z[r][j].x)[w]);
        bad = bad && k0 + 2 * t + (r & 1) + 8 * (r >> 1) > pos;
        if (bad)
#pragma unroll
          for (int j = 0; j < P / 64; ++j) z[r][j] = none;
        for (uint32_t lanes = __ballot_sync(0xffffffffu, bad); lanes != 0; lanes &= lanes - 1) {
          const int key = k0 + 2 * ((__ffs(lanes) - 1) & 3) + (r & 1) + 8 * (r >> 1);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              if (key <= seen[n][k]) l[n][k] = __int_as_float(0x7fc00000);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < P / 64; ++j)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t *x0 = &z[0][j].x, *x1 = &z[1][j].x, *x2 = &z[2][j].x, *x3 = &z[3][j].x;
        const uint32_t a[4] = {__byte_perm(x0[w], x1[w], 0x5410), __byte_perm(x0[w], x1[w], 0x7632), __byte_perm(x2[w], x3[w], 0x5410),
                               __byte_perm(x2[w], x3[w], 0x7632)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_bf16(o[n][4 * j + w], a, hi[n][0], hi[n][1]);
          mma_bf16(o[n][4 * j + w], a, lo[n][0], lo[n][1]);
        }
      }
  }

  // ---- join the warps
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float x = l[n][k];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      const int q = n * 8 + 2 * t + k;
      if (g == 0) stat[warp][q] = make_float2(m[n][k], x);
      float* to = sums + (warp * NT * 8 + q) * (P + 4) + (P / 8) * g;
#pragma unroll
      for (int i = 0; i < KS; i += 2)  // columns P / 8 * g + 2 i ..: rows g and g + 8 of the products i and i + 1
        *reinterpret_cast<float4*>(to + 2 * i) = make_float4(o[n][i][k], o[n][i][k + 2], o[n][i + 1][k], o[n][i + 1][k + 2]);
    }
  __syncthreads();
  if (split == p.splits - 1 && !waited) wait_predecessors();  // this grid ends after the one before it, whatever it had to read
  const long long all = (long long)c.B * c.G * p.rows;
  for (int i = threadIdx.x; i < NT * 8 * (P / 4); i += DW * 32) {
    const int q = i / (P / 4), d = i % (P / 4) * 4, r = row0 + q;
    if (r >= p.rows) break;
    float mx = -INFINITY, f[DW], sum = 0.f;
#pragma unroll
    for (int w = 0; w < DW; ++w) mx = fmaxf(mx, stat[w][q].x);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < DW; ++w) {
      const float2 st = stat[w][q];
      if (st.x == -INFINITY && st.y == st.y) continue;  // no visible key
      f[w] = st.x == -INFINITY ? 1.f : ex2(st.x - mx);  // zero times sums that are no numbers is none
      sum += st.y * f[w];
      const float4 y = *reinterpret_cast<const float4*>(sums + (w * NT * 8 + q) * (P + 4) + d);
      x.x += y.x * f[w];
      x.y += y.y * f[w];
      x.z += y.z * f[w];
      x.w += y.w * f[w];
    }
    const long long row = head * p.rows + r;
    if (p.splits > 1) {
      *reinterpret_cast<float4*>(p.a.part + (split * all + row) * P + d) = x;
      if (d == 0) reinterpret_cast<float2*>(p.a.part + p.splits * all * P)[split * all + row] = make_float2(mx, sum);
    } else if (d < D) {
      const int tok = r / p.rep, h = kvh * p.rep + r % p.rep;
      float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (!idle && start + tok >= c.C) inv = __int_as_float(0x7fc00000), x = make_float4(inv, inv, inv, inv);
      uint2 z = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
      *reinterpret_cast<uint2*>(p.a.out + (((long long)b * p.a.T + tok) * p.a.H + h) * D + d) = z;
    }
  }
}

// Joins the parts of a query's keys: four warps take every fourth part each, a lane P / 32 neighbouring columns.
template <int P>
__global__ void __launch_bounds__(128) kv8_join_kernel(const StepParams p) {
  constexpr int COLS = P / 32;
  __shared__ float weight[MOST_SPLITS], sum[4], acc[4][P];
  const Kv8Cache& c = p.a.c;
  const long long all = (long long)c.B * c.G * p.rows, row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = row % p.rows, kvh = row / p.rows % c.G, b = row / p.rows / c.G;
  wait_predecessors();
  const float2* st = reinterpret_cast<const float2*>(p.a.part + p.splits * all * P);
  float mx = -INFINITY, l = 0.f;
  for (int s = lane; s < p.splits; s += 32) mx = fmaxf(mx, st[s * all + row].x);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
  for (int s = threadIdx.x; s < p.splits; s += 128) {
    const float2 x = st[s * all + row];
    const bool none = x.x == -INFINITY && x.y == x.y;  // no visible key
    const float f = x.x == -INFINITY ? 1.f : ex2(x.x - mx);
    weight[s] = none ? -1.f : f;
    l += none ? 0.f : x.y * f;
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
  if (lane == 0) sum[warp] = l;
  __syncthreads();
  float x[COLS] = {};
#pragma unroll 4
  for (int s = warp; s < p.splits; s += 4) {
    const float f = weight[s];
    const float* part = p.a.part + (s * all + row) * P + COLS * lane;
#pragma unroll
    for (int i = 0; i < COLS; ++i) x[i] += f < 0.f ? 0.f : part[i] * f;  // zero times sums that are no numbers is none
  }
#pragma unroll
  for (int i = 0; i < COLS; ++i) acc[warp][COLS * lane + i] = x[i];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= p.a.D) return;
  const float total = sum[0] + sum[1] + sum[2] + sum[3];
  const long long start = p.a.pos.at(b);
  const int tok = r / p.rep, h = kvh * p.rep + r % p.rep;
  float y = total == 0.f ? 0.f : (acc[0][d] + acc[1][d] + acc[2][d] + acc[3][d]) / total;
  if (start >= 0 && start + tok >= c.C) y = __int_as_float(0x7fc00000);
  p.a.out[(((long long)b * p.a.T + tok) * p.a.H + h) * p.a.D + d] = __float2bfloat16(y);
}

template <int P, bool E4M3, int NT>
int resident_blocks() {  // of a GPU, by registers and shared memory
  static int count[PerDeviceOnce::kMaxDevices] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= PerDeviceOnce::kMaxDevices) return 148;
  if (count[dev] == 0) {
    int sms = 0, per = 0;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kv8_attention_kernel<P, E4M3, NT>, DW * 32, step_smem(P, NT));
    count[dev] = std::max(1, sms * per);
  }
  return count[dev];
}

// How many blocks share a head's keys: of the largest numbers that fit in one to four rounds of the resident blocks the one with the
// least time, in units of keys per warp, where a block's start and end count as 6.
int splits_for(long long ctas, int units, int resident) {
  const long long most = std::min(MOST_SPLITS, std::max(1, units / (2 * DW)));
  long long best = 1, least = (ctas + resident - 1) / resident * ((units + DW - 1) / DW + 6);
  for (int rounds = 1; rounds <= 4; ++rounds) {
    const long long s = std::min(most, rounds * (long long)resident / ctas);
    if (s < 1) continue;
    const long long t = rounds * ((units + s * DW - 1) / (s * DW) + 6);
    if (t < least) least = t, best = s;
  }
  return (int)best;
}

StepParams plan(const Kv8Attention& a) {
  StepParams p{a};
  p.rep = a.H / a.c.G;
  p.rows = a.T * p.rep;
  const int nt = p.rows > 8 ? 2 : 1;
  p.tiles = (p.rows + 8 * nt - 1) / (8 * nt);
  p.scale2 = a.scale * 1.4426950408889634f;
  const int resident = a.c.P == 64 ? (a.c.e4m3 ? (nt == 1 ? resident_blocks<64, true, 1>() : resident_blocks<64, true, 2>())
                                               : (nt == 1 ? resident_blocks<64, false, 1>() : resident_blocks<64, false, 2>()))
                                   : (a.c.e4m3 ? (nt == 1 ? resident_blocks<128, true, 1>() : resident_blocks<128, true, 2>())
                                               : (nt == 1 ? resident_blocks<128, false, 1>() : resident_blocks<128, false, 2>()));
  p.splits = splits_for((long long)a.c.B * a.c.G * p.tiles, std::min(a.most, a.c.C) / UNIT, resident);
  return p;
}

template <typename... K, typename... A>
void launch(void (*kernel)(K...), unsigned grid, int threads, int smem, bool dependent, cudaStream_t s, const char* what, A&&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<K>(std::forward<A>(args))...);
  attention_check_launch(what);
}

template <int P, bool E4M3, int NT>
void run(const StepParams& p, cudaStream_t s) {
  const unsigned grid = (unsigned)((long long)p.splits * p.tiles * p.a.c.G * p.a.c.B);
  launch(kv8_attention_kernel<P, E4M3, NT>, grid, DW * 32, step_smem(P, NT), p.a.appended, s, "kv8_attention", p);
  if (p.splits > 1) launch(kv8_join_kernel<P>, (unsigned)((long long)p.a.c.B * p.a.c.G * p.rows), 128, 0, true, s, "kv8_join", p);
}
template <int P, bool E4M3>
void run_rows(const StepParams& p, cudaStream_t s) {
  if (p.rows > 8) run<P, E4M3, 2>(p, s);
  else run<P, E4M3, 1>(p, s);
}

}  // namespace

long long kv8_attention_scratch(const Kv8Attention& a) {
  const StepParams p = plan(a);
  return p.splits > 1 ? (long long)p.splits * a.c.B * a.c.G * p.rows * (a.c.P + 2) * 4 : 0;
}

void launch_kv8_attention(const Kv8Attention& a, cudaStream_t s) {
  const StepParams p = plan(a);
  if (a.c.P == 64) a.c.e4m3 ? run_rows<64, true>(p, s) : run_rows<64, false>(p, s);
  else a.c.e4m3 ? run_rows<128, true>(p, s) : run_rows<128, false>(p, s);
}

}  // namespace tb
