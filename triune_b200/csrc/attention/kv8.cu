// Tokens into and out of the 8-bit cache. Both kernels pass over the data once, a CTA per block of 64 tokens of one head, of keys or
// of values; rows are read and written in 16-byte pieces (codes in 8-byte pieces). Bound by memory with many tokens, by arithmetic on the
// way in with e4m3: 32 x 8191 tokens, 8 heads of 128 (1.6 GB), with a cold L2: appending 373 us (4300 GB/s) in int8, 449 in e4m3; expanding
// 280 us (5700 GB/s). 4 x 4096 tokens: 36, 39 and 25 us.
#include <cuda_fp8.h>

#include "../common/dependent_launch.cuh"
#include "kv8.cuh"

namespace tb {
namespace {

struct AppendParams {
  Kv8Cache c;
  AttentionView k, v;
  int T, D, blocks;
  Kv8Pos pos;
};

template <bool E4M3>
__device__ __forceinline__ uint32_t code_of(float y) {
  if constexpr (E4M3) return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)__float2int_rn(y) & 0xffu;
}

// Four codes: the nearest ones to the quotients x / s, rounded to fp32 first. Divisions and conversions to integers took 85 % of the issue
// slots (37 us for 67 MB), so quotients are products with 1 / s, off by less than 2^-22 of themselves, and codes come from the last
// bits of a sum with 1.5 * 2^23, or in pairs (e4m3). Where a product is so near the border between two codes that the quotient might
// lie beyond it, the codes are formed from divisions.
template <bool E4M3>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float s, float inv) {
  float y[4];
  bool near = false;
  uint32_t code;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = x[i] * inv;
  if constexpr (E4M3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // borders: halfway between numbers of three bits; below the least normal number they are others
      const uint32_t bits = __float_as_uint(y[i]) & 0x7fffffffu;
      near = near || (bits & 0xfffffu) - 0x7fff0u <= 0x20u || (bits < 0x3c800000u && bits != 0) || bits > 0x7f800000u;
    }
    code = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3) |
           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3) << 16;
  } else {
    const float big = 12582912.f;
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = __fadd_rn(y[i], big);
      near = near || !(fabsf(y[i] - __fadd_rn(t[i], -big)) <= 0.4999f);
    }
    code = __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040), __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
  }
  if (near)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = code_of<E4M3>(__fdiv_rn(x[i], s));
      code = i == 0 ? c : code | c << (8 * i);
    }
  return code;
}

// A thread has PIECES pieces of 8 columns of a block.
template <int P, bool E4M3>
__global__ void __launch_bounds__(256) kv8_append_kernel(const AppendParams p) {
  constexpr int ACROSS = P / 8, PIECES = KV8_BLOCK * ACROSS / 256;
  __shared__ uint32_t most[8];
  allow_dependents();  // attention that reads other blocks may start
  long long at = blockIdx.x;
  const int i = at % p.blocks;
  at /= p.blocks;
  const int side = at & 1;
  at >>= 1;
  const int g = at % p.c.G, b = at / p.c.G;
  const long long start = p.pos.at(b);
  if (start < 0 || start >= p.c.C) return;
  const int begin = (int)start, end = (int)min((long long)p.c.C, start + p.T);
  const int m = begin / KV8_BLOCK + i, base = m * KV8_BLOCK;
  if (base >= end) return;
  const long long head = (long long)b * p.c.G + g;
  const AttentionView& x = side ? p.v : p.k;
  const __nv_bfloat16* rows = (const __nv_bfloat16*)x.p + b * x.sb + g * x.sh;
  uint4* ring = reinterpret_cast<uint4*>((side ? p.c.vt : p.c.kt) + head * KV8_RING * P);
  auto token = [&](int pos, int piece) {  // of the new ones
    return piece * 8 < p.D ? *reinterpret_cast<const uint4*>(rows + (long long)(pos - begin) * x.sr + piece * 8) : make_uint4(0, 0, 0, 0);
  };
  if (base + KV8_BLOCK <= end) {
    uint4 z[PIECES];
    uint32_t top = 0;  // magnitudes of bf16 numbers order like their bits, infinities and NaN above all
#pragma unroll
    for (int e = 0; e < PIECES; ++e) {
      const int at = threadIdx.x + 256 * e, row = at / ACROSS, piece = at % ACROSS;
      z[e] = base + row < begin ? ring[(m & 1) * KV8_BLOCK * ACROSS + at] : token(base + row, piece);
      const uint32_t* w = &z[e].x;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = max(top, most[w]);
    const float s = top >= 0x7f80u ? __int_as_float(0x7fc00000) : __fdiv_rn(__uint_as_float(top << 16), E4M3 ? 448.f : 127.f);
    if (threadIdx.x == 0) (side ? p.c.vs : p.c.ks)[head * (p.c.C / KV8_BLOCK) + m] = s;
    uint2* codes = reinterpret_cast<uint2*>((side ? p.c.v8 : p.c.k8) + (head * p.c.C + base) * P);
    // 1 / s is a normal number, or the block is zero throughout, reads as NaN whatever its codes, or is too small to be told from zero
    // in products: then divisions
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    const bool tiny = s > 0.f && s < 1e-36f;
#pragma unroll
    for (int e = 0; e < PIECES; ++e) {
      const uint32_t* w = &z[e].x;
      uint32_t o[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float x[4] = {__uint_as_float(w[2 * k] << 16), __uint_as_float(w[2 * k] & 0xffff0000u), __uint_as_float(w[2 * k + 1] << 16),
                            __uint_as_float(w[2 * k + 1] & 0xffff0000u)};
        o[k] = s > 0.f ? codes_of<E4M3>(x, s, tiny ? __int_as_float(0x7fc00000) : inv) : 0u;
      }
      codes[threadIdx.x + 256 * e] = make_uint2(o[0], o[1]);
    }
  }
  // The first two blocks write the ring, each its half: the newest token of every row. The first block's threads have read the old
  // rows of their own places above.
  if (i < 2) {
#pragma unroll
    for (int e = 0; e < PIECES; ++e) {
      const int at = threadIdx.x + 256 * e, row = at / ACROSS, slot = (m & 1) * KV8_BLOCK + row;
      const int pos = end - 1 - ((end - 1 - slot) & (KV8_RING - 1));
      if (pos >= begin) ring[(m & 1) * KV8_BLOCK * ACROSS + at] = token(pos, at % ACROSS);
    }
  }
}

struct ExpandParams {
  Kv8Cache c;
  Kv8Codes to;  // scales: null where values are asked for
  int rows, D, blocks;
  Kv8Pos pos;
  int T;  // the sequences' length is their position plus T; idle ones have none
};

template <int P, bool E4M3, bool CODES>
__global__ void __launch_bounds__(256) kv8_expand_kernel(const ExpandParams p) {
  constexpr int ACROSS = P / 8, PIECES = KV8_BLOCK * ACROSS / 256;
  long long at = blockIdx.x;
  const int m = at % p.blocks;
  at /= p.blocks;
  const int side = at & 1;
  at >>= 1;  // head
  const AttentionView& fresh = side ? p.to.new_v : p.to.new_k;
  const long long start = p.pos.at(at / p.c.G), given = start < 0 ? 0 : start + p.T;
  const int end = (int)min(given, (long long)p.c.C), base = m * KV8_BLOCK;
  const int n = CODES && fresh.p != nullptr ? (int)min(max(start, 0ll), (long long)end) : end;  // tokens that are read from the cache
  const bool full = base + KV8_BLOCK <= n;
  __nv_bfloat16* out = (side ? p.to.v : p.to.k) + (at * p.rows + base) * p.D;
  const uint2* codes = reinterpret_cast<const uint2*>((side ? p.c.v8 : p.c.k8) + (at * p.c.C + base) * P);
  const uint4* ring = reinterpret_cast<const uint4*>((side ? p.c.vt : p.c.kt) + (at * KV8_RING + (m & 1) * KV8_BLOCK) * P);
  float s = full ? (side ? p.c.vs : p.c.ks)[at * (p.c.C / KV8_BLOCK) + m] : 0.f;
  if constexpr (CODES) {
    if (threadIdx.x == 0) {
      (side ? p.to.v_scales : p.to.k_scales)[at * p.blocks + m] = full ? s : base < end ? 1.f : 0.f;
      if (p.to.ends != nullptr && m == 0 && side == 0 && at % p.c.G == 0) {
        p.to.starts[at / p.c.G] = start;
        p.to.ends[at / p.c.G] = end;
      }
    }
    s = 1.f;
  }
#pragma unroll
  for (int e = 0; e < PIECES; ++e) {
    const int i = threadIdx.x + 256 * e, row = i / ACROSS, piece = i % ACROSS;
    if (base + row >= p.rows || piece * 8 >= p.D || (CODES && base + row >= end)) continue;
    uint4 z = make_uint4(0, 0, 0, 0);
    if (full) {
      const uint2 c = codes[i];
      float x[8];
      if constexpr (E4M3) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((k < 2 ? c.x : c.y) >> (16 * (k & 1))), __NV_E4M3);
          const float2 y = __half22float2(__half2(r));
          x[2 * k] = y.x, x[2 * k + 1] = y.y;
        }
      } else {  // code + 128 in the last bits of 2^23 + ..
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(__byte_perm((k < 4 ? c.x : c.y) ^ 0x80808080u, 0x4b000000u, 0x7440 | (k & 3))) - 8388736.f;
      }
      uint32_t* w = &z.x;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const __nv_bfloat162 y = __floats2bfloat162_rn(x[2 * k] * s, x[2 * k + 1] * s);
        w[k] = *reinterpret_cast<const uint32_t*>(&y);
      }
    } else if (base + row < n) {
      z = ring[i];
    } else if (CODES && base + row < end) {
      z = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)fresh.p + at / p.c.G * fresh.sb + at % p.c.G * fresh.sh + (base + row - start) * fresh.sr + piece * 8);
    }
    *reinterpret_cast<uint4*>(out + (long long)row * p.D + piece * 8) = z;
  }
}

__global__ void __launch_bounds__(128) kv8_outside_kernel(__nv_bfloat16* out, int T, int width, int C, const Kv8Pos pos) {
  const long long row = blockIdx.x, start = pos.at(row / T);
  if (start < 0 || start + row % T < C) return;
  for (int i = threadIdx.x; i < width; i += 128) out[row * width + i] = __float2bfloat16(__int_as_float(0x7fc00000));
}

template <bool CODES>
void expand(const ExpandParams& p, cudaStream_t s) {
  const unsigned grid = (unsigned)((long long)p.blocks * 2 * p.c.B * p.c.G);
  if (p.c.P == 64) (p.c.e4m3 ? kv8_expand_kernel<64, true, CODES> : kv8_expand_kernel<64, false, CODES>)<<<grid, 256, 0, s>>>(p);
  else (p.c.e4m3 ? kv8_expand_kernel<128, true, CODES> : kv8_expand_kernel<128, false, CODES>)<<<grid, 256, 0, s>>>(p);
  attention_check_launch("kv8_expand");
}

}  // namespace

void launch_kv8_append(const Kv8Cache& c, const AttentionView& k, const AttentionView& v, int T, int D, const Kv8Pos& pos, cudaStream_t s) {
  const int blocks = (T + KV8_BLOCK - 2) / KV8_BLOCK + 1;  // that T tokens can touch
  const AppendParams p{c, k, v, T, D, blocks, pos};
  const unsigned grid = (unsigned)((long long)blocks * 2 * c.B * c.G);
  if (c.P == 64) (c.e4m3 ? kv8_append_kernel<64, true> : kv8_append_kernel<64, false>)<<<grid, 256, 0, s>>>(p);
  else (c.e4m3 ? kv8_append_kernel<128, true> : kv8_append_kernel<128, false>)<<<grid, 256, 0, s>>>(p);
  attention_check_launch("kv8_append");
}

void launch_kv8_expand(const Kv8Cache& c, __nv_bfloat16* k, __nv_bfloat16* v, int rows, int D, const Kv8Pos& length, cudaStream_t s) {
  expand<false>(ExpandParams{c, Kv8Codes{k, v}, rows, D, (rows + KV8_BLOCK - 1) / KV8_BLOCK, length, 0}, s);
}

void launch_kv8_codes(const Kv8Cache& c, const Kv8Codes& to, int rows, int D, const Kv8Pos& pos, int T, cudaStream_t s) {
  expand<true>(ExpandParams{c, to, rows, D, (rows + KV8_BLOCK - 1) / KV8_BLOCK, pos, T}, s);
}

void launch_kv8_outside(const Kv8Cache& c, __nv_bfloat16* out, int T, int width, const Kv8Pos& pos, cudaStream_t s) {
  kv8_outside_kernel<<<(unsigned)((long long)c.B * T), 128, 0, s>>>(out, T, width, c.C, pos);
  attention_check_launch("kv8_outside");
}

}  // namespace tb
