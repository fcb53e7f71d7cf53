// What the kernels of attention over bf16 keys share: which tiles of 128 keys a tile of 128 queries sees, and TMA maps.
#pragma once
#include "../common/ptx.cuh"
#include "../common/tma_desc.h"
#include "attention.cuh"

namespace tb {
namespace {

constexpr int AT_M = 128;             // queries of a tile, keys of a tile
constexpr int AT_BOX = AT_M * 64 * 2;  // bytes of a box of 128 rows and 64 columns
constexpr float LOG2E = 1.4426950408889634f;

struct Visible {  // of one sequence
  int start, length, window;
  bool causal;
  __device__ __forceinline__ Visible(const AttentionShape& a, int b) : window(a.window), causal(a.causal) {
    // positions past these limits see what those at the limits see
    const long long s0 = a.starts != nullptr ? a.starts[b] : a.start, lim = 1ll << 30;
    start = (int)(s0 < -lim ? -lim : s0 > lim ? lim : s0);
    const long long n = a.lengths != nullptr ? a.lengths[b] : a.S;
    length = (int)(n < 0 ? 0 : n > a.S ? a.S : n);
  }
  // keys low(t) .. high(t) are visible to query t; both grow with t
  __device__ __forceinline__ int low(int t) const { return window > 0 ? max(0, start + t - window + 1) : 0; }
  __device__ __forceinline__ int high(int t) const { return causal ? min(length - 1, start + t) : length - 1; }
  // queries first(j) .. last(j, T) see key j
  __device__ __forceinline__ int first(int j) const { return causal ? max(0, j - start) : 0; }
  __device__ __forceinline__ int last(int j, int T) const { return window > 0 ? (int)min((long long)T - 1, (long long)j + window - 1 - start) : T - 1; }
  // tiles [x, y) of keys that queries t0 .. t1 see
  __device__ __forceinline__ int2 tiles(int t0, int t1) const {
    const int lo = low(t0), hi = high(t1);
    return hi < lo ? make_int2(0, 0) : make_int2(lo / AT_M, hi / AT_M + 1);
  }
  // whether all of queries t0 .. t1 see all of the 128 keys from key on
  __device__ __forceinline__ bool whole(int t0, int t1, int key) const { return low(t1) <= key && high(t0) >= key + AT_M - 1; }
};

// 64-wide boxes of 128 rows of one head: coordinates (column, row, head, batch); what is outside reads as zero
inline CUtensorMap attention_map(const AttentionView& v, int d, int rows, int heads, int batch, uint32_t box_rows = AT_M) {
  return make_tmap_4d_bf16(v.p, {(uint64_t)d, (uint64_t)rows, (uint64_t)heads, (uint64_t)batch},
                           {(uint64_t)v.sr * 2, (uint64_t)v.sh * 2, (uint64_t)v.sb * 2}, box_rows);
}

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int N>
__device__ __forceinline__ void named_barrier(int id) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

// 16 bytes (8 bf16) at `o + c` of a row of D values from fp32 registers
__device__ __forceinline__ void store_row16(__nv_bfloat16* o, int c, int D, const uint32_t (&v)[16], float r) {
#pragma unroll
  for (int g = 0; g < 2; ++g)
    if (c + 8 * g < D) {
      uint4 u;
      uint32_t* up = &u.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) up[i] = pack_bf16x2(__uint_as_float(v[8 * g + 2 * i]) * r, __uint_as_float(v[8 * g + 2 * i + 1]) * r);
      *reinterpret_cast<uint4*>(o + c + 8 * g) = u;
    }
}

}  // namespace
}  // namespace tb
