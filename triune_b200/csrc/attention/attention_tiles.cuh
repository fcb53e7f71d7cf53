// What the kernels of attention over bf16 keys share: which tiles of 128 keys a tile of 128 queries sees, TMA maps, the number of SMs.
#pragma once
#include "../common/per_device.h"
#include "../common/ptx.cuh"
#include "../common/tma_desc.h"
#include "attention.cuh"

namespace tb {
namespace {

constexpr int AT_M = 128;             // queries of a tile, keys of a tile
constexpr int AT_BOX = AT_M * 64 * 2;  // bytes of a box of 128 rows and 64 columns
constexpr float LOG2E = 1.4426950408889634f;

// A value that all threads of the warp have, made known as such: what is formed from it stays in the warp's uniform registers, from
// which tensor-core instructions take their operands
template <typename T>
__device__ __forceinline__ T uniform(T x) {
  return __shfl_sync(0xffffffffu, x, 0);
}

struct Visible {  // of one sequence
  int start, before, length;  // before: what a query's first visible key is ahead of its number
  bool causal, window;
  __device__ __forceinline__ Visible(const AttentionShape& a, int b) : causal(a.causal), window(a.window > 0) {
    // positions past these limits see what those at the limits see
    const long long lim = 1ll << 30, far = 1ll << 61, given = a.starts != nullptr ? a.starts[b] : a.start;
    const long long s0 = given < -far ? -far : given > far ? far : given, w0 = s0 - a.window + 1;
    start = uniform((int)(s0 < -lim ? -lim : s0 > lim ? lim : s0));
    before = uniform((int)(w0 < -lim ? -lim : w0 > lim ? lim : w0));
    const long long n = a.lengths != nullptr ? a.lengths[b] : a.S;
    length = uniform((int)(n < 0 ? 0 : n > a.S ? a.S : n));
  }
  // keys low(t) .. high(t) are visible to query t; both grow with t
  __device__ __forceinline__ int low(int t) const { return window ? max(0, before + t) : 0; }
  __device__ __forceinline__ int high(int t) const { return causal ? min(length - 1, start + t) : length - 1; }
  // queries first(j) .. last(j, T) see key j
  __device__ __forceinline__ int first(int j) const { return causal ? max(0, j - start) : 0; }
  __device__ __forceinline__ int last(int j, int T) const { return window ? min(T - 1, j - before) : T - 1; }
  // tiles [x, y) of so many keys that queries t0 .. t1 see
  __device__ __forceinline__ int2 tiles(int t0, int t1, int keys = AT_M) const {
    const int lo = low(t0), hi = high(t1);
    return hi < lo ? make_int2(0, 0) : make_int2(lo / keys, hi / keys + 1);
  }
  // whether all of queries t0 .. t1 see all of so many keys from key on
  __device__ __forceinline__ bool whole(int t0, int t1, int key, int keys = AT_M) const { return low(t1) <= key && high(t0) >= key + keys - 1; }
};

// Bits lo .. hi of 32, whichever of them there are
__device__ __forceinline__ uint32_t visible_bits(int lo, int hi) {
  const uint32_t below = hi >= 31 ? 0xffffffffu : hi < 0 ? 0u : (2u << hi) - 1u, before = lo <= 0 ? 0u : lo > 31 ? 0xffffffffu : (1u << lo) - 1u;
  return below & ~before;
}

// 2^x of two values up to 2^7 (below 2^-126: 2^-126): x = n + r with |r| <= 1/2, a polynomial of degree 4 in r (minimax of the relative
// error, 2.6e-6, by the exchange algorithm of Remez), times 2^n. What is no number stays so. The units that multiply and add have room where
// the exponential unit, at 16 results per clock, is what a tile waits for.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  float a, b;
  unpack_f2(x, a, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-126.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-126.f));
  x = pack_f2(a, b);
  const float big = 12582912.f;  // 1.5 * 2^23: the sum's last bits are the rounded x
  const uint64_t t = add2(x, pack_f2(big, big));
  const uint64_t r = add2(x, mul2(add2(t, pack_f2(-big, -big)), pack_f2(-1.f, -1.f)));
  uint64_t y = pack_f2(9.570102207362652e-3f, 9.570102207362652e-3f);
  y = fma2(y, r, pack_f2(5.591785907745361e-2f, 5.591785907745361e-2f));
  y = fma2(y, r, pack_f2(0.240247443318367f, 0.240247443318367f));
  y = fma2(y, r, pack_f2(0.6931217908859253f, 0.6931217908859253f));
  y = fma2(y, r, pack_f2(0.9999992847442627f, 0.9999992847442627f));
  unpack_f2(t, a, b);
  return mul2(y, pack_f2(__uint_as_float(__float_as_uint(a) * 0x800000u + 0x3f800000u), __uint_as_float(__float_as_uint(b) * 0x800000u + 0x3f800000u)));
}

inline int multiprocessors() {
  static int count[PerDeviceOnce::kMaxDevices] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= PerDeviceOnce::kMaxDevices) return 148;
  if (count[dev] == 0) cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev);
  return count[dev];
}

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

// A warpgroup's registers per thread from here on; the shares of a block's warpgroups have to fit what it was launched with.
template <int N>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// Products of tiles, issued by one elected thread of a warp that stays together: every thread comes to the waits and to the end of each
// issue (`issue`), since the operands are in registers that all threads of a warp share. Descriptors are formed once per tile and moved
// on by constants: formed for each product, the issuing thread took 125 clocks a product, twice what the tensor core needs for it.
template <typename F>
__device__ __forceinline__ void issue(F f) {
  if (elect_one()) f();
  __syncwarp();
}
// D = A B^T over the head dimension, `steps` times 16 columns; tiles of DB boxes of 64 columns, A of 128 rows and B of N.
template <int DB, int N = AT_M>
__device__ __forceinline__ void scores_product(uint32_t d, uint32_t a, uint32_t b, int steps) {
  constexpr uint32_t idesc = make_idesc(AT_M, N, 1, 1, 0, 0);
  static_assert(N == AT_M || DB == 1, "the boxes of a tile are equally far apart in A and B");
  const uint64_t da = make_smem_desc(a, 16, 1024), db = make_smem_desc(b, 16, 1024);
#pragma unroll
  for (int k = 0; k < 4 * DB; ++k)
    if (k < steps) {
      const uint32_t off = ((k >> 2) * AT_BOX + (k & 3) * 32) >> 4;
      umma_bf16(d, da + off, db + off, idesc, k > 0);
    }
}
// D (+)= A B, A: 16-column steps K0 .. K0 + N - 1 of 128 x 128 bf16 in TMEM (step k at `a` + columns at(k)), B: rows of a [128][64 DB] tile
template <int DB, int K0, int N, typename At>
__device__ __forceinline__ void rows_product(uint32_t d, uint32_t a, uint32_t b, bool add, At at) {
  constexpr uint32_t idesc = make_idesc(AT_M, 64 * DB, 1, 1, 0, 1);
  const uint64_t db = make_smem_desc(b, AT_BOX, 1024);
#pragma unroll
  for (int k = K0; k < K0 + N; ++k) umma_bf16_ts(d, a + at(k), db + ((k * 2048) >> 4), idesc, k > 0 || add);
}

// Loads of 32, 64 or 16 columns of this warp's lanes that are complete when they return. Load and wait are one statement: a load lands
// in its registers whenever it does, and nothing else would keep the compiler from moving or spilling registers that it has still to
// write (which turns into wrong values and wrong addresses as soon as registers are short).
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&x)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
               "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]),
                 "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]), "=r"(x[20]),
                 "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]), "=r"(x[28]), "=r"(x[29]), "=r"(x[30]),
                 "=r"(x[31])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&x)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]),
                 "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&x)[32], uint32_t (&y)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
               "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, "
               "%46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]),
                 "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]), "=r"(x[20]),
                 "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]), "=r"(x[28]), "=r"(x[29]), "=r"(x[30]),
                 "=r"(x[31]), "=r"(y[0]), "=r"(y[1]), "=r"(y[2]), "=r"(y[3]), "=r"(y[4]), "=r"(y[5]), "=r"(y[6]), "=r"(y[7]), "=r"(y[8]), "=r"(y[9]),
                 "=r"(y[10]), "=r"(y[11]), "=r"(y[12]), "=r"(y[13]), "=r"(y[14]), "=r"(y[15]), "=r"(y[16]), "=r"(y[17]), "=r"(y[18]), "=r"(y[19]),
                 "=r"(y[20]), "=r"(y[21]), "=r"(y[22]), "=r"(y[23]), "=r"(y[24]), "=r"(y[25]), "=r"(y[26]), "=r"(y[27]), "=r"(y[28]), "=r"(y[29]),
                 "=r"(y[30]), "=r"(y[31])
               : "r"(at)
               : "memory");
}

// A wait of a whole warp. Its threads may see the barrier's phase end at different times; the tcgen05 loads and stores that follow
// are instructions of whole warps, so the warp is brought together here.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }

template <int N>
__device__ __forceinline__ void named_barrier(int id) {
  __syncwarp();  // warps are counted, not threads
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

// What bf16 loses of 16 values times r, as bf16, at `o + c` of a row of D values
__device__ __forceinline__ void store_rest16(__nv_bfloat16* o, int c, int D, const uint32_t (&v)[16], float r) {
#pragma unroll
  for (int g = 0; g < 2; ++g)
    if (c + 8 * g < D) {
      uint4 u;
      uint32_t* up = &u.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = __uint_as_float(v[8 * g + 2 * i]) * r, b = __uint_as_float(v[8 * g + 2 * i + 1]) * r;
        const uint32_t x = pack_bf16x2(a, b);
        up[i] = pack_bf16x2(a - __uint_as_float(x << 16), b - __uint_as_float(x & 0xffff0000u));
      }
      *reinterpret_cast<uint4*>(o + c + 8 * g) = u;
    }
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
