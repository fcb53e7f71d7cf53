// Key/value cache held in 8 bits: blocks of 64 tokens as codes times one scale per block and head, and the last 128 tokens as they
// came (bf16) in a ring, from which the block that is not full yet is read.
//
//   codes   [B, G, C, P]   int8: x = code * s, s = max|x| / 127;  e4m3: s = max|x| / 448;  C a multiple of 64, P 64 or 128 (>= D)
//   scales  [B, G, C / 64] fp32; a block that holds an infinity or NaN has the scale NaN and reads as NaN throughout
//   ring    [B, G, 128, P] position x is in row x % 128
// What the cache holds depends on the tokens alone, not on the portions in which they came. Up to 64 tokens can be taken back by
// going on from an earlier position. A sequence whose position is negative is idle: nothing of it is written, its outputs are zero.
// Tokens past the capacity C are not stored; their queries' outputs are NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attention.cuh"

namespace tb {

constexpr int KV8_BLOCK = 64, KV8_RING = 128;

struct Kv8Cache {
  uint8_t *k8, *v8;
  float *ks, *vs;
  __nv_bfloat16 *kt, *vt;
  int B, G, C, P;
  bool e4m3;
};

struct Kv8Pos {  // position per sequence: dev[b * step], or host where dev is null
  long long host;
  const long long* dev;
  int step;
  // positions past 2^62 are taken for that: tokens may be added to it
  __device__ __forceinline__ long long at(int b) const {
    const long long x = dev != nullptr ? dev[(long long)b * step] : host;
    return x < (1ll << 62) ? x : 1ll << 62;
  }
};

// k, v [B, T, G, D] (16-byte aligned rows) at positions pos .. pos + T - 1
void launch_kv8_append(const Kv8Cache& c, const AttentionView& k, const AttentionView& v, int T, int D, const Kv8Pos& pos, cudaStream_t s);
// k, v [B, G, rows, D] contiguous: the values of the first `length` positions, zero from there on
void launch_kv8_expand(const Kv8Cache& c, __nv_bfloat16* k, __nv_bfloat16* v, int rows, int D, const Kv8Pos& length, cudaStream_t s);

// For tensor-core attention over the cache: k, v [B, G, rows, D] hold codes (and the open block's tokens) as bf16 numbers, which they
// are exactly, k_scales and v_scales [B, G, ceil(rows / 64)] what blocks are multiplied by (1 for the open one, 0 past the end); rows
// past a sequence's end are left as they are. starts and ends [B] (or null): positions, and those plus T (0 for idle sequences).
// new_k, new_v [B, T, G, D] (or null): tokens from the position on as they came, in place of what the cache holds of them; it need not hold
// them yet, and must hold the open block before them (launch_kv8_append comes after).
struct Kv8Codes {
  __nv_bfloat16 *k, *v;
  float *k_scales, *v_scales;
  long long *starts, *ends;
  AttentionView new_k, new_v;
};
void launch_kv8_codes(const Kv8Cache& c, const Kv8Codes& to, int rows, int D, const Kv8Pos& pos, int T, cudaStream_t s);
// out [B, T, width]: NaN at the positions past the capacity
void launch_kv8_outside(const Kv8Cache& c, __nv_bfloat16* out, int T, int width, const Kv8Pos& pos, cudaStream_t s);

struct Kv8Attention {
  Kv8Cache c;
  AttentionView q;     // [B, T, H, D]
  __nv_bfloat16* out;  // [B, T, H, D] contiguous
  float* part;         // kv8_attention_scratch bytes, or null
  int T, H, D;
  Kv8Pos pos;
  float scale;
  int most;            // tokens that a sequence may hold after these: what the work is split by
  bool appended;       // launch_kv8_append of the same tokens comes right before on the stream
};
long long kv8_attention_scratch(const Kv8Attention& a);
void launch_kv8_attention(const Kv8Attention& a, cudaStream_t s);

}  // namespace tb
