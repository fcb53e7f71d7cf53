// Softmax attention of training batches and prompts, and from a key/value cache held in 8 bits.
//
// Queries are [B, T, H, D], keys and values [B, S, G, D] with H a multiple of G (query head h reads key/value head h / (H / G)); bf16,
// fp32 scores, statistics and accumulators. Query i of sequence b stands at position start(b) + i. Key j is visible to it when
//   j < length(b),   j <= position (causal),   j > position - window (window > 0).
// A query that sees no key has output zero and passes no gradient on.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <stdexcept>
#include <string>

namespace tb {

// Element (batch, row, head, d) is at b * sb + row * sr + head * sh + d.
struct AttentionView {
  const void* p;
  long long sr, sh, sb;
};

struct AttentionShape {
  int B, T, S, H, G, D;
  float scale;  // > 0
  bool causal;
  long long window;              // 0: none; up to 2^61
  const long long* lengths;      // [B] or null (S)
  const long long* starts;       // [B] or null (`start` for all)
  long long start;
};

// Rows of the statistics [B, H, attention_rows(T)]: whole tiles, so that they are fetched in whole tiles.
inline int attention_rows(int T) { return (T + 127) / 128 * 128; }

// out [B, T, H, D] contiguous; lse (or null): minus the base-2 logarithm of the sum of the rows' exponentials; -inf for rows that see
// no key and rows past T, whose weights are zero that way.
// rest (or null): what the outputs lost when they were rounded, for the backward pass: the rows' sums of dout times out enter every
// gradient, and with the rounded outputs alone those of short rows were off by up to 4e-3 of themselves instead of 2.4e-3. It costs a tensor of
// the outputs' size that is kept until the backward pass (queries, keys, values, outputs, this: a quarter more than without, where heads are not shared).
// part (attention_fwd_scratch(a) bytes or null): where the keys of few queries are split over blocks.
// k_scales, v_scales (or null): [B, G, blocks], what blocks of 64 keys and values are multiplied by.
struct AttentionFwd {
  AttentionShape a;
  AttentionView q, k, v;
  __nv_bfloat16 *out, *rest;
  float* lse;
  float* part;
  int* status;
  const float *k_scales, *v_scales;
  int blocks;
};
long long attention_fwd_scratch(const AttentionShape& a);
void launch_attention_fwd(const AttentionFwd& f, cudaStream_t s);

// dq [B, T, H, D], dk, dv [B, S, G, D] contiguous; delta [B, H, attention_rows(T)] is written and read
// (minus the rows' sums of dout times out).
struct AttentionBwd {
  AttentionShape a;
  AttentionView q, k, v, out, rest, dout;
  const float* lse;
  float* delta;
  __nv_bfloat16 *dq, *dk, *dv;
  int* status;
};
void launch_attention_bwd(const AttentionBwd& f, cudaStream_t s);

// whether one of two bf16 numbers is an infinity or NaN
__device__ __forceinline__ bool bf16x2_special(uint32_t w) { return (((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0; }

inline void attention_check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace tb
