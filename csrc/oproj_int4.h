// o_proj with 4-bit weights and group scales: host interface (kernel in oproj_int4.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace helix {

// y[n, r] = sum_k x[n, k] (q[r, k] - z[r, k / group]) s[r, k / group], q and z in 0 .. 15 (no zero points: z = 8).
//
// Packed weights: a record per 128 rows (a slab; rows behind `hidden` are zeros) and 128 columns, slab by slab (the last record of
// a slab holds 64 columns where K is not a multiple of 128):
//   * [16-row tile][32 columns][row][16 bytes], four words of eight columns; column c of eight is nibble c / 2 + 4 (c % 2), so that a word
//     shifted by 4 i and masked is the pair of columns 2 i, 2 i + 1;
//   * per group the slab's 128 scales of 16 bits, tile by tile the pairs (row g, row g + 8), g = 0 .. 7;
//   * with zero points per group 128 bytes in the same order.
struct OprojInt4Params {
  CUtensorMap x_map;          // [tokens, K], box (64, n_pad), SWIZZLE_128B: only for more than kInt4FewTokens tokens
  const uint16_t* x;          // [tokens, K], rows x_stride elements apart
  int64_t x_stride;
  const uint8_t* w;           // packed, 16-byte aligned
  uint16_t* y;                // [tokens, hidden]
  int64_t y_stride;
  int* error_flag;            // set to a helix::Status code when a bounded wait runs out
  unsigned long long timeout_ns;
  int tokens, hidden, K, group, zeros, is_bf16;
  int batch;                  // set by the launch (few tokens): row tiles whose sums a CTA keeps before it adds them up
};

constexpr int kInt4FewTokens = 16;       // up to so many the weights stay in registers
constexpr int kInt4MaxTokens = 128;      // of one launch
constexpr int int4_pad_tokens(int tokens) { return tokens <= 32 ? 32 : tokens <= 64 ? 64 : 128; }
// How up to kInt4FewTokens tokens are divided: clusters of `cl` CTAs side by side cover K, a warp 256 columns, and cluster i takes the 16-row
// tiles i, i + columns, ...
struct Int4FewPlan {
  int cl, warps, columns;
  int batch;        // row tiles whose sums a CTA keeps before it adds them up and sends them on
  int batches;      // of the cluster with the most tiles
  int inboxes;      // sets of other CTAs' sums in shared memory: the batches take turns at two, a single one needs only its own
  size_t bytes;     // of shared memory
};
// for a grid of at most `resident` clusters
Int4FewPlan int4_few_plan(int tokens, int hidden, int K, int resident);
constexpr size_t int4_slab_bytes(int64_t K, int64_t group, bool zeros) { return (size_t)(K * 64 + K / group * (zeros ? 384 : 256)); }
cudaError_t launch_oproj_int4(OprojInt4Params p, bool pdl, int sm_count, cudaStream_t stream);

}  // namespace helix
