// o_proj with 4-bit weights and group scales: host interface (kernels in oproj_int4.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace helix {

// y[n, r] = sum_k x[n, k] (q[r, k] - z[r, k / group]) s[r, k / group], q and z in 0 .. 15 (no zero points: z = 8).
//
// Packed weights: per 16 rows and 64 columns 512 bytes, 16 for each lane of a warp, four words of eight nibbles, one word per
// 16 x 16 x 8 MMA.  Nibbles i and i + 4 of word s of lane (g, t) are the A operand's register i:
//   row g + 8 (i & 1), columns k and k + 1,  k = 32 (s >> 1) + 8 t + 4 (s & 1) + 2 (i >> 1)
// so that a lane's B operands of 32 columns are 16 consecutive bytes of x.  Scales (16 bits) and zero points (8 bits): per 16 rows
// and group the pairs (row g, row g + 8), g = 0 .. 7.
struct OprojInt4Params {
  const uint16_t* x;          // [tokens, K], rows x_stride elements apart
  int64_t x_stride;
  const uint4* w;             // [hidden / 16][K / 64][32]
  const uint32_t* scales;     // [hidden / 16][K / group][8]
  const uint16_t* zeros;      // the same, or null
  uint16_t* y;                // [tokens, hidden]
  int64_t y_stride;
  int tokens, hidden, K, group, is_bf16;
};

constexpr int kInt4MaxTokens = 16;       // of one launch
constexpr int kInt4MaxK = 32768;
cudaError_t launch_oproj_int4(const OprojInt4Params& p, bool pdl, int sm_count, cudaStream_t stream);

}  // namespace helix
