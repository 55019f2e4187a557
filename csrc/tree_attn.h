// Attention of a tree of drafted tokens over the paged cache: host interface (kernels in tree_attn.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace helix {

struct TreeDecodeParams {
  CUtensorMap k_map;               // 4-D (d, token in page, kv head, page), box (64, box_tok, 1, 1), SWIZZLE_128B
  CUtensorMap v_map;               // 5-D (d % 64, token in page, d / 64, kv head, page), box (64, box_tok, 2, 1, 1), SWIZZLE_128B
  const uint16_t* q;               // [rows, Hq, 128] bf16 or fp16
  int64_t q_sr, q_sh;              // elements
  const uint16_t* v;               // the V cache itself, for values that are not finite
  int64_t v_sp, v_st, v_sh;        // elements
  const int32_t* block_table;      // [B, max_pages]
  int64_t bt_stride;
  const int32_t* seq_lens;         // [B] local tokens, drafted ones among them
  const int32_t* q_start;          // [B + 1]
  const int32_t* draft_lens;       // [B]
  const uint64_t* mask;            // [rows, words]
  int64_t mask_stride;
  uint16_t* o;                     // [rows, Hq, 128] contiguous
  float* lse;                      // [rows, Hq]
  float* part_o;                   // scratch: pieces [2 * ctas][128 * tiles][128]
  float* part_lse;                 // scratch: [2 * ctas][128 * tiles], behind it int4 [ctas] notes for the fold
  int* error_flag;
  int rows, B, Hq, Hkv, page_size, max_pages, n_pages, box_tok, words;
  int ctas, tiles;                 // tiles of 128 rows that a CTA works on: 1 or 2
  int whole;                       // 1: CTAs take units from end to end, nothing is split and no second kernel runs
  int is_bf16, lse_base2;
  float scale;
  unsigned long long timeout_ns;
};

constexpr int kTreeMaxWords = 4;
constexpr size_t tree_part_o_floats(int ctas, int tiles) { return (size_t)2 * ctas * 128 * tiles * 128; }
constexpr size_t tree_notes_at(int ctas, int tiles) { return (size_t)2 * ctas * 128 * tiles; }     // in part_lse
constexpr size_t tree_part_lse_floats(int ctas, int tiles) { return tree_notes_at(ctas, tiles) + (size_t)ctas * 4; }
// how a call with up to max_q new tokens per sequence and max_seq_len tokens of the longest is divided
struct TreePlan {
  int tiles, ctas, whole;
};
TreePlan tree_plan(int B, int Hkv, int group, int max_q, int max_seq_len, int sm_count);
// places on the line that the KV tiles lie on (see tree_attn.cu), at most: counted in 32 bits
constexpr int64_t tree_line_bound(int64_t rows, int64_t B, int64_t Hkv, int64_t group, int64_t max_tokens) {
  return (rows * group / 128 + B) * Hkv * (max_tokens / 128 + 4);
}

cudaError_t launch_tree_decode(const TreeDecodeParams& p, bool pdl, cudaStream_t stream);

}  // namespace helix
