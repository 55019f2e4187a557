// Paged cache bookkeeping and writes: host interface (kernels in paged.cu).
//
// The reference leaves both to vLLM's block manager and attention backends
// (benchmark/sbatch/run_gb200_aiperf_v3.sbatch:95); here they are what feeds the decode attention.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace helix {

constexpr int kTableMaxSeqs = 8192;     // sequences of one call: their pages are numbered in shared memory
constexpr int kTableMaxWords = 4;       // mask words per row: 256 drafted tokens of one sequence on one rank

struct ExtendTablesParams {
  int32_t* block_table;        // [B, max_pages], rows bt_stride apart; pages taken in this call are entered
  int64_t bt_stride;
  int32_t* held;               // [B] pages that a sequence holds, updated
  const int32_t* free_pages;   // [n_free]
  int32_t* free_used;          // [1] how many of them are taken, updated
  const int32_t* ctx_lens;     // [B] committed tokens over all ranks
  const int32_t* q_start;      // [B + 1] first row of each sequence's new tokens
  const int32_t* parents;      // [rows] parent inside the sequence or -1 (null: every token follows the one before)
  int64_t* slots;              // [rows]
  int32_t* positions;          // [rows]
  int32_t* seq_lens;           // [B] tokens this rank holds, the new ones among them
  int32_t* draft_lens;         // [B] new ones of these
  int32_t* missing;            // [1] pages that were not to be had
  uint64_t* mask;              // [rows, words]
  int B, rows, max_pages, n_free, words, page_size, cp_size, cp_rank, interleave;
};
cudaError_t launch_extend_tables(const ExtendTablesParams& p, bool pdl, cudaStream_t stream);

struct AppendKvParams {
  const uint8_t* k;            // row r, head h at k + r * k_sr + h * k_sh (bytes), head_bytes contiguous
  const uint8_t* v;
  uint8_t* kc;                 // token t of page g, head h at kc + g * c_sp + t * c_st + h * c_sh (bytes)
  uint8_t* vc;
  const int64_t* slots;        // [rows] page * page_size + token, or negative: not on this rank
  int64_t k_sr, k_sh, v_sr, v_sh, kc_sp, kc_st, kc_sh, vc_sp, vc_st, vc_sh;
  int64_t n_slots;             // pages * page_size
  int rows, heads, head_bytes, page_size;
};
cudaError_t launch_append_kv(const AppendKvParams& p, bool pdl, cudaStream_t stream);

}  // namespace helix
