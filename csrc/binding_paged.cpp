// Torch bindings of the paged cache's bookkeeping and writes.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cstdlib>
#include <string>
#include <tuple>

#include "paged.h"

namespace {

bool env_pdl() {
  const char* v = std::getenv("HELIX_A2A_ENABLE_PDL");
  return v && std::string(v) == "1";
}

void check_cuda(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, "helix: ", what, " failed: ", cudaGetErrorString(e));
}

void check_ints(const torch::Tensor& t, const char* name, const torch::Device& dev, int64_t numel) {
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev);
  TORCH_CHECK(t.scalar_type() == at::ScalarType::Int && t.dim() == 1 && t.is_contiguous(), name, " must be a contiguous 1-D int32 tensor");
  TORCH_CHECK(numel < 0 || t.size(0) == numel, name, " must have ", numel, " elements");
}

using Tables = std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>;

Tables extend_tables(torch::Tensor block_table, torch::Tensor held, torch::Tensor free_pages, torch::Tensor free_used,
                     torch::Tensor ctx_lens, torch::Tensor q_start, const c10::optional<torch::Tensor>& parents, int64_t rows,
                     int64_t page_size, int64_t words, int64_t cp_size, int64_t cp_rank, int64_t interleave) {
  TORCH_CHECK(block_table.is_cuda(), "all inputs must be on CUDA");
  const torch::Device dev = block_table.device();
  TORCH_CHECK(block_table.scalar_type() == at::ScalarType::Int && block_table.dim() == 2 && (block_table.numel() == 0 || block_table.size(1) == 1 || block_table.stride(1) == 1) &&
                  (block_table.size(0) <= 1 || block_table.stride(0) >= block_table.size(1)),
              "block_table must be int32 [B, max_pages] with the pages of a sequence side by side");
  const int64_t B = block_table.size(0);
  TORCH_CHECK(B <= helix::kTableMaxSeqs, "at most ", helix::kTableMaxSeqs, " sequences");
  check_ints(held, "held", dev, B);
  check_ints(ctx_lens, "ctx_lens", dev, B);
  check_ints(q_start, "q_start", dev, B + 1);
  check_ints(free_pages, "free_pages", dev, -1);
  check_ints(free_used, "free_used", dev, 1);
  constexpr int64_t kMax = 0x7fffffff;
  TORCH_CHECK(rows >= 0 && rows <= kMax / 2 && block_table.size(1) <= kMax && free_pages.size(0) <= kMax, "rows, max_pages and free pages are counted in 32 bits");
  if (parents) check_ints(*parents, "parents", dev, rows);
  TORCH_CHECK(!parents || rows <= (1 << 20), "trees have at most 2^20 rows");
  TORCH_CHECK(words >= 0 && words <= helix::kTableMaxWords, "mask_words must be 0 to ", helix::kTableMaxWords);
  TORCH_CHECK(page_size >= 1 && page_size <= (1 << 20), "page_size must be positive");
  TORCH_CHECK(cp_size >= 1 && cp_rank >= 0 && cp_rank < cp_size, "cp_rank must be in [0, cp_size)");
  constexpr int64_t kCycle = 1 << 28;
  TORCH_CHECK(interleave >= 1 && interleave <= kCycle && cp_size <= kCycle && interleave * cp_size <= kCycle,
              "interleave must be positive and interleave * cp_size at most 2^28");
  c10::cuda::CUDAGuard guard(dev);
  const auto i32 = [&](int64_t n) { return torch::Tensor(at::detail::empty_cuda({n}, at::kInt, dev, c10::nullopt)); };
  const auto i64 = [&](at::IntArrayRef n) { return torch::Tensor(at::detail::empty_cuda(n, at::kLong, dev, c10::nullopt)); };
  torch::Tensor slots = i64({rows}), mask = i64({rows, words}), positions = i32(rows), seq_lens = i32(B), draft_lens = i32(B), missing = i32(1);
  helix::ExtendTablesParams p{};
  p.block_table = block_table.data_ptr<int32_t>();
  p.bt_stride = block_table.stride(0);
  p.held = held.data_ptr<int32_t>();
  p.free_pages = free_pages.data_ptr<int32_t>();
  p.free_used = free_used.data_ptr<int32_t>();
  p.ctx_lens = ctx_lens.data_ptr<int32_t>();
  p.q_start = q_start.data_ptr<int32_t>();
  p.parents = parents ? parents->data_ptr<int32_t>() : nullptr;
  p.slots = slots.data_ptr<int64_t>();
  p.positions = positions.data_ptr<int32_t>();
  p.seq_lens = seq_lens.data_ptr<int32_t>();
  p.draft_lens = draft_lens.data_ptr<int32_t>();
  p.missing = missing.data_ptr<int32_t>();
  p.mask = reinterpret_cast<uint64_t*>(mask.data_ptr<int64_t>());
  p.B = (int)B; p.rows = (int)rows; p.max_pages = (int)block_table.size(1); p.n_free = (int)free_pages.size(0);
  p.words = (int)words; p.page_size = (int)page_size;
  p.cp_size = (int)cp_size; p.cp_rank = (int)cp_rank; p.interleave = (int)interleave;
  check_cuda(helix::launch_extend_tables(p, env_pdl(), at::cuda::getCurrentCUDAStream()), "extend tables launch");
  return {slots, positions, seq_lens, draft_lens, mask, missing};
}

void append_kv(torch::Tensor k, torch::Tensor v, torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor slots, bool hnd) {
  TORCH_CHECK(k.is_cuda(), "all inputs must be on CUDA");
  const torch::Device dev = k.device();
  TORCH_CHECK(v.device() == dev && k_cache.device() == dev && v_cache.device() == dev && slots.device() == dev,
              "k, v, the caches and slots must be on one device");
  TORCH_CHECK(k.dim() == 3 && v.sizes() == k.sizes(), "k and v must be [rows, kv heads, head_dim]");
  TORCH_CHECK(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes(), "the caches must be 4-D and alike");
  const auto type = k.scalar_type();
  TORCH_CHECK(v.scalar_type() == type && k_cache.scalar_type() == type && v_cache.scalar_type() == type,
              "k, v and the caches must have one type");
  const int64_t rows = k.size(0), heads = k.size(1), D = k.size(2), es = k.element_size();
  const int hd = hnd ? 1 : 2, td = hnd ? 2 : 1;
  TORCH_CHECK(k_cache.size(hd) == heads && k_cache.size(3) == D, "the caches must have the rows' kv heads and head_dim");
  TORCH_CHECK(slots.scalar_type() == at::ScalarType::Long && slots.dim() == 1 && slots.is_contiguous() && slots.size(0) == rows,
              "slots must be a contiguous int64 [rows]");
  TORCH_CHECK(rows <= 0x3fffffff, "at most 2^30 - 1 rows");
  if (k.numel() == 0 || k_cache.numel() == 0) return;
  TORCH_CHECK(D * es % 16 == 0, "a head's row must be a multiple of 16 bytes");
  for (const torch::Tensor* t : {&k, &v, &k_cache, &v_cache}) {
    TORCH_CHECK(t->stride(-1) == 1, "head_dim must be innermost and contiguous");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "k, v and the caches must start on a 16-byte boundary");
    for (int i = 0; i + 1 < t->dim(); ++i)
      TORCH_CHECK(t->stride(i) * es % 16 == 0 || t->size(i) <= 1, "strides must be multiples of 16 bytes");
  }
  c10::cuda::CUDAGuard guard(dev);
  helix::AppendKvParams p{};
  p.k = reinterpret_cast<const uint8_t*>(k.data_ptr());
  p.v = reinterpret_cast<const uint8_t*>(v.data_ptr());
  p.kc = reinterpret_cast<uint8_t*>(k_cache.data_ptr());
  p.vc = reinterpret_cast<uint8_t*>(v_cache.data_ptr());
  p.slots = slots.data_ptr<int64_t>();
  p.k_sr = k.stride(0) * es; p.k_sh = k.stride(1) * es;
  p.v_sr = v.stride(0) * es; p.v_sh = v.stride(1) * es;
  p.kc_sp = k_cache.stride(0) * es; p.kc_sh = k_cache.stride(hd) * es; p.kc_st = k_cache.stride(td) * es;
  p.vc_sp = v_cache.stride(0) * es; p.vc_sh = v_cache.stride(hd) * es; p.vc_st = v_cache.stride(td) * es;
  p.rows = (int)rows; p.heads = (int)heads; p.head_bytes = (int)(D * es); p.page_size = (int)k_cache.size(td);
  p.n_slots = k_cache.size(0) * k_cache.size(td);
  check_cuda(helix::launch_append_kv(p, env_pdl(), at::cuda::getCurrentCUDAStream()), "append kv launch");
}

}  // namespace

void register_paged_ops(torch::Library& m) {
  m.def(
      "extend_tables(Tensor(a!) block_table, Tensor(b!) held, Tensor free_pages, Tensor(c!) free_used, Tensor ctx_lens, Tensor "
      "q_start, Tensor? parents, int rows, int page_size, int mask_words, int cp_size, int cp_rank, int interleave) -> (Tensor, "
      "Tensor, Tensor, Tensor, Tensor, Tensor)",
      &extend_tables);
  m.def("append_kv(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, bool hnd) -> ()", &append_kv);
}
