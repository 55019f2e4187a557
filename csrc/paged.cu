// Block tables, slots and tree masks of a step's new tokens, and the tokens' way into the paged cache.
//
// extend_tables: rank r of N holds the tokens p of a sequence with (p / I) % N == r, in order, so of the first n tokens
//
//   L(n) = n / (I N) * I + clamp(n % (I N) - r I, 0, I)
//
// A sequence that grows from n0 to n1 tokens needs ceil(L(n1) / page) pages; what it does not hold yet it takes from the free
// list, sequence after sequence, i.e. from where a prefix sum over the sequences says.  The new token at position p is local
// token L(p) and goes to slot table[L(p) / page] * page + L(p) % page.  Its mask holds a bit for each new local token on its
// way to the root of the tree, itself included.
//
// A step's call is a few kilobytes, so what bounds it is the launch and a handful of dependent loads (prompts: 61000 rows are 0.8 MB, and a
// search and several divisions each, 10.0 us in a graph).  One cluster of up to
// sixteen CTAs does it in one launch and without scratch memory: every CTA numbers all sequences for itself (three loads
// per sequence), and a cluster barrier stands between everybody's reading of `held` and `free_used` and their update.
#include "paged.h"

#include <algorithm>
#include <atomic>

#include "helix_common.cuh"
#include "sm100.cuh"

namespace helix {
namespace {

using namespace sm100;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kPortable = 8, kMaxCtas = 16;      // CTAs of a cluster: on every GPU, and where a group of SMs is that large
constexpr int kStagedNodes = 64 * kTableMaxWords;

// What a CTA knows of every sequence, in shared memory.
struct Seq {
  int ctx, row0, rows;     // committed tokens, first row and number of the new ones
  int held, first, got;    // pages held before, first entry of the free list that is taken, how many are
};

// tokens that n pages hold, as far as 32 bits count
__device__ __forceinline__ int tokens_of(const ExtendTablesParams& p, int pages) {
  return (int)min((long long)pages * p.page_size, 0x7fffffffll);
}

struct Split {                                   // the ranks' shares of a sequence
  int il, cycle, skip;
  __device__ __forceinline__ int local(int n) const { return n / cycle * il + min(max(n % cycle - skip, 0), il); }
  __device__ __forceinline__ bool mine(int n) const { return (unsigned)(n % cycle - skip) < (unsigned)il; }
};

__global__ void __launch_bounds__(kThreads) extend_tables_kernel(const __grid_constant__ ExtendTablesParams p) {
  extern __shared__ Seq s_seq[];
  __shared__ long long s_warp[kWarps], s_want[kWarps];
  __shared__ int s_parent[kWarps][kStagedNodes];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ctas = gridDim.x, cta = blockIdx.x;
  const Split split{p.interleave, p.interleave * p.cp_size, p.interleave * p.cp_rank};
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- all sequences: lengths, and the prefix sum of the pages they take ---------------------------------
  const int used = max(__ldcg(p.free_used), 0);
  int base = 0;                                  // taken by the sequences before this round of kThreads
  long long short_of = 0;                        // (what all ask for together may take more than 32 bits)
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + tid;
    Seq s{0, 0, 0, 0, 0, 0};
    int want = 0, lack = 0;
    if (b < p.B) {
      s.ctx = max(__ldg(p.ctx_lens + b), 0);
      s.row0 = min(max(__ldg(p.q_start + b), 0), p.rows);
      s.rows = max(min(__ldg(p.q_start + b + 1), p.rows) - s.row0, 0);
      s.ctx = min(s.ctx, 0x7fffffff - s.rows);
      s.held = min(max(__ldcg(p.held + b), 0), p.max_pages);
      const int need = (int)(((unsigned)split.local(s.ctx + s.rows) + p.page_size - 1) / (unsigned)p.page_size);
      want = max(min(need, p.max_pages) - s.held, 0);
      lack = max(need - p.max_pages, 0);
    }
    long long before = want;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    if (lane == 31) s_warp[warp] = before;
    __syncthreads();
    long long all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) before += all;
      all += s_warp[w];
    }
    const long long first = (long long)min(used, p.n_free) + base + before - want;
    s.first = (int)min(first, (long long)p.n_free);
    s.got = min(want, p.n_free - s.first);
    short_of += (long long)want - s.got + lack;
    if (b < p.B) s_seq[b] = s;
    base = (int)min(base + all, (long long)p.n_free);      // nothing is left behind that point
    __syncthreads();
  }
  for (int o = 16; o > 0; o >>= 1) short_of += __shfl_xor_sync(0xffffffffu, short_of, o);
  if (lane == 0) s_want[warp] = short_of;
  __syncthreads();
  if (ctas > 1) cluster_arrive();                // this CTA has read held and free_used

  // ---- rows -------------------------------------------------------------------------------------------------
  const int last = p.B > 0 ? s_seq[p.B - 1].row0 + s_seq[p.B - 1].rows : 0;
  auto place = [&](const Seq& s, int b, int row, int pos) {
    int64_t slot = -1;
    if (split.mine(pos)) {
      const int at = split.local(pos), page = at / p.page_size;
      if (page < s.held + s.got) {
        const int id = page < s.held ? __ldcg(p.block_table + b * p.bt_stride + page) : __ldg(p.free_pages + s.first + page - s.held);
        slot = (int64_t)id * p.page_size + at % p.page_size;
      }
    }
    p.slots[row] = slot;
  };
  if (p.parents == nullptr) {
    // every token follows the one before it: rows one by one, the mask of a row is a run of ones
    for (int row = cta * kThreads + tid; row < p.rows; row += ctas * kThreads) {
      int lo = 0, hi = p.B;                      // the last sequence that starts at or before this row (empty ones share a start)
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (s_seq[mid].row0 <= row) lo = mid; else hi = mid;
      }
      if (p.B == 0 || row < s_seq[lo].row0 || row - s_seq[lo].row0 >= s_seq[lo].rows) {
        p.slots[row] = -1;
        p.positions[row] = 0;
        for (int w = 0; w < p.words; ++w) p.mask[(int64_t)row * p.words + w] = 0;
        continue;
      }
      const Seq s = s_seq[lo];
      const int pos = s.ctx + row - s.row0;
      place(s, lo, row, pos);
      p.positions[row] = pos;
      const int seen = min(split.local(pos + 1), tokens_of(p, s.held + s.got)) - split.local(s.ctx);
      for (int w = 0; w < p.words; ++w) {
        const int n = min(max(seen - 64 * w, 0), 64);
        p.mask[(int64_t)row * p.words + w] = n == 64 ? ~0ull : (1ull << n) - 1;
      }
    }
  } else {
    // trees: a warp per sequence, its parents in shared memory, every lane walks up from its node
    for (int b = cta * kWarps + warp; b < p.B; b += ctas * kWarps) {
      const Seq s = s_seq[b];
      __syncwarp();
      for (int j = lane; j < min(s.rows, kStagedNodes); j += 32) s_parent[warp][j] = __ldg(p.parents + s.row0 + j);
      __syncwarp();
      const int base_local = split.local(s.ctx), room = tokens_of(p, s.held + s.got);
      for (int j0 = 0; j0 < s.rows; j0 += 32) {
        const int j = min(j0 + lane, s.rows - 1);         // (lanes behind the end repeat the last node)
        uint64_t words[kTableMaxWords] = {0, 0, 0, 0};
        int depth = 0;
        for (int up = j;;) {
          if (up < j0 && j0 >= kStagedNodes) {            // a far walk goes on where this warp has been: at most 32 steps
            const int64_t row = s.row0 + up;
            depth += __ldcg(p.positions + row) - s.ctx;
#pragma unroll
            for (int w = 0; w < kTableMaxWords; ++w)
              if (w < p.words) words[w] |= __ldcg(reinterpret_cast<const unsigned long long*>(p.mask) + row * p.words + w);
            break;
          }
          const int pos = s.ctx + up;
          const int at = split.local(pos), bit = at - base_local;
          if (split.mine(pos) && at < room) {
#pragma unroll
            for (int w = 0; w < kTableMaxWords; ++w)
              if ((bit >> 6) == w) words[w] |= 1ull << (bit & 63);
          }
          const int parent = up < kStagedNodes ? s_parent[warp][up] : __ldg(p.parents + s.row0 + up);
          if (parent < 0 || parent >= up) break;          // a parent comes before its children: every walk ends
          up = parent;
          ++depth;
        }
        const int row = s.row0 + j;
        place(s, b, row, s.ctx + j);
        p.positions[row] = s.ctx + depth;
        for (int w = 0; w < p.words; ++w) p.mask[(int64_t)row * p.words + w] = words[w];
        __syncwarp();
      }
    }
    const int first = p.B > 0 ? s_seq[0].row0 : p.rows;
    for (int row = cta * kThreads + tid; row < p.rows; row += ctas * kThreads)
      if (row >= last || row < first) {
        p.slots[row] = -1;
        p.positions[row] = 0;
        for (int w = 0; w < p.words; ++w) p.mask[(int64_t)row * p.words + w] = 0;
      }
  }

  // ---- state: the pages that were taken, after everybody has read what was there before -----------------
  __syncwarp();
  if (ctas > 1) cluster_wait();
  for (int b = cta * kWarps + warp; b < p.B; b += ctas * kWarps) {
    const Seq s = s_seq[b];
    for (int i = lane; i < s.got; i += 32) p.block_table[b * p.bt_stride + s.held + i] = __ldg(p.free_pages + s.first + i);
    if (lane == 0) {
      const int len = min(split.local(s.ctx + s.rows), tokens_of(p, s.held + s.got));
      p.held[b] = s.held + s.got;
      p.seq_lens[b] = len;
      p.draft_lens[b] = max(len - split.local(s.ctx), 0);
    }
  }
  if (cta == 0 && tid == 0) {
    p.free_used[0] = (int)min((long long)min(used, p.n_free) + base, (long long)p.n_free);
    long long n = 0;
    for (int w = 0; w < kWarps; ++w) n += s_want[w];
    p.missing[0] = (int)min(n, 0x7fffffffll);
  }
}

// ---- rows into the cache ----------------------------------------------------------------------------------
// A row's K and V are 2 * heads * head_bytes / 16 chunks; threadIdx.x is the chunk, so what depends on it is worked out once,
// and a thread has kRowsAhead rows on their way at a time.
constexpr int kAppendThreads = 256, kRowsAhead = 4;

__global__ void __launch_bounds__(kAppendThreads) append_kv_kernel(const __grid_constant__ AppendKvParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int per_head = p.head_bytes / 16, per_row = 2 * p.heads * per_head;
  const int step = gridDim.x * blockDim.y;
  for (int c = threadIdx.x; c < per_row; c += blockDim.x) {
    const bool is_v = c >= per_row / 2;
    const int hc = is_v ? c - per_row / 2 : c, head = hc / per_head, off = (hc - head * per_head) * 16;
    const uint8_t* src = is_v ? p.v + head * p.v_sh + off : p.k + head * p.k_sh + off;
    uint8_t* dst = is_v ? p.vc + head * p.vc_sh + off : p.kc + head * p.kc_sh + off;
    const int64_t sr = is_v ? p.v_sr : p.k_sr, sp = is_v ? p.vc_sp : p.kc_sp, st = is_v ? p.vc_st : p.kc_st;
    for (int r0 = blockIdx.x * blockDim.y + threadIdx.y; r0 < p.rows; r0 += kRowsAhead * step) {
      int64_t slot[kRowsAhead];
      uint4 x[kRowsAhead];
#pragma unroll
      for (int i = 0; i < kRowsAhead; ++i) {
        const int64_t r = (int64_t)r0 + (int64_t)i * step;
        slot[i] = r < p.rows ? __ldg(p.slots + r) : -1;
      }
#pragma unroll
      for (int i = 0; i < kRowsAhead; ++i)
        if (slot[i] >= 0 && slot[i] < p.n_slots) x[i] = __ldg(reinterpret_cast<const uint4*>(src + ((int64_t)r0 + (int64_t)i * step) * sr));
#pragma unroll
      for (int i = 0; i < kRowsAhead; ++i)
        if (slot[i] >= 0 && slot[i] < p.n_slots) {
          // (64-bit divisions are some 100 instructions, which only slots behind 2^32 need)
          const int64_t page = slot[i] >> 32 ? slot[i] / p.page_size : (uint32_t)slot[i] / (uint32_t)p.page_size;
          *reinterpret_cast<uint4*>(dst + page * sp + (slot[i] - page * p.page_size) * st) = x[i];
        }
    }
  }
}

cudaLaunchConfig_t config(dim3 grid, dim3 block, size_t smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  return cfg;
}

}  // namespace

cudaError_t launch_extend_tables(const ExtendTablesParams& p, bool pdl, cudaStream_t stream) {
  if (p.B < 0 || p.B > kTableMaxSeqs || p.words < 0 || p.words > kTableMaxWords || p.rows < 0) return cudaErrorInvalidValue;
  static std::atomic<int> largest[64];             // cluster; 0: not asked yet
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (largest[dev] == 0) {
    cudaError_t e = cudaFuncSetAttribute(extend_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTableMaxSeqs * (int)sizeof(Seq));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(extend_tables_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    int there = 0;
    if (e == cudaSuccess) {
      cudaLaunchAttribute attr;
      cudaLaunchConfig_t cfg = config(dim3(kMaxCtas), dim3(kThreads), kTableMaxSeqs * sizeof(Seq), stream);
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = kMaxCtas;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&there, extend_tables_kernel, &cfg);
    }
    if (e != cudaSuccess) return e;
    largest[dev] = there > 0 ? kMaxCtas : kPortable;
  }
  // A row per thread, or a sequence per warp: one CTA for small calls, a cluster for large ones.  64 prompts, 61000 tokens, in a graph: 10.0 us
  // with 16 CTAs, 17.2 with 8; 256 trees 6.2 and 9.5.
  const int64_t work = p.parents ? ((int64_t)p.B + kWarps - 1) / kWarps : ((int64_t)p.rows + kThreads - 1) / kThreads;
  const int ctas = work > kPortable ? largest[dev].load() : (int)std::max<int64_t>(work, 1);
  cudaLaunchConfig_t cfg = config(dim3(ctas), dim3(kThreads), (size_t)std::max(p.B, 1) * sizeof(Seq), stream);
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = ctas;
  attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, extend_tables_kernel, p);
}

cudaError_t launch_append_kv(const AppendKvParams& p, bool pdl, cudaStream_t stream) {
  if (p.rows <= 0 || p.heads <= 0) return cudaSuccess;
  if (p.head_bytes <= 0 || p.head_bytes % 16 != 0 || p.page_size <= 0) return cudaErrorInvalidValue;
  const int per_row = 2 * p.heads * (p.head_bytes / 16);
  const int x = std::min((per_row + 31) / 32 * 32, kAppendThreads), y = std::max(kAppendThreads / x, 1);
  const int64_t blocks = std::min<int64_t>(((int64_t)p.rows + y - 1) / y, 148 * 8);
  cudaLaunchConfig_t cfg = config(dim3((unsigned)blocks), dim3(x, y), 0, stream);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, append_kv_kernel, p);
}

}  // namespace helix
