// o_proj with 4-bit weights: a GEMM whose weights become tensor-core operands on the way.
//
// Bound by streaming the weights once for a few tokens (8192 x 8192: 33.5 MB, 5.1 us at the copy rate), by the tensor cores only beyond
// some hundred.  A CTA owns 128 rows (a slab, M of the MMA) and a run of columns; tokens are the MMA's N.
//   * Records of the packed weight arrive by bulk copy.  Eight warps turn nibbles into numbers: with 0x4300 in front (0x6400 for fp16) a
//     nibble is 128 + q (1024 + q), from which 128 + z is subtracted exactly; 16 bytes go into the swizzled A operand at a time.
//   * tcgen05 sums each group's products in fp32 from these exact integers, into one of a few accumulators in tensor memory.  The
//     same eight warps, a thread per row (and half of the tokens), fetch a finished group and add it, times its scale, to their sums in registers:
//     scales and zero points cost no rounding, which folding them into 16-bit weights would (half a step per weight).
//   * The CTAs of a cluster share out a slab's columns and send each other their sums through distributed shared memory, each finishing
//     a part of the rows: no scratch memory, no atomics, one launch, one order of summation.
// The same product on warp-level MMAs, weights in registers, took 13.4 us for 8 tokens (8192 x 8192) and 126 us for 100 (7168 x 8192): they
// cost ~16 cycles per 256 weights and 8 tokens.
#include "oproj_int4.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <tuple>

#include "helix_common.cuh"
#include "sm100.cuh"

namespace helix {
namespace {

using namespace sm100;

constexpr int kRows = 128;
constexpr int kWorkers = 8, kMmaWarp = 8, kThreads = 320;        // and a warp that loads
constexpr int kBlockBytes = kRows * 128;               // A operand of 64 columns
constexpr int kStages = 4;                             // records of 128 columns on their way
constexpr int kNibbles = 4096;                         // bytes of a block of 64 columns
constexpr int kMaxRecord = 2 * kNibbles + 4 * 384;     // 128 columns in groups of 32, with zero points
constexpr int kMaxCluster = 8;

template <int N>
struct Shape {
  static constexpr int ctas = N <= 64 ? 2 : 1;         // per SM
  static constexpr int slots = N <= 64 ? 3 : 4;        // operand blocks between dequantisation and MMA
  static constexpr int accs = 4;                       // accumulators in tensor memory
  static constexpr int cols = accs * N;
  static constexpr int x_bytes = N * 128;              // B operand of 64 columns
  static constexpr int ring = slots * (kBlockBytes + x_bytes) + kStages * kMaxRecord;
  static constexpr int row = N * 4 + 16;               // bytes between rows of sums that CTAs send each other
  static constexpr int smem = ring + 1024;
};

template <bool BF16>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  if (BF16) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
template <bool BF16>
__device__ __forceinline__ float widen(uint16_t x) {
  return BF16 ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
}
template <bool BF16>
__device__ __forceinline__ uint16_t narrow(float x) {
  return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
}
__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}

template <bool BF16, int N>
__global__ void __launch_bounds__(kThreads, Shape<N>::ctas) oproj_int4_kernel(const __grid_constant__ OprojInt4Params p) {
  using S = Shape<N>;
  constexpr int NH = N / 2;                            // tokens of a worker thread
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t w_full[kStages], w_free[kStages], a_full[S::slots], x_full[S::slots], a_free[S::slots], d_full[S::accs],
      d_free[S::accs], drain;
  __shared__ uint32_t tmem_slot;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const a_ring = smem;
  uint8_t* const x_ring = smem + S::slots * kBlockBytes;
  uint8_t* const w_ring = x_ring + S::slots * S::x_bytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cl = (int)gridDim.y, rank = (int)blockIdx.y, slab = (int)blockIdx.x;          // a cluster is a column of the grid
  const int records = (p.K + 127) / 128, r0 = (int)((int64_t)records * rank / cl), r1 = (int)((int64_t)records * (rank + 1) / cl);
  const int b0 = 2 * r0, blocks = min(2 * r1, p.K / 64) - b0;        // of 64 columns
  const int group = p.group, group_bytes = p.zeros ? 384 : 256;

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&w_full[i], 1);
      mbar_init(&w_free[i], kWorkers);
    }
    for (int i = 0; i < S::slots; ++i) {
      mbar_init(&a_full[i], kWorkers);
      mbar_init(&x_full[i], 1);
      mbar_init(&a_free[i], 1);
    }
    for (int i = 0; i < S::accs; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_free[i], kWorkers);
    }
    mbar_init(&drain, 1);
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&tmem_slot, S::cols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  const unsigned long long deadline = now_ns() + p.timeout_ns;
  bool ok = true;

  float acc[NH];
#pragma unroll
  for (int j = 0; j < NH; ++j) acc[j] = 0.f;
  if (warp < kWorkers) {
    // =========================== dequantisation, and the sums ===========================
    const int row = tid & (kRows - 1), half = tid >> 7;              // 32 of a block's columns; half of the tokens
    const uint32_t tq = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + half * NH;
    // both in registers: with two constants the compiler makes two instructions of (w & mask) | magic
    uint32_t mask, magic;
    asm volatile("mov.u32 %0, 0x000f000f;" : "=r"(mask));
    asm volatile("mov.u32 %0, %1;" : "=r"(magic) : "n"(BF16 ? 0x43004300 : 0x64006400));
    int n_done = 0;                                                  // groups added up so far
    float s_now[2] = {0.f, 0.f}, s_last[2];                          // scales of this block's groups and of the one before
    int ends_now = 0, ends_last;                                     // groups that end with the block
    auto add_groups = [&](int n, const float (&s)[2]) {
      for (int i = 0; i < n && ok; ++i, ++n_done) {
        const int d = n_done % S::accs;
        ok = __all_sync(0xffffffffu, mbar_wait(&d_full[d], (n_done / S::accs) & 1, deadline));
        if (!ok) break;
        tc_fence_after_sync();
        uint32_t v[NH];
        if constexpr (NH == 8) tmem_ld_x8(tq + d * N, v);
        else if constexpr (NH == 16) tmem_ld_32x32b_x16(tq + d * N, v);
        else if constexpr (NH == 32) tmem_ld_x32(tq + d * N, v);
        else {
          tmem_ld_x32(tq + d * N, *reinterpret_cast<uint32_t(*)[32]>(v));
          tmem_ld_x32(tq + d * N + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
        }
        tmem_ld_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&d_free[d]);
        const float sc = i == 0 ? s[0] : s[1];
#pragma unroll
        for (int j = 0; j < NH; ++j) acc[j] += sc * __uint_as_float(v[j]);
      }
    };
    for (int b = 0; b < blocks && ok; ++b) {
      const int rec = b >> 1, st = rec % kStages, sl = b % S::slots;
      const int in_record = min(2, blocks - 2 * rec) * 64, col = (b & 1) * 64;           // columns of the record; the block's first
      if ((b & 1) == 0) ok = __all_sync(0xffffffffu, mbar_wait(&w_full[st], (rec / kStages) & 1, deadline));
      if (ok && b >= S::slots) ok = __all_sync(0xffffffffu, mbar_wait(&a_free[sl], (b / S::slots - 1) & 1, deadline));
      if (!ok) break;
      const uint8_t* w = w_ring + st * kMaxRecord;
      const uint4 q = *reinterpret_cast<const uint4*>(w + (b & 1) * kNibbles + half * (kRows * 16) + row * 16);
      const uint8_t* scales = w + in_record * 64;
      const uint32_t z = p.zeros ? scales[in_record / group * 256 + (col + 32 * half) / group * kRows + row] : 8u;
      const uint32_t z2 = magic + (z & 0xfu) * 0x00010001u;          // 128 + z, twice
      s_last[0] = s_now[0], s_last[1] = s_now[1];
      ends_last = ends_now;
      ends_now = group == 32 ? 2 : group == 64 ? 1 : b & 1;
      s_now[0] = widen<BF16>(reinterpret_cast<const uint16_t*>(scales + col / group * 256)[row]);
      s_now[1] = group == 32 ? widen<BF16>(reinterpret_cast<const uint16_t*>(scales + (col / group + 1) * 256)[row]) : 0.f;
      const uint32_t words[4] = {q.x, q.y, q.z, q.w};
      uint8_t* a = a_ring + sl * kBlockBytes;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = sub2<BF16>(and_or(words[c] >> (4 * i), mask, magic), z2);
        *reinterpret_cast<uint4*>(a + swz128(row, 4 * half + c)) = make_uint4(v[0], v[1], v[2], v[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&a_full[sl]);
        if ((b & 1) == 1 || b + 1 == blocks) mbar_arrive(&w_free[st]);
      }
      add_groups(ends_last, s_last);
    }
    if (ok) add_groups(ends_now, s_now);
  } else if (warp == kMmaWarp) {
    // =========================== MMA issue ===========================
    constexpr uint32_t idesc = BF16 ? umma_idesc_bf16(kRows, N) : umma_idesc_bf16(kRows, N) & ~((1u << 7) | (1u << 10));
    const uint64_t d_a = umma_desc_k_sw128(smem_u32(a_ring)), d_x = umma_desc_k_sw128(smem_u32(x_ring));
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, deadline)) != 0; };
    uint32_t n_group = 0;
    for (int b_lane = 0; b_lane < blocks && ok; ++b_lane) {
      // the block number through a shuffle: what is computed from it is then known to be the same in all lanes
      const int b = __shfl_sync(0xffffffffu, b_lane, 0), sl = b % S::slots;
      ok = wait(&x_full[sl], (b / S::slots) & 1) && wait(&a_full[sl], (b / S::slots) & 1);
      for (int k0 = 0; k0 < 64 && ok; k0 += 32) {
        const uint32_t n = __shfl_sync(0xffffffffu, n_group, 0), d = n % S::accs;
        const bool first = (b * 64 + k0) % group == 0, last = (b * 64 + k0 + 32) % group == 0;
        if (first && n >= (uint32_t)S::accs) ok = wait(&d_free[d], (n / S::accs - 1) & 1);
        if (!ok) break;
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const uint32_t off = k0 * 2 + ks * 32;
            umma_bf16(tmem + d * N, d_a + ((sl * kBlockBytes + off) >> 4), d_x + ((sl * S::x_bytes + off) >> 4), idesc, !(first && ks == 0));
          }
          if (last) umma_commit(&d_full[d]);
          if (k0 == 32) umma_commit(&a_free[sl]);
        }
        __syncwarp();
        n_group += last;
      }
    }
    // the last commits have to arrive before this CTA leaves
    for (int b = max(0, blocks - S::slots); b < blocks && ok; ++b) ok = wait(&a_free[b % S::slots], (b / S::slots) & 1);
    if (!ok) {
      if (elect_one()) umma_commit(&drain);            // nothing of this CTA's may be in flight when it leaves
      mbar_wait(&drain, 0, now_ns() + 10000000ull);
    }
  } else {
    // =========================== loads ===========================
    const uint8_t* w = p.w + (int64_t)slab * (int64_t)((int64_t)p.K * 64 + p.K / group * group_bytes) + (int64_t)r0 * (128 * 64 + 128 / group * group_bytes);
    const int n_rec = r1 - r0;
    int w_at = 0, x_at = 0;
    auto load_w = [&]() {
      const int st = w_at % kStages, cols = min(2, blocks - 2 * w_at) * 64;
      if (w_at >= kStages) ok = __all_sync(0xffffffffu, mbar_wait(&w_free[st], (w_at / kStages - 1) & 1, deadline));
      if (!ok) return;
      const uint32_t bytes = cols * 64 + cols / group * group_bytes;
      if (lane == 0) {
        mbar_expect_tx(&w_full[st], bytes);
        bulk_load_1d(w_ring + st * kMaxRecord, w + (int64_t)w_at * (128 * 64 + 128 / group * group_bytes), bytes, &w_full[st]);
      }
      __syncwarp();
      ++w_at;
    };
    while (w_at < min(n_rec, kStages) && ok) load_w();               // weights do not depend on the kernel before this one
    asm volatile("griddepcontrol.wait;" ::: "memory");
    while (x_at < blocks && ok) {
      const int sl = x_at % S::slots;
      if (x_at >= S::slots) ok = __all_sync(0xffffffffu, mbar_wait(&a_free[sl], (x_at / S::slots - 1) & 1, deadline));
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(&x_full[sl], S::x_bytes);
        tma_load_2d(x_ring + sl * S::x_bytes, &p.x_map, &x_full[sl], (b0 + x_at) * 64, 0);
      }
      __syncwarp();
      ++x_at;
      // a record's place is free when its last block has been dequantised, long before that block's x is used
      if ((x_at & 1) == 0 && w_at < n_rec) load_w();
    }
    while (w_at < n_rec && ok) load_w();
    if (!ok) {
      // nothing may land in this CTA's shared memory after it has left
      const unsigned long long limit = now_ns() + 10000000ull;
      for (int i = max(0, w_at - kStages); i < w_at; ++i) mbar_wait(&w_full[i % kStages], (i / kStages) & 1, limit);
      for (int i = max(0, x_at - S::slots); i < x_at; ++i) mbar_wait(&x_full[i % S::slots], (i / S::slots) & 1, limit);
    }
  }
  if (!ok && lane == 0) atomicCAS(p.error_flag, 0, (int)kTimeoutMbarrier);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, S::cols);
  }

  // ---- results: thread (row, half) holds tokens half * NH ... of its row ----------------------------------
  const int row = tid & (kRows - 1), half = tid >> 7;
  const int rows_here = min(kRows, p.hidden - slab * kRows);
  if (cl == 1) {
    if (warp < kWorkers && row < rows_here) {
#pragma unroll
      for (int j = 0; j < NH; ++j) {
        const int n = half * NH + j;
        if (n < p.tokens) p.y[n * p.y_stride + slab * kRows + row] = narrow<BF16>(acc[j]);
      }
    }
    return;
  }
  // Rank r finishes rows r * per ... of the slab.  Everybody is through with its rings, so they take the others' sums.
  const int per = (kRows / 8 + cl - 1) / cl * 8;
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (warp < kWorkers) {
    const uint32_t to = map_to_cta(smem_u32(smem) + (rank * per + row % per) * S::row + half * NH * 4, row / per);
#pragma unroll
    for (int j = 0; j < NH; j += 4) st_cluster_f32x4(to + j * 4, acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  const int mine = max(min(per, rows_here - rank * per), 0);
  for (int e = tid; e < per * p.tokens; e += kThreads) {
    const int n = e / per, r = e % per;
    if (r >= mine) continue;
    const uint8_t* from = smem + r * S::row + n * 4;
    float v = *reinterpret_cast<const float*>(from);
    for (int c = 1; c < cl; ++c) v += *reinterpret_cast<const float*>(from + c * per * S::row);
    p.y[n * p.y_stride + slab * kRows + rank * per + r] = narrow<BF16>(v);
  }
}

using Fn = void (*)(OprojInt4Params);
template <bool BF16>
Fn pick(int n, size_t* smem) {
  if (n == 16) return *smem = Shape<16>::smem, (Fn)oproj_int4_kernel<BF16, 16>;
  if (n == 32) return *smem = Shape<32>::smem, (Fn)oproj_int4_kernel<BF16, 32>;
  if (n == 64) return *smem = Shape<64>::smem, (Fn)oproj_int4_kernel<BF16, 64>;
  return *smem = Shape<128>::smem, (Fn)oproj_int4_kernel<BF16, 128>;
}

cudaLaunchConfig_t config(int slabs, int cl, size_t smem, bool pdl, cudaStream_t stream, cudaLaunchAttribute (&attrs)[2]) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)slabs, (unsigned)cl, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = 1;
  attrs[0].val.clusterDim.y = (unsigned)cl;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = pdl ? 2 : 1;
  return cfg;
}

// Clusters of each size that are resident together, asked once per kernel and device
struct Resident {
  int clusters[kMaxCluster + 1];
};
cudaError_t resident(const void* fn, int dev, size_t smem, int sm_count, Resident* out) {
  static std::mutex mu;
  static std::map<std::tuple<int, const void*>, Resident> known;
  std::lock_guard<std::mutex> lk(mu);
  const auto key = std::make_tuple(dev, fn);
  const auto it = known.find(key);
  if (it != known.end()) {
    *out = it->second;
    return cudaSuccess;
  }
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  Resident r{};
  for (int cl = 1; cl <= kMaxCluster; ++cl) {
    cudaLaunchAttribute attrs[2];
    const cudaLaunchConfig_t cfg = config(sm_count, cl, smem, false, nullptr, attrs);
    e = cudaOccupancyMaxActiveClusters(&r.clusters[cl], fn, &cfg);
    if (e != cudaSuccess) return e;
  }
  known[key] = r;
  *out = r;
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_oproj_int4(const OprojInt4Params& p, bool pdl, int sm_count, cudaStream_t stream) {
  if (p.tokens <= 0 || p.hidden <= 0) return cudaSuccess;
  if (p.tokens > kInt4MaxTokens || p.K <= 0 || p.K % 64 != 0 || (p.group != 32 && p.group != 64 && p.group != 128) || p.K % p.group != 0)
    return cudaErrorInvalidValue;
  size_t smem = 0;
  const int n = int4_pad_tokens(p.tokens);
  const Fn fn = p.is_bf16 ? pick<true>(n, &smem) : pick<false>(n, &smem);
  int dev = 0;
  cudaGetDevice(&dev);
  Resident r;
  cudaError_t e = resident((const void*)fn, dev, smem, sm_count, &r);
  if (e != cudaSuccess) return e;
  // As many CTAs per slab as make the launch shortest: rounds of resident clusters times the records of a CTA, and about three records'
  // time for a CTA's start, the exchange and the end.
  const int slabs = (p.hidden + kRows - 1) / kRows, records = (p.K + 127) / 128;
  int best = 1;
  int64_t cost = INT64_MAX;
  for (int cl = 1; cl <= std::min(kMaxCluster, records); ++cl) {
    if (r.clusters[cl] < 1) continue;
    const int64_t c = (int64_t)((slabs + r.clusters[cl] - 1) / r.clusters[cl]) * ((records + cl - 1) / cl + 3);
    if (c < cost) {
      cost = c;
      best = cl;
    }
  }
  cudaLaunchAttribute attrs[2];
  const cudaLaunchConfig_t cfg = config(slabs, best, smem, pdl, stream, attrs);
  return cudaLaunchKernelEx(&cfg, fn, p);
}

}  // namespace helix
