// o_proj with 4-bit weights, in two forms over one packed layout.
//
// Bound by streaming the weights once for a few tokens (8192 x 8192: 33.5 MB, 5.1 us at the copy rate), by the tensor cores only beyond
// some hundred.  In both forms a nibble becomes a number with 0x4300 in front (0x6400 for fp16): 128 + q (1024 + q), from which 128 + z is
// subtracted exactly; a group's products are summed in fp32 from these exact integers, and only their sum is multiplied by the scale, in
// fp32.  So scales and zero points cost no rounding, which folding them into 16-bit weights would (half a step per weight).
//
// Up to 16 tokens (oproj_int4_few_kernel) the weights go through registers into the warp-level MMA: a warp owns 256 columns, whose x it
// holds as B operands for the whole launch, and walks over 16-row tiles, the next tile's weights on their way.
//
// More tokens (oproj_int4_kernel) run on tcgen05.  A CTA owns a slab of 128 rows (M of the MMA; tokens are N) and a run of columns.
// It works in rounds of 256 columns, two records of the packed weight, because what a round takes is mostly chains of waits (a barrier that
// is ready costs 100 to 200 cycles) and latencies, and every role below is one:
//   * A warp brings the records by bulk copy, one x.  Eight warps turn nibbles into numbers and put them into tensor memory as the MMA's A
//     operand, a thread per row and 64 columns of a record.  (In shared memory a record is 32 KB written and 32 KB read for 8 KB that arrived.)
//   * A warp issues the MMAs.  Every group has an accumulator of its own in tensor memory, a ring of them.
//   * Further warps add each group, times its scale, to their sums in registers: a thread per row and 32 tokens, 64 with more than 64 (of
//     32 tokens each, 16 warps took issue slots from the others: 100 tokens 32.2 us).
// 8192 x 8192 in groups of 128, bf16, in a graph: 32 tokens 21.6 us, 64 tokens 23.7, 100 tokens 27.5.  Before, with teams of warps that did
// both jobs record by record: 24.7, 28.0, 39.0.  A round takes ~1900 cycles with 32 tokens and ~2900 with 128, of which the tensor cores work
// ~700 and ~1100; with 128 tokens and groups of 64 the two accumulators that fit are handed to and fro every 64 columns, ~900 cycles each.
//
// In both the warps or CTAs that share out the columns meet in shared memory, across a cluster by distributed shared memory: no scratch
// memory, no atomics, one launch, one order of summation.
#include "oproj_int4.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <tuple>
#include <type_traits>

#include "helix_common.cuh"
#include "sm100.cuh"

namespace helix {
namespace {

using namespace sm100;

constexpr int kRows = 128;
constexpr int kTeam = 8;                               // warps that dequantise, a row and 64 columns of a record per thread
constexpr int kOperand = 128;                          // columns of tensor memory of a round's A operand
constexpr int kNibbles = 4096;                         // packed bytes of 64 columns
constexpr int kMaxRecord = 2 * kNibbles + 4 * 384;     // 128 columns in groups of 32, with zero points
constexpr int kMaxCluster = 8;
constexpr int kFewWarps = 16;
constexpr int kRow = 20;                               // floats between tokens of a tile's sums: 16 rows, and no bank conflicts
constexpr int kFewSmem = 200 * 1024;

template <int N>
struct Shape {
  static constexpr int tokens = N == 128 ? 64 : 32;    // of a thread that sums
  static constexpr int sum_warps = 4 * N / tokens;
  static constexpr int mma_warp = kTeam + sum_warps, w_warp = mma_warp + 1, x_warp = mma_warp + 2, threads = (mma_warp + 3) * 32;
  static constexpr int slots = 2;                      // rounds, and their x, between dequantisation and MMA
  static constexpr int stages = 4;                     // packed rounds on their way
  static constexpr int accs = (512 - slots * kOperand) / N;      // groups between MMA and sums
  static constexpr int a_col = accs * N;               // tensor memory: accumulators, then operands
  static constexpr int x_bytes = N * 128;              // B operand of 64 columns
  static constexpr int ring = slots * 4 * x_bytes + stages * 2 * kMaxRecord;
  static constexpr int row = N * 4 + 16;               // bytes between rows of sums on their way, up to 168 rows
  static constexpr int smem = (ring > 168 * row ? ring : 168 * row) + 1024;
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
// N consecutive columns of this warp's lanes
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&v)[N]) {
  if constexpr (N == 16) tmem_ld_32x32b_x16(taddr, v);
  else tmem_ld_x32(taddr, v);
}

template <bool BF16, int N>
__global__ void __launch_bounds__(Shape<N>::threads, 1) oproj_int4_kernel(const __grid_constant__ OprojInt4Params p) {
  using S = Shape<N>;
  constexpr int NT = S::tokens;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t w_full[S::stages], w_free[S::stages], a_full[S::slots], a_free[S::slots],
      g_full[S::accs], g_free[S::accs], drain;
  __shared__ uint32_t tmem_slot;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const x_ring = smem;
  uint8_t* const w_ring = x_ring + S::slots * 4 * S::x_bytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cl = (int)gridDim.y, rank = (int)blockIdx.y, slab = (int)blockIdx.x;          // a cluster is a column of the grid
  const int all = (p.K + 127) / 128, r0 = (int)((int64_t)all * rank / cl), r1 = (int)((int64_t)all * (rank + 1) / cl), rounds = (r1 - r0 + 1) / 2;
  const int k0 = r0 * 128, k1 = min(r1 * 128, p.K);    // this CTA's columns
  const int gshift = p.group == 32 ? 5 : p.group == 64 ? 6 : 7, group_bytes = p.zeros ? 384 : 256;
  const int record_bytes = 128 * 64 + (128 >> gshift) * group_bytes;
  auto columns = [&](int r) { return min(256, k1 - k0 - r * 256); };                      // of a round: 64 to 256

  if (tid == 0) {
    for (int i = 0; i < S::stages; ++i) {
      mbar_init(&w_full[i], 1);
      mbar_init(&w_free[i], kTeam + S::sum_warps);     // its nibbles and its scales have been read
    }
    for (int i = 0; i < S::slots; ++i) {
      mbar_init(&a_full[i], kTeam + 1);                // and the bytes of x
      mbar_init(&a_free[i], 1);
    }
    for (int i = 0; i < S::accs; ++i) {
      mbar_init(&g_full[i], 1);
      mbar_init(&g_free[i], S::sum_warps);
    }
    mbar_init(&drain, 1);
    mbar_fence_init();
  }
  if (warp == S::mma_warp) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  const unsigned long long deadline = now_ns() + p.timeout_ns;
  auto wait = [&](uint64_t* bar, int phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, deadline)) != 0; };
  bool ok = true;

  const int row = tid & (kRows - 1);
  const int part = warp < kTeam ? warp >> 2 : (warp - kTeam) >> 2;   // 64 columns of a record; NT of the tokens
  const int pair = (row & ~15) + (row & 7) * 2 + (row >> 3 & 1);     // of the row among the scales
  const uint32_t tq = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
  float2 acc[NT / 2];                                  // of the warps that sum
  if (warp < kTeam) {
    // =========================== dequantisation ===========================
    // both in registers: with two constants the compiler makes two instructions of (w & mask) | magic
    uint32_t mask, magic;
    asm volatile("mov.u32 %0, 0x000f000f;" : "=r"(mask));
    asm volatile("mov.u32 %0, %1;" : "=r"(magic) : "n"(BF16 ? 0x43004300 : 0x64006400));
    for (int r = 0; r < rounds; ++r) {
      const int st = r % S::stages, sl = r % S::slots, cols = columns(r);
      ok = wait(&w_full[st], r / S::stages);
      if (!ok) break;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int here = min(cols - 128 * j, 128);     // columns of the record
        uint32_t a[32];
        if (part * 64 < here) {
          const uint8_t* w = w_ring + st * (2 * kMaxRecord) + j * record_bytes;
          const uint8_t* zeros = w + here * 64 + ((here >> gshift) << 8);
#pragma unroll
          for (int h = 0; h < 2; ++h) {                // of 32 columns
            const uint4 q = *reinterpret_cast<const uint4*>(w + (row >> 4) * (here * 8) + (part * 2 + h) * 256 + (row & 15) * 16);
            const uint32_t z = p.zeros ? zeros[((part * 64 + h * 32) >> gshift) * kRows + pair] : 8u;
            const uint32_t z2 = magic + (z & 0xfu) * 0x00010001u;    // 128 + z, twice
            const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 4; ++i) a[16 * h + 4 * c + i] = sub2<BF16>(and_or(words[c] >> (4 * i), mask, magic), z2);
          }
        }
        if (j == 0 && r >= S::slots) {
          ok = wait(&a_free[sl], r / S::slots - 1);
          if (!ok) break;
          tc_fence_after_sync();
        }
        if (part * 64 < here) tmem_st_x32(tq + S::a_col + sl * kOperand + 64 * j + 32 * part, a);
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&a_full[sl]);
        mbar_arrive(&w_free[st]);
      }
    }
  } else if (warp < S::mma_warp) {
    // =========================== sums ===========================
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) acc[j] = make_float2(0.f, 0.f);
    for (int r = 0; r < rounds && ok; ++r) {
      const int st = r % S::stages, cols = columns(r), groups = cols >> gshift;
      ok = wait(&w_full[st], r / S::stages);
      if (!ok) break;
#pragma unroll 1
      for (int g = 0; g < groups; ++g) {
        const int n = r * (256 >> gshift) + g, at = n % S::accs;
        ok = wait(&g_full[at], n / S::accs);
        if (!ok) break;
        tc_fence_after_sync();
        const int j = g << gshift >> 7, here = min(cols - 128 * j, 128);       // record
        const uint16_t* scales = reinterpret_cast<const uint16_t*>(w_ring + st * (2 * kMaxRecord) + j * record_bytes + here * 64) + pair;
        const float s = widen<BF16>(scales[(g - (j << 7 >> gshift)) * kRows]);
        const float2 s2 = make_float2(s, s);
        constexpr int kRun = NT == 64 ? 16 : NT;         // as registers allow
#pragma unroll
        for (int c = 0; c < NT; c += kRun) {
          uint32_t v[kRun];
          tmem_ld<kRun>(tq + at * N + part * NT + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < kRun / 2; ++i) acc[c / 2 + i] = fma2(s2, make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), acc[c / 2 + i]);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&g_free[at]);
      }
      if (ok && lane == 0) mbar_arrive(&w_free[st]);
      __syncwarp();
    }
  } else if (warp == S::mma_warp) {
    // =========================== MMA issue ===========================
    constexpr uint32_t idesc = BF16 ? umma_idesc_bf16(kRows, N) : umma_idesc_bf16(kRows, N) & ~((1u << 7) | (1u << 10));
    const uint64_t d_x = umma_desc_k_sw128(smem_u32(x_ring));
    auto role = [&](auto shift) {
      constexpr int kShift = decltype(shift)::value;
      constexpr int kGroups = 256 >> kShift;
      for (int r_lane = 0; r_lane < rounds && ok; ++r_lane) {
        // through a shuffle: what is computed from it is then known to be the same in all lanes, which the MMA's operands want to be
        const int r = __shfl_sync(0xffffffffu, r_lane, 0), sl = r % S::slots, cols = columns(r);
        ok = wait(&a_full[sl], r / S::slots);
        if (!ok) break;
        const uint32_t ta = tmem + S::a_col + sl * kOperand, x_lo = (uint32_t)d_x + (sl * 4 * S::x_bytes >> 4), x_hi = (uint32_t)(d_x >> 32);
#pragma unroll
        for (int g = 0; g < 256; g += 1 << kShift) {
          if (g >= cols) break;
          const int i = g >> kShift, n = r * kGroups + i, at = kGroups < S::accs ? n % S::accs : i % S::accs;
          if (n >= S::accs && !(ok = wait(&g_free[at], n / S::accs - 1))) break;
          tc_fence_after_sync();
          if (elect_one()) {
#pragma unroll
            for (int k = g; k < g + (1 << kShift); k += 16) {
              const uint32_t lo = x_lo + ((k / 64 * S::x_bytes + k % 64 * 2) >> 4);
              if (k == g) umma_bf16_ts_first(tmem + at * N, ta + k / 2, lo, x_hi, idesc, 0u);
              else umma_bf16_ts(tmem + at * N, ta + k / 2, lo, x_hi, idesc);
            }
            umma_commit(&g_full[at]);
          }
          __syncwarp();
        }
        if (ok && elect_one()) umma_commit(&a_free[sl]);
        __syncwarp();
      }
    };
    if (gshift == 5) role(std::integral_constant<int, 5>{});
    else if (gshift == 6) role(std::integral_constant<int, 6>{});
    else role(std::integral_constant<int, 7>{});
    // the last arrivals have to be there before this CTA leaves
    for (int r = max(rounds - S::slots, 0); r < rounds && ok; ++r) ok = wait(&a_free[r % S::slots], r / S::slots);
    if (!ok) {
      if (elect_one()) umma_commit(&drain);            // nothing of this CTA's may be in flight when it leaves
      mbar_wait(&drain, 0, now_ns() + 10000000ull);
    }
  } else if (warp == S::w_warp) {
    // =========================== weights ===========================
    // (they do not depend on the kernel before this one)
    const uint8_t* w = p.w + (int64_t)slab * ((int64_t)p.K * 64 + (int64_t)(p.K >> gshift) * group_bytes) + (int64_t)r0 * record_bytes;
    for (int r = 0; r < rounds; ++r) {
      const int st = r % S::stages, cols = columns(r);
      if (r >= S::stages) ok = wait(&w_free[st], r / S::stages - 1);
      if (!ok) break;
      const uint32_t bytes = cols * 64 + (cols >> gshift) * group_bytes;
      if (lane == 0) {
        mbar_expect_tx(&w_full[st], bytes);
        bulk_load_1d(w_ring + st * (2 * kMaxRecord), w + (int64_t)r * 2 * record_bytes, bytes, &w_full[st]);
      }
      __syncwarp();
    }
  } else {
    // =========================== x ===========================
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int r = 0; r < rounds; ++r) {
      const int sl = r % S::slots, cols = columns(r);
      if (r >= S::slots) ok = wait(&a_free[sl], r / S::slots - 1);
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(&a_full[sl], cols / 64 * S::x_bytes);
        for (int c = 0; c < cols; c += 64) tma_load_2d(x_ring + (sl * 4 + c / 64) * S::x_bytes, &p.x_map, &a_full[sl], k0 + r * 256 + c, 0);
      }
      __syncwarp();
    }
  }
  if (!ok && lane == 0) atomicCAS(p.error_flag, 0, (int)kTimeoutMbarrier);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc_fence_before_sync();
  if (__syncthreads_or(ok ? 0 : 1) != 0) {
    // a wait ran out: nothing may land in this CTA's shared memory after it has left
    const unsigned long long limit = now_ns() + 1000000ull;
    while (now_ns() < limit) {
    }
  }
  if (warp == S::mma_warp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }

  // ---- results: thread (part, row) of the sums holds tokens part * NT ... of its row -------------------------------
  // Rank r finishes rows r * per ... of the slab.  Everybody is through with its rings, so they take the sums: [rank][row].
  const int rows_here = min(kRows, p.hidden - slab * kRows);
  const int per = (kRows / 8 + cl - 1) / cl * 8;
  auto meet = [&]() {
    if (cl == 1) {
      __syncthreads();
    } else {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
    }
  };
  meet();
  if (warp >= kTeam && warp < S::mma_warp) {
    uint8_t* const at = smem + (rank * per + row % per) * S::row + part * NT * 4;
    const int owner = row / per;
    const uint32_t to = map_to_cta(smem_u32(at), owner);
#pragma unroll
    for (int j = 0; j < NT; j += 4) {
      const float2 a = acc[j / 2], b = acc[j / 2 + 1];
      if (owner == rank) *reinterpret_cast<float4*>(at + j * 4) = make_float4(a.x, a.y, b.x, b.y);
      else st_cluster_f32x4(to + j * 4, a.x, a.y, b.x, b.y);
    }
  }
  meet();
  // a row and four tokens at a time: 16-byte reads of rows that lie 16 bytes past a multiple of 128 apart meet no bank twice
  const int mine = max(min(per, rows_here - rank * per), 0), quads = (p.tokens + 3) / 4;
  for (int e = tid; e < per * quads; e += S::threads) {
    const int n = e / per * 4, r = e % per;
    if (r >= mine) continue;
    const uint8_t* from = smem + r * S::row + n * 4;
    float4 v = *reinterpret_cast<const float4*>(from);
    for (int c = 1; c < cl; ++c) {
      const float4 w = *reinterpret_cast<const float4*>(from + c * per * S::row);
      v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
    }
    const float o[4] = {v.x, v.y, v.z, v.w};
    uint16_t* y = p.y + (int64_t)n * p.y_stride + slab * kRows + rank * per + r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.tokens) y[i * p.y_stride] = narrow<BF16>(o[i]);
  }
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16) {
    mma_bf16_16816(c, a[0], a[1], a[2], a[3], b0, b1);
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

__device__ __forceinline__ uint32_t ldg_stream(const uint8_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

// NT: tiles of eight tokens
template <bool BF16, int NT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kFewWarps * 32, 1) oproj_int4_few_kernel(const __grid_constant__ OprojInt4Params p) {
  constexpr int kGroups = 256 / GROUP;                 // of a warp's columns
  constexpr int kSum = 8 * NT * kRow;                  // sums of one row tile
  extern __shared__ __align__(128) uint8_t smem[];     // [warps][batch] sums, [inboxes][ranks][batch] of other CTAs
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warps = blockDim.x >> 5, cl = (int)gridDim.y, rank = (int)blockIdx.y;        // a cluster is a column of the grid
  const int col0 = (rank * warps + warp) * 256, blocks = min(max(p.K - col0, 0), 256) / 32;        // of 32 columns
  const int tiles = (p.hidden + 15) / 16, step = gridDim.x;
  if (cl > 1) cluster_arrive_relaxed();                // this CTA has started, its shared memory may be written by the others
  constexpr int kGroupBytes = ZEROS ? 384 : 256;
  constexpr int kRecord = 128 * 64 + 128 / GROUP * kGroupBytes;
  const int64_t slab_bytes = (int64_t)p.K * 64 + (int64_t)(p.K / GROUP) * kGroupBytes;
  struct Tile {
    uint32_t w[8][2];                                  // 32 columns: eight columns of row g, of row g + 8
    uint32_t s[kGroups], z[ZEROS ? kGroups : 1];
  };
  // Tiles behind the last are read as the last one: their sums go nowhere.
  auto fetch = [&](int tile, Tile& f) {
    tile = min(tile, tiles - 1);
    const uint8_t* slab = p.w + (tile >> 3) * slab_bytes + (int64_t)(col0 >> 7) * kRecord;
#pragma unroll
    for (int r = 0; r < 2; ++r) {                      // records
      const int in = min(max(blocks - 4 * r, 0), 4);   // blocks of 32 columns of it: 4, 2 or none
      const uint8_t* rec = slab + r * kRecord;
      const uint8_t* w = rec + (tile & 7) * (in * 256) + g * 16 + t * 4;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f.w[4 * r + b][0] = b < in ? ldg_stream(w + b * 256) : 0u;
        f.w[4 * r + b][1] = b < in ? ldg_stream(w + b * 256 + 128) : 0u;
      }
      const uint8_t* s = rec + in * 2048 + (tile & 7) * 32 + g * 4;
      const uint8_t* z = rec + in * 2048 + (in * 32 / GROUP) * 256 + (tile & 7) * 16 + g * 2;
#pragma unroll
      for (int i = 0; i < 128 / GROUP; ++i) {
        const bool there = i * GROUP < in * 32;
        f.s[r * (128 / GROUP) + i] = there ? __ldg(reinterpret_cast<const uint32_t*>(s + i * 256)) : 0u;
        if (ZEROS) f.z[r * (128 / GROUP) + i] = there ? __ldg(reinterpret_cast<const uint16_t*>(z + i * 128)) : 0u;
      }
    }
  };
  Tile next;
  fetch(blockIdx.x, next);                             // weights do not depend on the kernel before this one
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint32_t x[NT][8][4];                                // per 32 columns: 8 t ... 8 t + 7 of token g
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int n = nt * 8 + g;
    const uint4* row = reinterpret_cast<const uint4*>(p.x + n * p.x_stride + col0) + t;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint4 v = n < p.tokens && b < blocks ? __ldg(row + b * 4) : make_uint4(0, 0, 0, 0);
      x[nt][b][0] = v.x, x[nt][b][1] = v.y, x[nt][b][2] = v.z, x[nt][b][3] = v.w;
    }
  }

  float* const sums = reinterpret_cast<float*>(smem);
  float* const mine = sums + warp * (p.batch * kSum);
  // both in registers: with two constants the compiler makes two instructions of (w & mask) | magic
  uint32_t mask, magic;
  asm volatile("mov.u32 %0, 0x000f000f;" : "=r"(mask));
  asm volatile("mov.u32 %0, %1;" : "=r"(magic) : "n"(BF16 ? 0x43004300 : 0x64006400));
  constexpr uint32_t kMagic = BF16 ? 0x43004300u : 0x64006400u;
  // All have started; what came before has hidden most of the wait (8192 x 8192, 8 and 16 tokens 11.90 and 16.35 us, without the barrier 11.83 and 16.33;
  // with the wait before the first remote store, inside the loop, 11.98 and 16.9).
  if (cl > 1) cluster_wait();
  int turn = 0;
  const int all = (tiles - (int)blockIdx.x + step - 1) / step;         // of every warp alike
  for (int j0 = 0; j0 < all; j0 += p.batch) {
    const int batch = min(p.batch, all - j0);
#pragma unroll 1
    for (int j = j0; j < j0 + batch; ++j) {
      // with two tiles of tokens the registers do not hold a second tile of weights (8192 x 8192: 23.1 us with it, spilled, 16.6 without)
      if (NT == 2 && j > 0) fetch(blockIdx.x + j * step, next);
      const Tile f = next;
      if (NT == 1) fetch(blockIdx.x + (j + 1) * step, next);
      float acc[NT][4], part[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const int grp = b * 32 / GROUP;
        if (b * 32 % GROUP == 0) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[nt][i] = 0.f;
        }
        uint32_t z0 = kMagic + 0x00080008u, z1 = z0;                   // 128 + z of rows g and g + 8, twice each
        if (ZEROS) {
          z0 = kMagic + (f.z[grp] & 0xfu) * 0x00010001u;
          z1 = kMagic + (f.z[grp] >> 8 & 0xfu) * 0x00010001u;
        }
        // k of the MMA's step h: columns 8 t + 4 h ... + 3 of the 32, in the order in which x has them
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            a[i] = sub2<BF16>(and_or(f.w[b][i & 1] >> (8 * h + 4 * (i >> 1)), mask, magic), i & 1 ? z1 : z0);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<BF16>(part[nt], a, x[nt][b][2 * h], x[nt][b][2 * h + 1]);
        }
        if ((b + 1) * 32 % GROUP == 0) {
          const float s0 = widen<BF16>((uint16_t)f.s[grp]), s1 = widen<BF16>((uint16_t)(f.s[grp] >> 16));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            acc[nt][0] += s0 * part[nt][0];
            acc[nt][1] += s0 * part[nt][1];
            acc[nt][2] += s1 * part[nt][2];
            acc[nt][3] += s1 * part[nt][3];
          }
        }
      }
      // [token][row], tokens 2 t and 2 t + 1
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float* to = mine + (j - j0) * kSum + (nt * 8 + 2 * t) * kRow + g;
        to[0] = acc[nt][0];
        to[kRow] = acc[nt][1];
        to[8] = acc[nt][2];
        to[kRow + 8] = acc[nt][3];
      }
    }
    __syncthreads();
    // The warps' sums, in the order of the columns, four rows at a time; then the CTAs': run e of four rows is finished by rank e / 32 % cl,
    // whom the others send theirs.  (A run is rows 4 (e % 4) ... of token e / 4 % (8 NT) of tile e / (32 NT).)
    constexpr int kRuns = 32 * NT;
    auto at = [&](int e) { return e / kRuns * kSum + e % kRuns / 4 * kRow + e % 4 * 4; };
    auto store = [&](int e, float4 v) {
      const int n = e % kRuns / 4;
      const int row = (blockIdx.x + (j0 + e / kRuns) * step) * 16 + e % 4 * 4;
      if (n >= p.tokens || row >= p.hidden) return;
      uint16_t* to = p.y + n * p.y_stride + row;
      alignas(8) const uint16_t out[4] = {narrow<BF16>(v.x), narrow<BF16>(v.y), narrow<BF16>(v.z), narrow<BF16>(v.w)};
      if (p.hidden % 4 == 0) {
        *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(out);
      } else {
        for (int i = 0; i < min(4, p.hidden - row); ++i) to[i] = out[i];
      }
    };
    float4* const inbox = reinterpret_cast<float4*>(sums + warps * (p.batch * kSum)) + (turn & 1) * (cl * p.batch * kRuns);     // [rank][run]
    for (int e = threadIdx.x; e < batch * kRuns; e += blockDim.x) {
      const float* from = sums + at(e);
      float4 v = *reinterpret_cast<const float4*>(from);
#pragma unroll 4
      for (int w = 1; w < warps; ++w) {
        const float4 a = *reinterpret_cast<const float4*>(from + w * (p.batch * kSum));
        v = make_float4(v.x + a.x, v.y + a.y, v.z + a.z, v.w + a.w);
      }
      if (cl == 1) store(e, v);
      else st_cluster_f32x4(map_to_cta(smem_u32(inbox + rank * (p.batch * kRuns) + e), e / 32 % cl), v.x, v.y, v.z, v.w);
    }
    if (cl > 1) {
      // one barrier per batch: a CTA's own shared memory is all that is read behind it, and the inbox of the next batch is the other one
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      for (int e = (warp * cl + rank) * 32 + lane; e < batch * kRuns; e += blockDim.x * cl) {
        float4 v = inbox[e];
        for (int c = 1; c < cl; ++c) {
          const float4 a = inbox[c * (p.batch * kRuns) + e];
          v = make_float4(v.x + a.x, v.y + a.y, v.z + a.z, v.w + a.w);
        }
        store(e, v);
      }
      ++turn;
    } else {
      __syncthreads();
    }
  }
}

using Fn = void (*)(OprojInt4Params);
template <bool BF16>
Fn pick(int n, int* threads, size_t* smem) {
  if (n == 32) return *threads = Shape<32>::threads, *smem = Shape<32>::smem, (Fn)oproj_int4_kernel<BF16, 32>;
  if (n == 64) return *threads = Shape<64>::threads, *smem = Shape<64>::smem, (Fn)oproj_int4_kernel<BF16, 64>;
  return *threads = Shape<128>::threads, *smem = Shape<128>::smem, (Fn)oproj_int4_kernel<BF16, 128>;
}
template <bool BF16, int NT>
Fn pick_few(int group, bool zeros) {
  if (group == 32) return zeros ? (Fn)oproj_int4_few_kernel<BF16, NT, 32, true> : (Fn)oproj_int4_few_kernel<BF16, NT, 32, false>;
  if (group == 64) return zeros ? (Fn)oproj_int4_few_kernel<BF16, NT, 64, true> : (Fn)oproj_int4_few_kernel<BF16, NT, 64, false>;
  return zeros ? (Fn)oproj_int4_few_kernel<BF16, NT, 128, true> : (Fn)oproj_int4_few_kernel<BF16, NT, 128, false>;
}

cudaLaunchConfig_t config(int columns, int cl, int threads, size_t smem, bool pdl, cudaStream_t stream, cudaLaunchAttribute (&attrs)[2]) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)columns, (unsigned)cl, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
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

// Clusters of each size that are resident together, asked once per kernel, device and kind of launch
struct Resident {
  int clusters[kMaxCluster + 1];
};
cudaError_t resident(const void* fn, int dev, int threads, size_t smem, size_t max_smem, int sm_count, Resident* out) {
  static std::mutex mu;
  static std::map<std::tuple<int, const void*, int, size_t>, Resident> known;
  std::lock_guard<std::mutex> lk(mu);
  const auto key = std::make_tuple(dev, fn, threads, smem);
  const auto it = known.find(key);
  if (it != known.end()) {
    *out = it->second;
    return cudaSuccess;
  }
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)max_smem);
  if (e != cudaSuccess) return e;
  Resident r{};
  for (int cl = 1; cl <= kMaxCluster; ++cl) {
    cudaLaunchAttribute attrs[2];
    const cudaLaunchConfig_t cfg = config(sm_count, cl, threads, smem, false, nullptr, attrs);
    e = cudaOccupancyMaxActiveClusters(&r.clusters[cl], fn, &cfg);
    if (e != cudaSuccess) return e;
  }
  known[key] = r;
  *out = r;
  return cudaSuccess;
}

cudaError_t launch_few(OprojInt4Params p, bool pdl, int sm_count, int dev, cudaStream_t stream) {
  const int nt = (p.tokens + 7) / 8, tiles = (p.hidden + 15) / 16;
  const bool zeros = p.zeros != 0;
  const Fn fn = p.is_bf16 ? (nt == 1 ? pick_few<true, 1>(p.group, zeros) : pick_few<true, 2>(p.group, zeros))
                          : (nt == 1 ? pick_few<false, 1>(p.group, zeros) : pick_few<false, 2>(p.group, zeros));
  Int4FewPlan plan = int4_few_plan(p.tokens, p.hidden, p.K, sm_count);
  Resident r{};
  cudaError_t e;
  if (plan.cl == 1) {
    // Row tiles per CTA as if as many CTAs as have registers fitted on an SM; no more room for sums than that takes.  Without other CTAs'
    // sums any number of batches is right, so the grid may turn out another one.
    plan = int4_few_plan(p.tokens, p.hidden, p.K, sm_count * (kFewWarps / plan.warps));
    e = resident((const void*)fn, dev, plan.warps * 32, plan.bytes, kFewSmem, sm_count, &r);
    plan.columns = std::min(tiles, r.clusters[1]);
  } else {
    // The plan has to be that of the grid: a second batch writes to a second set of inboxes.  (A CTA of nine or more warps has an SM to
    // itself, so it costs nothing to ask with the largest size.)
    e = resident((const void*)fn, dev, plan.warps * 32, kFewSmem, kFewSmem, sm_count, &r);
    if (e == cudaSuccess && r.clusters[plan.cl] > 0) plan = int4_few_plan(p.tokens, p.hidden, p.K, r.clusters[plan.cl]);
  }
  if (e != cudaSuccess) return e;
  if (r.clusters[plan.cl] < 1 || plan.bytes > (size_t)kFewSmem) return cudaErrorInvalidConfiguration;
  p.batch = plan.batch;
  cudaLaunchAttribute attrs[2];
  const cudaLaunchConfig_t cfg = config(plan.columns, plan.cl, plan.warps * 32, plan.bytes, pdl, stream, attrs);
  return cudaLaunchKernelEx(&cfg, fn, p);
}

}  // namespace

Int4FewPlan int4_few_plan(int tokens, int hidden, int K, int resident) {
  const int slices = (K + 255) / 256, nt = (tokens + 7) / 8, tiles = (hidden + 15) / 16;
  Int4FewPlan plan{};
  plan.cl = 1;
  while (slices > plan.cl * kFewWarps) plan.cl *= 2;
  plan.warps = (slices + plan.cl - 1) / plan.cl;
  plan.columns = std::max(std::min(tiles, resident), 1);
  const int per = (tiles + plan.columns - 1) / plan.columns;
  for (plan.batch = std::min(per, 8);; --plan.batch) {
    plan.batches = (per + plan.batch - 1) / plan.batch;
    plan.inboxes = plan.cl == 1 ? 0 : std::min(plan.batches, 2);
    plan.bytes = (size_t)plan.batch * 8 * nt * (plan.warps * kRow + plan.inboxes * plan.cl * 16) * sizeof(float);
    if (plan.batch == 1 || plan.bytes <= (size_t)kFewSmem) return plan;
  }
}

cudaError_t launch_oproj_int4(OprojInt4Params p, bool pdl, int sm_count, cudaStream_t stream) {
  if (p.tokens <= 0 || p.hidden <= 0) return cudaSuccess;
  if (p.K <= 0 || p.K % 64 != 0 || (p.group != 32 && p.group != 64 && p.group != 128) || p.K % p.group != 0 || p.tokens > kInt4MaxTokens)
    return cudaErrorInvalidValue;
  int dev = 0;
  cudaGetDevice(&dev);
  // Measured in graphs, 8192 x 8192: 8 tokens 11.9 us, 16 tokens 16.4 (two launches of eight 24), the other kernel 21.2 from 17 tokens on.  A
  // wider K than a cluster's warps hold takes the other kernel, too.
  if (p.tokens <= kInt4FewTokens && p.K <= kMaxCluster * kFewWarps * 256) return launch_few(p, pdl, sm_count, dev, stream);
  size_t smem = 0;
  const int n = int4_pad_tokens(p.tokens);
  int threads = 0;
  const Fn fn = p.is_bf16 ? pick<true>(n, &threads, &smem) : pick<false>(n, &threads, &smem);
  Resident r;
  const cudaError_t e = resident((const void*)fn, dev, threads, smem, smem, sm_count, &r);
  if (e != cudaSuccess) return e;
  // As many CTAs per slab as make the launch shortest: rounds of resident clusters times the records of a CTA, and about ten records'
  // time for a CTA's start, the exchange and the end.  Measured with 100 tokens, clusters of 1 / 2 / 3 / 4 CTAs (74 clusters of two fit, 33 of
  // four, the output then 2 us slower): 8192 x 8192 45.6 / 29.5 / 46.1 / 39.5 us, 4096 x 4096 26.9 / 19.0 / 16.9 / 15.1, 28672 x 8192 91.0 / 110.7 / 125.1 / 132.6; the least is chosen
  // at all nine shapes that were tried, with 32 and 64 tokens too.
  const int slabs = (p.hidden + kRows - 1) / kRows, records = (p.K + 127) / 128;
  int best = 1;
  int64_t cost = INT64_MAX;
  for (int cl = 1; cl <= std::min(kMaxCluster, records); ++cl) {
    if (r.clusters[cl] < 1) continue;
    const int64_t c = (int64_t)((slabs + r.clusters[cl] - 1) / r.clusters[cl]) * ((records + cl - 1) / cl + 10);
    if (c < cost) {
      cost = c;
      best = cl;
    }
  }
  cudaLaunchAttribute attrs[2];
  const cudaLaunchConfig_t cfg = config(slabs, best, threads, smem, pdl, stream, attrs);
  return cudaLaunchKernelEx(&cfg, fn, p);
}

}  // namespace helix
