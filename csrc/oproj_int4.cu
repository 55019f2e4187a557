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
//   * Records of the packed weight arrive by bulk copy.  Two teams of eight warps take them in turn, turn nibbles into numbers and put them
//     into tensor memory as the MMA's A operand, a thread per row and 64 columns.  (In shared memory a record is 32 KB written and 32 KB read
//     for 8 KB that arrived.  A record is a chain of waits, loads and stores of ~1600 cycles for its team, so one team alone is half as fast.)
//   * Every group of a record has an accumulator of its own in tensor memory, filled while the team turns its next record into numbers;
//     then the same warps, a thread per row and half of the tokens, add it, times its scale, to their sums in registers.
//   * One barrier tells the MMA warp that a record is in place, its x too, and the accumulators read; one that its MMAs are through.
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
constexpr int kTeam = 8, kParts = kTeam / 4;     // warps that dequantise; threads that share a row
constexpr int kOperand = 64;                           // columns of tensor memory of a record's A operand
constexpr int kNibbles = 4096;                         // packed bytes of 64 columns
constexpr int kMaxRecord = 2 * kNibbles + 4 * 384;     // 128 columns in groups of 32, with zero points
constexpr int kMaxCluster = 8;
constexpr int kFewWarps = 16;
constexpr int kRow = 20;                               // floats between tokens of a tile's sums: 16 rows, and no bank conflicts
constexpr int kFewSmem = 200 * 1024;

template <int N>
struct Shape {
  // With more than 64 tokens the sums take the registers of a second team, and its accumulators the tensor memory.
  static constexpr int teams = N <= 64 ? 2 : 1, workers = teams * kTeam;
  static constexpr int mma_warp = workers, threads = (workers + 2) * 32;           // and a warp that loads
  static constexpr int slots = 2 * teams;              // records between dequantisation and MMA
  static constexpr int stages = 8;                     // packed records on their way
  static constexpr int accs = N <= 32 ? 4 : 2;     // groups of a record: more tokens want larger groups (int4_max_tokens)
  static constexpr int a_col = teams * accs * N;      // tensor memory: accumulators, then operands
  static_assert(a_col + slots * kOperand <= 512);
  static constexpr int x_bytes = N * 128;              // B operand of 64 columns
  static constexpr int ring = slots * 2 * x_bytes + stages * kMaxRecord;
  static constexpr int row = N * 4 + 16;               // bytes between rows of sums on their way, up to 168 rows of either team
  static constexpr int sums = teams * 168 * row;
  static constexpr int smem = (ring > sums ? ring : sums) + 1024;
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
  if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
  else if constexpr (N == 16) tmem_ld_32x32b_x16(taddr, v);
  else tmem_ld_x32(taddr, v);
}

template <bool BF16, int N>
__global__ void __launch_bounds__(Shape<N>::threads, 1) oproj_int4_kernel(const __grid_constant__ OprojInt4Params p) {
  using S = Shape<N>;
  constexpr int NT = N / kParts;                       // tokens of a worker thread
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t w_full[S::stages], w_free[S::stages], a_full[S::slots], a_free[S::slots], drain;
  __shared__ uint32_t tmem_slot;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const x_ring = smem;
  uint8_t* const w_ring = x_ring + S::slots * 2 * S::x_bytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cl = (int)gridDim.y, rank = (int)blockIdx.y, slab = (int)blockIdx.x;          // a cluster is a column of the grid
  const int all = (p.K + 127) / 128, r0 = (int)((int64_t)all * rank / cl), records = (int)((int64_t)all * (rank + 1) / cl) - r0;
  const int gshift = p.group == 32 ? 5 : p.group == 64 ? 6 : 7, group_bytes = p.zeros ? 384 : 256;
  auto columns = [&](int r) { return min(128, p.K - (r0 + r) * 128); };                   // of a record: 128, or 64 at the end of K

  if (tid == 0) {
    for (int i = 0; i < S::stages; ++i) {
      mbar_init(&w_full[i], 1);
      mbar_init(&w_free[i], kTeam);
    }
    for (int i = 0; i < S::slots; ++i) {
      mbar_init(&a_full[i], kTeam + 1);                // and the bytes of x
      mbar_init(&a_free[i], 1);
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
  bool ok = true;

  float acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = 0.f;
  if (warp < S::workers) {
    // =========================== dequantisation, and the sums ===========================
    const int row = tid & (kRows - 1), part = tid >> 7 & 1, team = tid >> 8;               // 64 of a record's columns; half of the tokens
    const int pair = (row & ~15) + (row & 7) * 2 + (row >> 3 & 1);   // of the row among the scales
    const uint32_t tq = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + team * (S::accs * N) + part * NT;
    // both in registers: with two constants the compiler makes two instructions of (w & mask) | magic
    uint32_t mask, magic;
    asm volatile("mov.u32 %0, 0x000f000f;" : "=r"(mask));
    asm volatile("mov.u32 %0, %1;" : "=r"(magic) : "n"(BF16 ? 0x43004300 : 0x64006400));
    // x of record r, into the place that record r - slots has left
    auto load_x = [&](int r) {
      if (warp % kTeam != 0 || lane != 0 || r >= records) return;
      const int sl = r % S::slots, cols = columns(r);
      mbar_expect_tx(&a_full[sl], cols / 64 * S::x_bytes);
      for (int c = 0; c < cols; c += 64)
        tma_load_2d(x_ring + (sl * 2 + c / 64) * S::x_bytes, &p.x_map, &a_full[sl], (r0 + r) * 128 + c, 0);
    };
    if (warp % kTeam == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int r = team; r < S::slots; r += S::teams) load_x(r);
    float s[S::accs], s_last[S::accs];                             // scales of the row's groups, of this record and of the one before
    int groups = 0;
    // the groups of record r, whose MMAs are waited for
    auto add_groups = [&](int r) {
      ok = __all_sync(0xffffffffu, mbar_wait(&a_free[r % S::slots], (r / S::slots) & 1, deadline));
      if (!ok) return;
      tc_fence_after_sync();
#pragma unroll
      for (int i = 0; i < S::accs; ++i) {
        if (i < groups) {
          constexpr int kRun = NT < 32 ? NT : 32;
#pragma unroll
          for (int c = 0; c < NT; c += kRun) {
            uint32_t v[kRun];
            tmem_ld<kRun>(tq + i * N + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < kRun; ++j) acc[c + j] += s_last[i] * __uint_as_float(v[j]);
          }
        }
      }
      tc_fence_before_sync();
    };
    int last = -1;                                     // the team's record before
    for (int r = team; r < records; last = r, r += S::teams) {
      const int st = r % S::stages, sl = r % S::slots, cols = columns(r);
      ok = __all_sync(0xffffffffu, mbar_wait(&w_full[st], (r / S::stages) & 1, deadline));
      if (!ok) break;
      // (the operand's place is free: the groups of the record that was there have been added up)
      const uint8_t* w = w_ring + st * kMaxRecord;
      const uint8_t* scales = w + cols * 64;
#pragma unroll
      for (int i = 0; i < S::accs; ++i) {
        s_last[i] = s[i];
        s[i] = (i << gshift) < cols ? widen<BF16>(reinterpret_cast<const uint16_t*>(scales)[i * kRows + pair]) : 0.f;
      }
      if (part * 64 < cols) {
        uint32_t a[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {                  // of 32 columns
          const uint4 q = *reinterpret_cast<const uint4*>(w + (row >> 4) * (cols * 8) + (part * 2 + h) * 256 + (row & 15) * 16);
          const uint32_t z = p.zeros ? scales[((cols >> gshift) << 8) + ((part * 64 + h * 32) >> gshift) * kRows + pair] : 8u;
          const uint32_t z2 = magic + (z & 0xfu) * 0x00010001u;      // 128 + z, twice
          const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) a[16 * h + 4 * c + i] = sub2<BF16>(and_or(words[c] >> (4 * i), mask, magic), z2);
        }
        tmem_st_x32(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + S::a_col + sl * kOperand + part * 32, a);
        tmem_st_wait();
        tc_fence_before_sync();
      }
      if (last >= 0) {
        add_groups(last);
        if (ok) load_x(last + S::slots);
      }
      groups = cols >> gshift;
      __syncwarp();
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive(&a_full[sl]);
        mbar_arrive(&w_free[st]);
      }
    }
#pragma unroll
    for (int i = 0; i < S::accs; ++i) s_last[i] = s[i];
    if (ok && last >= 0) add_groups(last);
  } else if (warp == S::mma_warp) {
    // =========================== MMA issue ===========================
    constexpr uint32_t idesc = BF16 ? umma_idesc_bf16(kRows, N) : umma_idesc_bf16(kRows, N) & ~((1u << 7) | (1u << 10));
    const uint64_t d_x = umma_desc_k_sw128(smem_u32(x_ring));
    auto role = [&](auto shift) {
      constexpr int kShift = decltype(shift)::value;
      for (int r_lane = 0; r_lane < records && ok; ++r_lane) {
        // through a shuffle: what is computed from it is then known to be the same in all lanes, which the MMA's operands want to be
        const int r = __shfl_sync(0xffffffffu, r_lane, 0), sl = r % S::slots, cols = columns(r);
        ok = __all_sync(0xffffffffu, mbar_wait(&a_full[sl], (r / S::slots) & 1, deadline));
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t td = tmem + r % S::teams * (S::accs * N), ta = tmem + S::a_col + sl * kOperand, x_lo = (uint32_t)d_x + (sl * 2 * S::x_bytes >> 4), x_hi = (uint32_t)(d_x >> 32);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 128; k += 16) {
            if (k == 64 && cols == 64) break;
            const uint32_t lo = x_lo + ((k / 64 * S::x_bytes + k % 64 * 2) >> 4), d = td + (k >> kShift) * N;
            if (k % (1 << kShift) == 0) umma_bf16_ts_first(d, ta + k / 2, lo, x_hi, idesc, 0u);
            else umma_bf16_ts(d, ta + k / 2, lo, x_hi, idesc);
          }
          umma_commit(&a_free[sl]);
        }
        __syncwarp();
      }
    };
    if (gshift == 5) role(std::integral_constant<int, 5>{});
    else if (gshift == 6) role(std::integral_constant<int, 6>{});
    else role(std::integral_constant<int, 7>{});
    if (!ok) {
      if (elect_one()) umma_commit(&drain);            // nothing of this CTA's may be in flight when it leaves
      mbar_wait(&drain, 0, now_ns() + 10000000ull);
    }
  } else {
    // =========================== loads ===========================
    const int record_bytes = 128 * 64 + (128 >> gshift) * group_bytes;
    const uint8_t* w = p.w + (int64_t)slab * ((int64_t)p.K * 64 + (int64_t)(p.K >> gshift) * group_bytes) + (int64_t)r0 * record_bytes;
    int w_at = 0;
    auto load_w = [&]() {
      const int st = w_at % S::stages, cols = columns(w_at);
      if (w_at >= S::stages) ok = __all_sync(0xffffffffu, mbar_wait(&w_free[st], (w_at / S::stages - 1) & 1, deadline));
      if (!ok) return;
      const uint32_t bytes = cols * 64 + (cols >> gshift) * group_bytes;
      if (lane == 0) {
        mbar_expect_tx(&w_full[st], bytes);
        bulk_load_1d(w_ring + st * kMaxRecord, w + (int64_t)w_at * record_bytes, bytes, &w_full[st]);
      }
      __syncwarp();
      ++w_at;
    };
    while (w_at < records && ok) load_w();             // weights do not depend on the kernel before this one
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

  // ---- results: thread (team, part, row) holds tokens part * NT ... of its row, the sum over its team's records ------
  // Rank r finishes rows r * per ... of the slab.  Everybody is through with its rings, so they take the sums: [rank][team][row].
  const int row = tid & (kRows - 1), part = tid >> 7 & 1, team = tid >> 8, rows_here = min(kRows, p.hidden - slab * kRows);
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
  if (warp < S::workers) {
    const uint32_t at = smem_u32(smem) + ((rank * S::teams + team) * per + row % per) * S::row + part * NT * 4;
    const uint32_t to = cl == 1 ? at : map_to_cta(at, row / per);
#pragma unroll
    for (int j = 0; j < NT; j += 4) {
      if (cl == 1) *reinterpret_cast<float4*>(smem + (at - smem_u32(smem)) + j * 4) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
      else st_cluster_f32x4(to + j * 4, acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
    }
  }
  meet();
  const int mine = max(min(per, rows_here - rank * per), 0);
  for (int e = tid; e < per * p.tokens; e += S::threads) {
    const int n = e / per, r = e % per;
    if (r >= mine) continue;
    const uint8_t* from = smem + r * S::row + n * 4;
    float v = *reinterpret_cast<const float*>(from);
    for (int c = 1; c < cl * S::teams; ++c) v += *reinterpret_cast<const float*>(from + c * per * S::row);
    p.y[n * p.y_stride + slab * kRows + rank * per + r] = narrow<BF16>(v);
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
  extern __shared__ __align__(128) uint8_t smem[];     // [warps][batch] sums, [2][ranks][batch] of other CTAs
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warps = blockDim.x >> 5, cl = (int)gridDim.y, rank = (int)blockIdx.y;        // a cluster is a column of the grid
  const int col0 = (rank * warps + warp) * 256, blocks = min(max(p.K - col0, 0), 256) / 32;        // of 32 columns
  const int tiles = (p.hidden + 15) / 16, step = gridDim.x;
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
      // the only barrier: a CTA's own shared memory is all that is read behind it, and the inbox of the next batch is the other one
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
  const int slices = (p.K + 255) / 256, nt = (p.tokens + 7) / 8, tiles = (p.hidden + 15) / 16;
  const bool zeros = p.zeros != 0;
  const Fn fn = p.is_bf16 ? (nt == 1 ? pick_few<true, 1>(p.group, zeros) : pick_few<true, 2>(p.group, zeros))
                          : (nt == 1 ? pick_few<false, 1>(p.group, zeros) : pick_few<false, 2>(p.group, zeros));
  int cl = 1;
  while (slices > cl * kFewWarps) cl *= 2;
  const int warps = (slices + cl - 1) / cl;
  // Row tiles per CTA as if as many CTAs as have registers fitted on an SM; no more room for sums than that takes.
  const int guess = std::max(sm_count * (kFewWarps / warps) / cl, 1), per = (tiles + guess - 1) / guess;
  auto bytes = [&](int batch) {
    const int inboxes = cl == 1 ? 0 : per <= batch ? cl : 2 * cl;
    return (size_t)batch * 8 * nt * (warps * kRow + inboxes * 16) * sizeof(float);
  };
  p.batch = std::min(per, 8);
  while (p.batch > 1 && bytes(p.batch) > (size_t)kFewSmem) --p.batch;
  Resident r;
  const cudaError_t e = resident((const void*)fn, dev, warps * 32, bytes(p.batch), kFewSmem, sm_count, &r);
  if (e != cudaSuccess) return e;
  if (r.clusters[cl] < 1) return cudaErrorInvalidConfiguration;
  cudaLaunchAttribute attrs[2];
  const cudaLaunchConfig_t cfg = config(std::min(tiles, r.clusters[cl]), cl, warps * 32, bytes(p.batch), pdl, stream, attrs);
  return cudaLaunchKernelEx(&cfg, fn, p);
}

}  // namespace

cudaError_t launch_oproj_int4(OprojInt4Params p, bool pdl, int sm_count, cudaStream_t stream) {
  if (p.tokens <= 0 || p.hidden <= 0) return cudaSuccess;
  if (p.K <= 0 || p.K % 64 != 0 || (p.group != 32 && p.group != 64 && p.group != 128) || p.K % p.group != 0 || p.tokens > int4_max_tokens(p.group))
    return cudaErrorInvalidValue;
  int dev = 0;
  cudaGetDevice(&dev);
  // Measured in graphs, 8192 x 8192: 8 tokens 12.1 us, 16 tokens 16.6 (two launches of eight 24), the other kernel 24.2 from 17 tokens on.  A
  // wider K than a cluster's warps hold takes the other kernel, too.
  if (p.tokens <= kInt4FewTokens && p.K <= kMaxCluster * kFewWarps * 256) return launch_few(p, pdl, sm_count, dev, stream);
  size_t smem = 0;
  const int n = int4_pad_tokens(p.tokens);
  int threads = 0;
  const Fn fn = p.is_bf16 ? pick<true>(n, &threads, &smem) : pick<false>(n, &threads, &smem);
  Resident r;
  const cudaError_t e = resident((const void*)fn, dev, threads, smem, smem, sm_count, &r);
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
  const cudaLaunchConfig_t cfg = config(slabs, best, threads, smem, pdl, stream, attrs);
  return cudaLaunchKernelEx(&cfg, fn, p);
}

}  // namespace helix
