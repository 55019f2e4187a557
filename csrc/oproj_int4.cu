// o_proj with 4-bit weights for few tokens: a matrix-vector product on the warp-level tensor-core MMA.
//
// Bound by streaming the weights once (8192 x 8192: 33.5 MB, 5.1 us at the copy rate).  Everything is arranged so that a
// weight costs one pass through registers:
//   * A warp owns 256 columns, whose x it holds in registers as MMA B operands for the whole launch, and walks over 16-row tiles.  The
//     packed layout hands every lane its A operand as words of eight nibbles; with 0x4300 in front (0x6400 for fp16) a nibble is the
//     number 128 + q (1024 + q), from which 128 + z is subtracted exactly: three instructions for two weights.
//   * The products of a group are summed by the MMA in fp32 from exact integers, and only their sum is multiplied by the scale.
//   * The warps of a CTA, and up to eight CTAs of a cluster, share out the columns.  Their sums meet in shared memory, by distributed
//     shared memory across the cluster: no scratch memory, no atomics, one launch, one order of summation.
//   * Weights of the next tiles are requested before the present one is used; the first ones before the preceding kernel is waited for.
#include "oproj_int4.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "helix_common.cuh"
#include "sm100.cuh"

namespace helix {
namespace {

using namespace sm100;

constexpr int kUnits = 4;                 // 64-column units per warp
constexpr int kMaxWarps = 16;
constexpr int kBatch = 8;                 // row tiles whose sums a CTA keeps before it adds them up
constexpr int kAhead = 2;                 // tiles requested ahead

template <bool BF16>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  if (BF16) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
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
template <bool BF16>
__device__ __forceinline__ float2 widen2(uint32_t x) {
  if (BF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ uint4 ldg_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// NT: tiles of eight tokens
template <bool BF16, int NT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kMaxWarps * 32, 1) oproj_int4_kernel(const __grid_constant__ OprojInt4Params p) {
  constexpr int kGroups = kUnits * 64 / GROUP;         // of a warp's columns
  constexpr int kSum = 16 * 8 * NT;                    // sums of one row tile
  extern __shared__ float s_sum[];                     // [warps][kBatch][kSum], behind it [kBatch][kSum] of the whole CTA
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warps = blockDim.x >> 5, cl = (int)(gridDim.y), rank = (int)blockIdx.y;      // a cluster is a column of the grid
  const int units = p.K / 64, unit0 = (rank * warps + warp) * kUnits;
  const int n_units = min(max(units - unit0, 0), kUnits);
  const int tiles = p.hidden / 16, n_groups = p.K / GROUP;
  struct Tile {
    uint4 w[kUnits];
    uint32_t s[kGroups];
    uint32_t z[ZEROS ? kGroups : 1];
  };
  auto fetch = [&](int tile, Tile& f) {
    const uint4* w = p.w + ((int64_t)tile * units + unit0) * 32 + lane;
    const int64_t s0 = ((int64_t)tile * n_groups + unit0 * 64 / GROUP) * 8 + g;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) f.w[u] = tile < tiles && u < n_units ? ldg_stream(w + u * 32) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const bool in = tile < tiles && i * GROUP < n_units * 64;
      f.s[i] = in ? __ldg(p.scales + s0 + i * 8) : 0u;
      if (ZEROS) f.z[i] = in ? __ldg(p.zeros + s0 + i * 8) : 0u;
    }
  };
  Tile ahead[kAhead];
  const int step = gridDim.x;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) fetch(blockIdx.x + i * step, ahead[i]);

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint32_t x[NT][kUnits][8];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int n = nt * 8 + g;
    const uint4* row = reinterpret_cast<const uint4*>(p.x + n * p.x_stride + unit0 * 64 + 8 * t);
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint4 v = n < p.tokens && u < n_units ? __ldg(row + u * 8 + c * 4) : make_uint4(0, 0, 0, 0);
        x[nt][u][4 * c] = v.x, x[nt][u][4 * c + 1] = v.y, x[nt][u][4 * c + 2] = v.z, x[nt][u][4 * c + 3] = v.w;
      }
  }

  float* const mine = s_sum + warp * (kBatch * kSum);
  float* const whole = s_sum + warps * (kBatch * kSum);
  constexpr uint32_t kMagic = BF16 ? 0x43004300u : 0x64006400u;
  for (int tile0 = blockIdx.x; tile0 < tiles; tile0 += kBatch * step) {
    const int batch = min(kBatch, (tiles - tile0 + step - 1) / step);
#pragma unroll 2
    for (int j = 0; j < batch; ++j) {
      const Tile f = ahead[0];
#pragma unroll
      for (int i = 0; i + 1 < kAhead; ++i) ahead[i] = ahead[i + 1];
      fetch(tile0 + (j + kAhead) * step, ahead[kAhead - 1]);
      float acc[NT][4], part[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const uint32_t w[4] = {f.w[u].x, f.w[u].y, f.w[u].z, f.w[u].w};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int k = u * 64 + s * 16, grp = k / GROUP;
          if (k % GROUP == 0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i) part[nt][i] = 0.f;
          }
          // 128 + z of rows g and g + 8, twice each
          uint32_t z0 = kMagic + 0x00080008u, z1 = z0;
          if (ZEROS) {
            z0 = kMagic + (f.z[grp] & 0xfu) * 0x00010001u;
            z1 = kMagic + (f.z[grp] >> 8 & 0xfu) * 0x00010001u;
          }
          uint32_t a[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) a[i] = sub2<BF16>((w[s] >> (4 * i) & 0x000f000fu) | kMagic, i & 1 ? z1 : z0);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<BF16>(part[nt], a, x[nt][u][2 * s], x[nt][u][2 * s + 1]);
          if ((k + 16) % GROUP == 0) {
            const float2 sc = widen2<BF16>(f.s[grp]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              acc[nt][0] += sc.x * part[nt][0];
              acc[nt][1] += sc.x * part[nt][1];
              acc[nt][2] += sc.y * part[nt][2];
              acc[nt][3] += sc.y * part[nt][3];
            }
          }
        }
      }
      // [token][row], tokens 2 t and 2 t + 1
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float* to = mine + j * kSum + (nt * 8 + 2 * t) * 16 + g;
        to[0] = acc[nt][0];
        to[16] = acc[nt][1];
        to[8] = acc[nt][2];
        to[24] = acc[nt][3];
      }
    }
    __syncthreads();
    // the warps' sums, in the order of the columns
    for (int e = threadIdx.x; e < batch * kSum; e += blockDim.x) {
      float v = s_sum[e];
      for (int w = 1; w < warps; ++w) v += s_sum[w * (kBatch * kSum) + e];
      whole[e] = v;
    }
    auto store = [&](int e, float v) {
      const int j = e / kSum, n = e % kSum / 16, r = e % 16;
      if (n >= p.tokens) return;
      uint16_t* to = p.y + n * p.y_stride + (int64_t)(tile0 + j * step) * 16 + r;
      if (BF16) *reinterpret_cast<__nv_bfloat16*>(to) = __float2bfloat16_rn(v);
      else *reinterpret_cast<__half*>(to) = __float2half_rn(v);
    };
    if (cl == 1) {
      for (int e = threadIdx.x; e < batch * kSum; e += blockDim.x) store(e, whole[e]);
      __syncthreads();
    } else {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      // rank r finishes runs of 32 sums
      for (int e = rank * 32 + (threadIdx.x & 31) + warp * 32 * cl; e < batch * kSum; e += blockDim.x * cl) {
        float v = 0.f;
        for (int c = 0; c < cl; ++c) v += ld_cluster_f32(map_to_cta(smem_u32(whole + e), c));
        store(e, v);
      }
      __syncwarp();
      cluster_arrive();                                // nobody leaves, or begins the next batch, while a peer reads
      cluster_wait();
    }
  }
}

using Fn = void (*)(OprojInt4Params);
template <bool BF16, int NT>
Fn pick(int group, bool zeros) {
  if (group == 32) return zeros ? (Fn)oproj_int4_kernel<BF16, NT, 32, true> : (Fn)oproj_int4_kernel<BF16, NT, 32, false>;
  if (group == 64) return zeros ? (Fn)oproj_int4_kernel<BF16, NT, 64, true> : (Fn)oproj_int4_kernel<BF16, NT, 64, false>;
  return zeros ? (Fn)oproj_int4_kernel<BF16, NT, 128, true> : (Fn)oproj_int4_kernel<BF16, NT, 128, false>;
}

}  // namespace

cudaError_t launch_oproj_int4(const OprojInt4Params& p, bool pdl, int sm_count, cudaStream_t stream) {
  if (p.tokens <= 0 || p.hidden <= 0) return cudaSuccess;
  if (p.tokens > kInt4MaxTokens || p.K <= 0 || p.K > kInt4MaxK || p.K % 64 != 0 || p.hidden % 16 != 0 ||
      (p.group != 32 && p.group != 64 && p.group != 128) || p.K % p.group != 0)
    return cudaErrorInvalidValue;
  const int units = p.K / 64, slices = (units + kUnits - 1) / kUnits, nt = (p.tokens + 7) / 8;
  int cl = 1;
  while (slices > cl * kMaxWarps) cl *= 2;
  const int warps = (slices + cl - 1) / cl;
  const int tiles = p.hidden / 16, columns = std::max(sm_count * (kMaxWarps / warps) / cl, 1);
  const Fn fn = p.is_bf16 ? (nt == 1 ? pick<true, 1>(p.group, p.zeros != nullptr) : pick<true, 2>(p.group, p.zeros != nullptr))
                          : (nt == 1 ? pick<false, 1>(p.group, p.zeros != nullptr) : pick<false, 2>(p.group, p.zeros != nullptr));
  const size_t smem = (size_t)(warps + 1) * kBatch * 16 * 8 * nt * sizeof(float);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)std::min(tiles, columns), (unsigned)cl, 1);
  cfg.blockDim = dim3((unsigned)warps * 32, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = 1;
  attrs[0].val.clusterDim.y = (unsigned)cl;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, p);
}

}  // namespace helix
