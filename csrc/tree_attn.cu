// Attention of a tree of drafted tokens over the paged cache, head_dim 128, bf16 or fp16.
//
// Row (t, h) of a sequence and KV head, t a drafted token and h one of the group's query heads, sees all committed tokens of this
// rank's shard and those drafted ones whose mask bit is set:
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j - m),   lse = m + log sum_j p_j
//
// A group of 8 heads and 16 drafted tokens fill the 128 rows of one tensor-core tile, so both products run on tcgen05: S = Q K^T with
// both operands in shared memory, P back into tensor memory over S, O += P V with V as it lies in the cache (MN-major).
//   * Two streams per CTA, a softmax warpgroup each (a thread per row), keep tensor cores and exponentials busy.  With more than 128 rows
//     (`tiles` = 2) a stream is a tile of rows and every KV tile serves both.  With up to 128 rows a stream is half of every KV tile's
//     tokens, for all rows, with sums of its own that are joined at the end; scores have two buffers then, so that the next tile's are
//     there when this one's probabilities are.  (Streams that took alternate KV tiles held two tiles' V each through their softmax, which
//     left one place of the ring for loads: 128k tokens, 16 drafted 141 us.)
//   * The KV tiles of all (sequence, row tile, KV head) units form one line that is cut into equal shares, a CTA per SM.  A unit that
//     does not lie inside one share is left in pieces (normalised rows and their LSE), which a second kernel folds.
//   * The mask only concerns tiles that reach behind the committed tokens: there a row's mask words are shifted into place.
//     Masked scores are selected away, V rows behind the sequence are cleared in shared memory, and V elements of drafted tokens that are
//     not finite are cleared too and added at the end to the rows that see them, because 0 * inf would reach all rows.
//   * P is rounded to the inputs' type for the tensor cores, half a step per probability, which averages out over a row;
//     maxima, sums and O stay in fp32.  For fp16 P is held 2^7 larger, so that probabilities down to 2^-31 of the largest count.
// Every mbarrier wait is bounded; on expiry the kernel raises the error flag and leaves.
#include "tree_attn.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "helix_common.cuh"
#include "sm100.cuh"

namespace helix {
namespace {

using namespace sm100;

constexpr int kD = 128, kTile = 128, kRows = 128;
constexpr int kSlotBytes = kTile * kD * 2;             // 32768: one K tile, two halves of [128 tokens x 64 dims], or V tile (v_at)
constexpr int kHalf = kTile * 128;                     // 16384
constexpr int kSmWarps = 8, kMmaWarp = 8, kFirstLoad = 10, kLoadWarps = 2, kThreads = 384;      // an MMA warp per stream
constexpr int kSlots = 5;                              // beside two tiles of Q
constexpr int kSmem = (2 + kSlots) * kSlotBytes + 1024;
constexpr uint32_t kColS = 0, kColO = 256;             // S0, S1, O0, O1: 128 columns each; P lies over its S
constexpr int kSeqTable = 512;
constexpr int kWholeTiles = 4;                         // units of up to so many tiles stay whole, a CTA each
constexpr int kUnitCost = 2;                           // what a unit costs besides its tiles, in tiles
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescale = 8.f;                        // the running maximum moves when a row's grew by more than 2^8

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// maxima that pass a NaN on
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 32 bytes, a whole sector
__device__ __forceinline__ void st_global_x8(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint16_t x) {
  constexpr uint16_t e = BF16 ? 0x7f80 : 0x7c00;
  return (x & e) == e;
}
template <bool BF16>
__device__ __forceinline__ float widen(uint16_t x) {
  return BF16 ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
}
__device__ __forceinline__ void bar_sync_named(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

__device__ __forceinline__ int bar_or_named(int id, int n, int pred) {
  int r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.s32 p, %3, 0;\n"
      "bar.red.or.pred q, %1, %2, p;\n"
      "selp.s32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r)
      : "r"(id), "r"(n), "r"(pred)
      : "memory");
  return r;
}

__device__ __forceinline__ int seq_len_of(const TreeDecodeParams& p, int b) {
  return (int)min((long long)max(p.seq_lens[b], 0), (long long)p.max_pages * p.page_size);
}
__device__ __forceinline__ int row0_of(const TreeDecodeParams& p, int b) { return min(max(p.q_start[b], 0), p.rows); }

// One unit: the KV tiles of (sequence, tile group of rows, KV head).  On the line a unit is its tiles behind kUnitCost places that stand
// for what a unit costs besides (Q, the last tile's way through the pipeline, its output): without them CTAs with many short units
// were the last by far (24 ragged sequences up to 9000 tokens: 160 us against 85 for the others).  A segment is the part of a unit
// inside this CTA's share.  With `whole` a CTA takes units blockIdx.x, blockIdx.x + gridDim.x, ... from end to end.
// Sequences that all have the same number G > 1 of row tile groups lie on G lines, a lane of every G-th CTA each: the groups of a sequence
// then read the same KV tile at the same time, and all but one from L2 (128k tokens, 64 drafted, two groups: 537 MB from HBM instead of
// 1078, 269 us instead of 279, and under the power cap, where energy counts, 308 instead of 329).
struct Segment {
  int b, kvh, rg;
  int len, row0, n_rows;       // tokens; first row of the sequence's new tokens; rows of this unit (tokens * group, behind rg's start)
  int n_tiles, t_begin, count;
  int end;                     // of the unit, on the line
};

struct Walk {
  int gcur, g1, base, b;
  int lane;                    // -1: one line
  static __device__ __forceinline__ int units(const TreeDecodeParams& p, int b) {
    const int per = kRows * p.tiles, t = max(row0_of(p, b + 1) - row0_of(p, b), 0);
    return seq_len_of(p, b) > 0 ? (int)(((unsigned)t * (unsigned)(p.Hq / p.Hkv) + per - 1) / per) * p.Hkv : 0;
  }
  static __device__ __forceinline__ int length(const TreeDecodeParams& p, int b) {     // of a unit
    return p.whole ? 1 : (seq_len_of(p, b) + kTile - 1) / kTile + kUnitCost;
  }
  __device__ __forceinline__ bool next(const TreeDecodeParams& p, Segment& s) {
    while (gcur < g1 && b < p.B) {
      const int per = length(p, b), all = units(p, b), n = (lane < 0 ? all : min(all, p.Hkv)) * per;
      if (gcur >= base + n) {
        base += n;
        ++b;
        continue;
      }
      const int unit = (gcur - base) / per, at = gcur - base - unit * per, to = min(per, at + g1 - gcur);
      s.b = b;
      s.len = seq_len_of(p, b);
      s.row0 = row0_of(p, b);
      s.n_tiles = (s.len + kTile - 1) / kTile;
      s.rg = lane < 0 ? unit / p.Hkv : lane;
      s.kvh = lane < 0 ? unit - s.rg * p.Hkv : unit;
      s.n_rows = (row0_of(p, b + 1) - s.row0) * (p.Hq / p.Hkv) - s.rg * kRows * p.tiles;
      s.t_begin = p.whole ? 0 : max(at - kUnitCost, 0);
      s.count = p.whole ? s.n_tiles : max(to - kUnitCost, 0) - s.t_begin;
      s.end = base + (unit + 1) * per;
      gcur += p.whole ? gridDim.x : to - at;
      if (s.count > 0) return true;
    }
    return false;
  }
};

// Where token `tok` of a V tile begins, dims 0 ... 63 (before the swizzle): boxes of 2^shift tokens, both halves of the dims in each
__device__ __forceinline__ uint32_t v_at(int tok, int shift) { return ((tok >> shift) << (shift + 8)) + (tok & ((1 << shift) - 1)) * 128; }

// 32 visibility bits from drafted token `off` on (negative: committed ones before the first) of a row's mask words
__device__ __forceinline__ uint32_t mask_bits(const uint64_t* words, int n_words, int off) {
  if (off <= -32) return 0xffffffffu;
  auto at = [&](int w) { return w >= 0 && w < 2 * n_words ? reinterpret_cast<const uint32_t*>(words)[w] : 0u; };
  if (off < 0) return (n_words > 0 ? at(0) << -off : 0u) | (0xffffffffu >> (32 + off));
  const int w = off >> 5, sh = off & 31;
  return sh == 0 ? at(w) : at(w) >> sh | at(w + 1) << (32 - sh);
}

template <bool BF16, int MT>
__global__ void __launch_bounds__(kThreads, 1) tree_decode_kernel(const __grid_constant__ TreeDecodeParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t kv_full[kSlots], kv_free[kSlots], s_full[2], p_full[2][2], o_full[2], q_full, scrubbed, turn[2], drain[2];
  __shared__ uint32_t tmem_slot, s_poison[2][2 * kTreeMaxWords];      // by turns: a segment's is cleared behind its end
  __shared__ float s_x[2][kRows];                  // what the streams tell each other at the end of a segment
  __shared__ int s_rest, s_least, s_most;          // groups of row tiles of a sequence

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * kSlotBytes;           // behind two tiles of Q: both row tiles, or this segment's and the next one's
  int* s_base = reinterpret_cast<int*>(smem);      // [kSeqTable] first place of each sequence on the line, until Q comes
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = p.Hq / p.Hkv;
  const int box_shift = 31 - __clz(p.box_tok);

  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&kv_full[i], kLoadWarps);          // each announces its own bytes
      mbar_init(&kv_free[i], MT);                  // every stream that reads the tile
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i][0], 4);                 // halves of 64 tokens; with one row tile, every other KV tile
      mbar_init(&p_full[i][1], 4);
      mbar_init(&turn[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(&q_full, kSmWarps);
    mbar_init(&scrubbed, kSmWarps);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    s_rest = 0;
    s_least = 0x7fffffff;
    s_most = 0;
    mbar_fence_init();
  }
  if (tid < 4 * kTreeMaxWords) s_poison[0][tid] = 0;
  if (warp == kFirstLoad && lane == 0) {
    tma_prefetch_desc(&p.k_map);
    tma_prefetch_desc(&p.v_map);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  const unsigned long long deadline = now_ns() + p.timeout_ns;

  // ---- where the sequences lie on the line ---------------------------------------------------------------
  const int n_tab = min(p.B, kSeqTable);
  for (int b = tid; b < p.B; b += kThreads) {
    const int all = Walk::units(p, b), n = all * Walk::length(p, b);
    if (MT == 2 && all > 0) {
      atomicMin(&s_least, all / p.Hkv);
      atomicMax(&s_most, all / p.Hkv);
    }
    if (b < kSeqTable) s_base[b] = n;
    else if (n) atomicAdd(&s_rest, n);
  }
  __syncthreads();
  int total;
  {
    // every warp scans the table, and warp 0 leaves the result there
    const int run = (n_tab + 31) / 32, lo = min(lane * run, n_tab), hi = min(lo + run, n_tab);
    int mine = 0;
    for (int b = lo; b < hi; ++b) mine += s_base[b];
    int end = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += below;
    }
    total = __shfl_sync(0xffffffffu, end, 31);
    __syncthreads();
    if (warp == 0) {
      int at = end - mine;
      for (int b = lo; b < hi; ++b) {
        const int n = s_base[b];
        s_base[b] = at;
        at += n;
      }
    }
    __syncthreads();
  }
  int in_table = total;
  total += s_rest;
  // lanes, unless they leave more than one CTA in 32 without work (one row tile: a unit has all rows, or the caller's bound was too low)
  const int groups = s_most, lanes = MT == 2 && !p.whole && groups > 1 && groups == s_least && gridDim.x % groups * 32 <= gridDim.x && (int)gridDim.x >= groups ? groups : 1;
  total /= lanes;                                  // exact: every sequence has as many places on each
  in_table /= lanes;
  const int ctas = gridDim.x / lanes, share = max((int)(((unsigned)total + ctas - 1) / ctas), 1);
  const bool idle = (int)blockIdx.x >= ctas * lanes;
  const int here = (int)blockIdx.x / lanes;        // along the line
  const int cta = idle ? (int)blockIdx.x : (int)blockIdx.x % lanes * ctas + here;      // by which pieces and notes go: a line's are consecutive
  Walk walk;
  walk.lane = lanes > 1 ? (int)blockIdx.x % lanes : -1;
  walk.gcur = p.whole ? (int)blockIdx.x : idle ? total : (int)min((long long)here * share, (long long)total);
  walk.g1 = p.whole ? total : min(total, walk.gcur + share);
  if (walk.gcur < in_table) {
    int lo = 0, hi = n_tab;                        // the last sequence that starts at or before the share
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (s_base[mid] / lanes <= walk.gcur) lo = mid; else hi = mid;
    }
    walk.b = lo;
    walk.base = s_base[lo] / lanes;
  } else {
    walk.b = n_tab;
    walk.base = in_table;
  }
  __syncthreads();                                 // the table's place is Q's from here on
  Segment seg{};
  bool ok = true;
  uint32_t gt = 0;                                 // KV tiles this CTA has been through: fixes slots and phases

  if (warp < kSmWarps) {
    // =========================== softmax ===========================
    // 2 * 216 + 72 registers per thread of a warpgroup are what the block was launched with, 3 * 168
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int st = warp >> 2;                      // this warpgroup's stream
    const int quad = warp & 3, row = 32 * quad + lane;
    const uint32_t tq = tmem + ((uint32_t)(32 * quad) << 16);
    const uint32_t col_o = kColO + 128 * st;
    constexpr int kHere = MT == 1 ? 64 : 128, kChunks = kHere / 32;  // tokens of a tile that this stream takes
    const int first = MT == 1 ? 64 * st : 0;
    constexpr float kBias = BF16 ? 0.f : 7.f;
    const float sl2 = p.scale * kLog2e;
    const float2 sl22 = make_float2(sl2, sl2);
    uint32_t steps = 0, n_seg = 0, n_scrub = 0;    // of this stream, over all segments

    // Q of a segment into shared memory: K-major, 128-byte swizzle, halves of 64 dims
    auto load_q = [&](const Segment& sg, uint32_t n) {
      const int unit_row = (MT == 2 ? kRows * st : 0) + row, grow = sg.rg * kRows * MT + unit_row, node = grow / group;
      uint8_t* dst = smem + (MT == 2 ? st : n & 1) * kSlotBytes;
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)(sg.row0 + node) * p.q_sr + (int64_t)(sg.kvh * group + grow - node * group) * p.q_sh);
      const bool valid = unit_row < sg.n_rows;
      const int c0 = MT == 1 ? 8 * st : 0;
#pragma unroll
      for (int c = 0; c < (MT == 1 ? 8 : 16); ++c)
        *reinterpret_cast<uint4*>(dst + ((c0 + c) >> 3) * kHalf + swz128(row, c & 7)) = valid ? __ldg(src + c0 + c) : make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    };
    bool more = walk.next(p, seg);
    if (more) load_q(seg, 0);

    while (ok && more) {
      const int unit_row = (MT == 2 ? kRows * st : 0) + row;         // row of the unit
      const bool valid = unit_row < seg.n_rows;
      const int grow = seg.rg * kRows * MT + unit_row, node = grow / group;
      const int64_t qrow = seg.row0 + node, head = seg.kvh * group + grow - node * group;
      const bool warp_valid = __any_sync(0xffffffffu, valid);
      const int committed = seg.len - min(max(p.draft_lens[seg.b], 0), seg.len);
      const uint64_t* words = p.mask + (valid ? qrow : 0) * p.mask_stride;
      float m = -INFINITY, l = 0.f;
      bool huge = false;

      for (int i = 0; i < seg.count; ++i, ++steps) {
        const int tok0 = (seg.t_begin + i) * kTile;
        const bool special = tok0 + kTile > committed;               // reaches behind the committed tokens
        // the scores' place: the stream's own, or the tile's
        const int buf = MT == 1 ? steps & 1 : st;
        const uint32_t col_s = kColS + 128 * buf + first;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[buf], (MT == 1 ? steps >> 1 : steps) & 1, deadline));
        if (!ok) break;
        tc_fence_after_sync();
        if (special) {
          // V: rows behind the sequence become zeros, elements of drafted tokens that are not finite too.  A tile that both streams read
          // is shared out, and neither stream's P V starts before it is done; half tiles are each stream's own.
          const uint32_t r = 2 * (gt + i) + 1;
          uint8_t* v = ring + (r % kSlots) * kSlotBytes;
          ok = __all_sync(0xffffffffu, mbar_wait(&kv_full[r % kSlots], (r / kSlots) & 1, deadline));
          if (!ok) break;
          const int who = MT == 2 ? tid : row;
          for (int tok = max(committed - tok0, first) + (who >> 4); tok < first + kHere; tok += 8 * MT) {
            // (rows of 128 bytes, boxes of whole groups of eight: the swizzle goes by the token)
            uint4* at = reinterpret_cast<uint4*>(v + v_at(tok, box_shift) + ((row >> 3) & 1) * (p.box_tok * 128) + (((row & 7) ^ (tok & 7)) << 4));
            uint4 x = make_uint4(0, 0, 0, 0);
            if (tok0 + tok < seg.len) {
              x = *at;
              uint16_t* e = reinterpret_cast<uint16_t*>(&x);
              bool bad = false;
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (not_finite<BF16>(e[j])) {
                  e[j] = 0;
                  bad = true;
                }
              if (!bad) continue;
              const int d = tok0 + tok - committed;
              if (d < 64 * kTreeMaxWords) atomicOr(&s_poison[n_seg & 1][d >> 5], 1u << (d & 31));
            }
            *at = x;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (MT == 2) {
            if (lane == 0) mbar_arrive(&scrubbed);
            ok = __all_sync(0xffffffffu, mbar_wait(&scrubbed, n_scrub & 1, deadline));
            ++n_scrub;
            if (!ok) break;
          }
        }
        if (warp_valid) {
          if (special) {
            // masked scores become -inf where they lie; what is rare is kept in short loops, for the sake of the instruction cache
#pragma unroll 1
            for (int c = 0; c < kChunks; ++c) {
              uint32_t seen = mask_bits(words, p.words, tok0 + first + 32 * c - committed);
              const int left = seg.len - tok0 - first - 32 * c;
              if (left < 32) seen &= left <= 0 ? 0u : (1u << left) - 1u;
              uint32_t x[32];
              tmem_ld_x32(tq + col_s + 32 * c, x);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if ((seen >> j & 1u) == 0) x[j] = 0xff800000u;
              tmem_st_x32(tq + col_s + 32 * c, x);
            }
            tmem_st_wait();
          }
          uint32_t v[kChunks][32];
#pragma unroll
          for (int c = 0; c < kChunks; ++c) tmem_ld_x32(tq + col_s + 32 * c, v[c]);
          tmem_ld_wait();
          // The exponentials are what a step is made of (16 a cycle and SM: 1024 cycles a tile).  Two streams that start on the same KV tile
          // would stay in step, both at their exponentials and then both waiting for the tensor cores, so they take turns.
          if (MT == 2) {
            ok = __all_sync(0xffffffffu, mbar_wait(&turn[st], (steps & 1) ^ (st == 0 ? 1 : 0), deadline));
            if (!ok) break;
          }
          // P in two halves, so that P V of the first runs under the exponentials of the second.  The first half is computed with the
          // maximum so far, and the tile's own maximum beside it on a pipe that is idle then; if a row's grew by more than 2^8 the
          // maximum moves and the half is done again.
          float2 sum;
          float2 f2 = sl22;
          uint32_t pk[16];
          auto half_chunk = [&](int c, float2 mn2) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 d = fma2(make_float2(__uint_as_float(v[c][2 * j]), __uint_as_float(v[c][2 * j + 1])), f2, mn2);
              const float2 e = make_float2(fast_exp2(d.x), fast_exp2(d.y));
              sum = add2(sum, e);
              pk[j] = pack2<BF16>(e.x, e.y);
            }
            tmem_st_x16(tq + col_s + 16 * c, pk);
          };
          float mn = m == -INFINITY ? 0.f : -m;
          for (bool again = false;; again = true) {
            const float2 mn2 = make_float2(mn, mn);
            sum = make_float2(0.f, 0.f);
            if (huge && f2.x != 1.f) {
              f2 = make_float2(1.f, 1.f);
#pragma unroll
              for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int j = 0; j < 32; ++j) v[c][j] = __float_as_uint(__uint_as_float(v[c][j]) * sl2);
            }
            half_chunk(0, mn2);
            half_chunk(1, mn2);
            if (again) break;
            float mx[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) mx[c] = max_nan(__uint_as_float(v[c % kChunks][c]), __uint_as_float(v[c % kChunks][c + 4]));
#pragma unroll
            for (int j = 0; j < 32; j += 2)
#pragma unroll
              for (int c = 0; c < kChunks; ++c) mx[(c + j) & 3] = max_nan(mx[(c + j) & 3], __uint_as_float(v[c][j]), __uint_as_float(v[c][j + 1]));
            // a NaN or +inf among the scores makes the row's maximum NaN, and so all that is computed with it
            float top = max_nan(max_nan(mx[0], mx[1]), mx[2], mx[3]) * f2.x - kBias;
            if (top == INFINITY) top = __int_as_float(0x7fffffff);
            // (a row whose maximum is -inf, the first tile's, has nothing to take back if all its scores are -inf)
            const bool move = !(top <= m + kRescale) && top != -INFINITY;
            if (!__any_sync(0xffffffffu, move)) break;
            const float m_new = move ? max_nan(m, top) : m;
            const float alpha = m == m_new ? 1.f : m == -INFINITY ? 0.f : fast_exp2(m - m_new);
            l *= alpha;
            m = m_new;
            tmem_st_wait();                        // the half that will be done again
            if (i > 0) {
              if (MT == 1) {
                // scores come a tile early here; O is complete when V of the tile before has been read (its place in the ring was given out
                // before that of the K whose scores are here, so the parity is the right one)
                const uint32_t r = 2 * (gt + i) - 1;
                ok = __all_sync(0xffffffffu, mbar_wait(&kv_free[r % kSlots], (r / kSlots) & 1, deadline));
                if (!ok) break;
                tc_fence_after_sync();
              }
              // two row tiles: the scores' commit covers the P V before them, O is complete
#pragma unroll 1
              for (int c0 = 0; c0 < kD; c0 += 16) {
                uint32_t x[16];
                tmem_ld_32x32b_x16(tq + col_o + c0, x);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * alpha);
                tmem_st_x16(tq + col_o + c0, x);
              }
            }
            mn = m == -INFINITY ? 0.f : -m;
            // m is a rounded product, so s * sl2 - m is off by the rounding, alike for the whole row: up to 2^24 a factor of two at most.
            // Beyond, the products are rounded too, or the factor could overflow.
            huge |= __any_sync(0xffffffffu, fabsf(mn) > 16777216.f) != 0;
          }
          if (!ok) break;
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          // (one row tile: by turns, because a warp may be a tile ahead of its neighbours)
          if (lane == 0) mbar_arrive(&p_full[st][MT == 1 ? buf : 0]);
          if (MT == 2 && lane == 0) mbar_arrive(&turn[st ^ 1]);
          if constexpr (MT == 2) {
            half_chunk(2, make_float2(mn, mn));
            half_chunk(3, make_float2(mn, mn));
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[st][1]);
          }
          l += sum.x + sum.y;
        } else {
          if (MT == 2) ok = __all_sync(0xffffffffu, mbar_wait(&turn[st], (steps & 1) ^ (st == 0 ? 1 : 0), deadline));
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive(&p_full[st][MT == 1 ? buf : 0]);
            if (MT == 2) {
              mbar_arrive(&p_full[st][1]);
              mbar_arrive(&turn[st ^ 1]);
            }
          }
        }
      }

      // ---- the next segment's Q, while this one's last products run: its place is not read any more ------------
      Segment nx;
      more = ok && walk.next(p, nx);
      if (more) load_q(nx, n_seg + 1);

      // ---- join the streams -------------------------------------------------------------------------------------
      constexpr bool both = MT == 1;
      float f0, f1 = 0.f, M = m, L = l;
      if (MT == 1) {
        if (st == 1) {
          s_x[0][row] = m;
          s_x[1][row] = l;
        }
        bar_sync_named(1, 32 * kSmWarps);
        if (st == 0) {
          const float m1 = s_x[0][row];
          M = max_nan(m, m1);
          f0 = m == -INFINITY ? 0.f : fast_exp2(m - M);
          f1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - M);
          L = l * f0 + s_x[1][row] * f1;
          const float inv = L == 0.f ? 0.f : 1.f / L;                // a NaN stays one
          f0 *= inv;
          f1 *= inv;
          s_x[0][row] = f0;
          s_x[1][row] = f1;
        }
        bar_sync_named(1, 32 * kSmWarps);
        if (st == 1) {
          f0 = s_x[0][row];
          f1 = s_x[1][row];
        }
      } else {
        f0 = L == 0.f ? 0.f : 1.f / L;
      }
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&o_full[MT == 2 ? st : 0], n_seg & 1, deadline));
      tc_fence_after_sync();

      // ---- write the result or a piece ----------------------------------------------------------------------------
      uint32_t* const poison = s_poison[n_seg & 1];
      uint32_t poisoned = 0;
#pragma unroll
      for (int w = 0; w < 2 * kTreeMaxWords; ++w) poisoned |= poison[w];
      const bool whole = seg.count == seg.n_tiles;
      // slot 1: the piece that starts its unit; a CTA has at most one of each kind
      const int64_t piece = ((int64_t)cta * 2 + (seg.t_begin == 0 ? 1 : 0)) * kRows * MT + unit_row;
      const int c_begin = MT == 1 ? 64 * st : 0, c_end = MT == 1 ? c_begin + 64 : kD;
      if (warp_valid) {
        uint8_t* out = whole ? reinterpret_cast<uint8_t*>(p.o) + (qrow * p.Hq + head) * (kD * 2) : reinterpret_cast<uint8_t*>(p.part_o + piece * kD);
#pragma unroll 1
        for (int c0 = c_begin; c0 < c_end; c0 += 32) {
          uint32_t x[32], y[32];
          tmem_ld_x32(tq + (MT == 1 ? kColO : col_o) + c0, x);
          if (both) tmem_ld_x32(tq + kColO + 128 + c0, y);
          tmem_ld_wait();
          float o[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            o[j] = f0 == 0.f ? 0.f : __uint_as_float(x[j]) * f0;
            if (both) o[j] += f1 == 0.f ? 0.f : __uint_as_float(y[j]) * f1;
          }
          // whole sectors: 16-byte stores, a row per thread, took 13 us per segment of 256 rows
          if (valid && whole) {
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = pack2<BF16>(o[2 * j], o[2 * j + 1]);
            st_global_x8(out + c0 * 2, x);
            st_global_x8(out + c0 * 2 + 32, x + 8);
          } else if (valid) {
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(o[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j) st_global_x8(out + c0 * 4 + 32 * j, x + 8 * j);
          }
          __syncwarp();
        }
        if (poisoned != 0 && valid) {
          // the elements that were cleared, to the rows that see their token: a finite sum plus an infinity is that infinity
          for (int d = 0; d < 64 * p.words; ++d) {
            const int tok = committed + d;
            if (tok >= seg.len || (poison[d >> 5] >> (d & 31) & 1u) == 0 || (words[d >> 6] >> (d & 63) & 1u) == 0) continue;
            const int pg = p.block_table[seg.b * p.bt_stride + tok / p.page_size];
            if (pg < 0 || pg >= p.n_pages) continue;
            const uint16_t* src = p.v + pg * p.v_sp + (tok % p.page_size) * p.v_st + seg.kvh * p.v_sh;
#pragma unroll 1
            for (int c = c_begin; c < c_end; ++c) {
              if (!not_finite<BF16>(src[c])) continue;
              if (whole) {
                uint16_t* e = reinterpret_cast<uint16_t*>(out) + c;
                *e = (uint16_t)pack2<BF16>(widen<BF16>(*e) + widen<BF16>(src[c]), 0.f);
              } else {
                reinterpret_cast<float*>(out)[c] += widen<BF16>(src[c]);
              }
            }
          }
        }
        if (valid && (MT == 2 || st == 0)) {
          const float lse2 = L == 0.f ? -INFINITY : M + log2f(L);
          if (whole) p.lse[qrow * p.Hq + head] = p.lse_base2 ? lse2 : lse2 * kLn2;
          else p.part_lse[piece] = lse2;
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      // O and s_x are free; a warp that gave up takes the others with it, or they would wait for it
      if (bar_or_named(1, 32 * kSmWarps, ok ? 0 : 1)) ok = false;
      if (tid < 2 * kTreeMaxWords) poison[tid] = 0;                  // used again after the next segment's barrier
      ++n_seg;
      gt += seg.count;
      if (more) seg = nx;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  }
  if (warp >= kFirstLoad) {
    // =========================== loads ===========================
    // With pages of 16 tokens a tile is many small boxes, and a box costs the copy engine ~100 cycles whatever its size: 32 boxes of
    // 2 KB per tile, as K still has them, bounded everything (1 x 128k tokens, 16 drafted 141 us).  V, whose layout the MMA takes 16 tokens
    // at a time, comes with both halves of the dims in one box.
    const int per_tile = kTile / p.box_tok, lw = warp - kFirstLoad;
    uint32_t issued = 0;
    while (ok && walk.next(p, seg)) {
      const int32_t* bt = p.block_table + (int64_t)seg.b * p.bt_stride;
      auto page_at = [&](int i) {                  // page of block `lane` in tile i of the segment
        const int tok = (seg.t_begin + i) * kTile + lane * p.box_tok;
        return i < seg.count && lane < per_tile && tok < seg.len ? __ldg(bt + tok / p.page_size) : 0;
      };
      int page = page_at(0);
      for (int i = 0; i < seg.count && ok; ++i) {
        const int tok0 = (seg.t_begin + i) * kTile, in_page = (tok0 + lane * p.box_tok) % p.page_size;
        const int blocks = (min(seg.len - tok0, kTile) + p.box_tok - 1) / p.box_tok;
        const int next = page_at(i + 1);
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t r = 2 * (gt + i) + kv, slot = r % kSlots;
          if (r >= (uint32_t)kSlots) ok = __all_sync(0xffffffffu, mbar_wait(&kv_free[slot], (r / kSlots - 1) & 1, deadline));
          if (!ok) break;
          // K: a box per half of the dims, the halves shared by the two warps.  V: boxes of both halves, every other block.
          const int mine = kv == 0 ? blocks : (blocks - lw + kLoadWarps - 1) / kLoadWarps;
          if (lane == 0) mbar_expect_tx(&kv_full[slot], (uint32_t)mine * p.box_tok * (kv == 0 ? kD : 2 * kD));
          __syncwarp();
          for (int j = kv == 0 ? 0 : lw; j < blocks; j += kv == 0 ? 1 : kLoadWarps) {
            const int pg = __shfl_sync(0xffffffffu, page, j), at = __shfl_sync(0xffffffffu, in_page, j);
            if (elect_one()) {
              uint8_t* dst = ring + slot * kSlotBytes;
              if (kv == 0) tma_load_4d(dst + lw * kHalf + j * p.box_tok * 128, &p.k_map, &kv_full[slot], 64 * lw, at, seg.kvh, pg);
              else tma_load_5d(dst + j * p.box_tok * 256, &p.v_map, &kv_full[slot], 0, at, 0, seg.kvh, pg);
            }
            __syncwarp();
          }
          issued = r + 1;
        }
        page = next;
      }
      gt += seg.count;
    }
    // the last commits on kv_free have to arrive before this CTA leaves too
    for (uint32_t r = issued > (uint32_t)kSlots ? issued - kSlots : 0; r < issued && ok; ++r)
      ok = __all_sync(0xffffffffu, mbar_wait(&kv_free[r % kSlots], (r / kSlots) & 1, deadline));
    if (!ok) {
      // nothing may land in this CTA's shared memory after it has left
      const unsigned long long limit = now_ns() + 10000000ull;
      for (uint32_t r = issued > (uint32_t)kSlots ? issued - kSlots : 0; r < issued; ++r) mbar_wait(&kv_full[r % kSlots], (r / kSlots) & 1, limit);
    }
  } else if (warp >= kMmaWarp) {
    // =========================== MMA issue ===========================
    // rows that no unit covers: those of sequences without a token here, and those before the first and behind the last sequence
    if (warp == kMmaWarp) {
      auto clear = [&](int r0, int r1) {
        for (int64_t i = (int64_t)r0 * p.Hq * 16 + lane; i < (int64_t)r1 * p.Hq * 16; i += 32) {
          reinterpret_cast<uint4*>(p.o)[i] = make_uint4(0, 0, 0, 0);
          if (i % 16 == 0) p.lse[i / 16] = -INFINITY;
        }
      };
      for (int b = blockIdx.x; b < p.B; b += gridDim.x)
        if (seq_len_of(p, b) == 0) clear(row0_of(p, b), row0_of(p, b + 1));
      for (int r = blockIdx.x; r < row0_of(p, 0); r += gridDim.x) clear(r, r + 1);
      for (int r = row0_of(p, p.B) + blockIdx.x; r < p.rows; r += gridDim.x) clear(r, r + 1);
    }
    constexpr uint32_t fmt = BF16 ? umma_idesc_bf16(kRows, kTile) : umma_idesc_bf16(kRows, kTile) & ~((1u << 7) | (1u << 10));
    constexpr uint32_t id_s = fmt, id_o = fmt | (1u << 16);          // V is MN-major
    // all 512 columns are this CTA's: tensor memory starts at column 0, and no register holds the base
    const uint64_t d_q = umma_desc_k_sw128(smem_u32(smem)), d_k = umma_desc_k_sw128(smem_u32(ring)),
                   d_v = umma_desc_mn_sw128(smem_u32(ring), p.box_tok * 128);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, deadline)) != 0; };
    auto tile_there = [&](uint32_t r) { return wait(&kv_full[r % kSlots], (r / kSlots) & 1); };
    // scores of a tile that is there: S, 128 columns, and its commits
    auto scores = [&](uint32_t col, uint32_t qb, uint32_t r, uint64_t* done) {
      tc_fence_after_sync();
      const uint32_t kb = r % kSlots * kSlotBytes;
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < kD / 16; ++ks) {
          const uint32_t off = (ks >> 2) * kHalf + (ks & 3) * 32;
          umma_bf16(col, d_q + ((qb + off) >> 4), d_k + ((kb + off) >> 4), id_s, ks > 0);
        }
        umma_commit(done);
        umma_commit(&kv_free[r % kSlots]);
      }
      __syncwarp();
    };
    // O += P V for 64 tokens of a tile
    auto values = [&](uint32_t col_o, uint32_t col_p, uint32_t r, int tok, uint32_t later) {
      tc_fence_after_sync();
      const uint32_t v_lo = (uint32_t)d_v + (r % kSlots * kSlotBytes >> 4), v_hi = (uint32_t)(d_v >> 32);
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint32_t lo = v_lo + (v_at(tok + 16 * ks, box_shift) >> 4);
          if (ks == 0) umma_bf16_ts_first(col_o, col_p, lo, v_hi, id_o, later);
          else umma_bf16_ts(col_o, col_p + 8 * ks, lo, v_hi, id_o);
        }
      }
      __syncwarp();
    };
    uint32_t n_seg = 0, steps = 0;
    if constexpr (MT == 1) {
      // One warp: scores of the next but one tile follow the P V that frees their place.
      if (warp == kMmaWarp) {
        while (ok && walk.next(p, seg)) {
          const uint32_t qb = (__shfl_sync(0xffffffffu, n_seg, 0) & 1) * kSlotBytes;
          ok = wait(&q_full, n_seg & 1);
          ++n_seg;
          for (int i_lane = -2; i_lane < seg.count && ok; ++i_lane) {
            // through a shuffle: what is computed from it is then known to be the same in all lanes and stays in uniform registers,
            // where the MMA reads its operands (moving them there costs some 100 cycles each)
            const int i = __shfl_sync(0xffffffffu, i_lane, 0);
            const uint32_t tile = __shfl_sync(0xffffffffu, gt, 0) + i, r = 2 * tile + 1;
            if (i >= 0) {
              ok = tile_there(r);
              for (int st = 0; st < 2 && ok; ++st) {
                ok = wait(&p_full[st][tile & 1], (tile >> 1) & 1);
                if (!ok) break;
                values(kColO + 128 * st, kColS + 128 * (tile & 1) + 64 * st, r, 64 * st, i);
              }
              if (ok && elect_one()) umma_commit(&kv_free[r % kSlots]);
              __syncwarp();
            }
            if (ok && i + 2 < seg.count) {
              ok = tile_there(r + 3);
              if (ok) scores(kColS + 128 * (tile & 1), qb, r + 3, &s_full[tile & 1]);
            }
          }
          if (ok && elect_one()) umma_commit(&o_full[0]);
          __syncwarp();
          gt += seg.count;
        }
      }
    } else {
      // A warp per stream: one warp for both, in a fixed order, held a stream up behind the other (128k tokens, 64 drafted 315 us).  (The
      // stream is a constant of the code, so that the columns are.)
      auto role = [&](auto stream) {
        constexpr int st = decltype(stream)::value;
        while (ok && walk.next(p, seg)) {
          ok = wait(&q_full, n_seg & 1);
          ++n_seg;
          if (ok && (ok = tile_there(2 * __shfl_sync(0xffffffffu, gt, 0)))) scores(kColS + 128 * st, st * kSlotBytes, 2 * __shfl_sync(0xffffffffu, gt, 0), &s_full[st]);
          for (int i_lane = 0; i_lane < seg.count && ok; ++i_lane, ++steps) {
            const int i = __shfl_sync(0xffffffffu, i_lane, 0);
            const uint32_t r = 2 * (__shfl_sync(0xffffffffu, gt, 0) + i) + 1;
            // V first, and the next K before the second half: what is there already still takes a wait's time
            ok = tile_there(r) && wait(&p_full[st][0], steps & 1);
            if (!ok) break;
            values(kColO + 128 * st, kColS + 128 * st, r, 0, i);
            if (i + 1 < seg.count) ok = tile_there(r + 1);
            if (!ok || !(ok = wait(&p_full[st][1], steps & 1))) break;
            values(kColO + 128 * st, kColS + 128 * st + 32, r, 64, 1);
            if (elect_one()) umma_commit(&kv_free[r % kSlots]);
            __syncwarp();
            if (i + 1 < seg.count) scores(kColS + 128 * st, st * kSlotBytes, r + 1, &s_full[st]);
          }
          if (ok && elect_one()) umma_commit(&o_full[st]);
          __syncwarp();
          gt += seg.count;
        }
      };
      if (warp == kMmaWarp) role(std::integral_constant<int, 0>{});
      else role(std::integral_constant<int, 1>{});
    }
    if (!ok) {
      uint64_t* const mine = &drain[warp - kMmaWarp];
      if (elect_one()) umma_commit(mine);          // nothing of this CTA's may be in flight when it leaves
      mbar_wait(mine, 0, now_ns() + 10000000ull);
    }
  }
  if (!ok && lane == 0) atomicCAS(p.error_flag, 0, (int)kTimeoutMbarrier);

  // ---- what the fold has to do: the unit that this CTA begins and the next ones finish ---------------------
  if (tid == 0 && !p.whole) {
    int4 note = make_int4(-1, 0, 0, 0);
    if (seg.count > 0 && seg.t_begin == 0 && seg.count < seg.n_tiles) note = make_int4(seg.b, seg.kvh, seg.rg, cta - here + (seg.end - 1) / share);
    reinterpret_cast<int4*>(p.part_lse + tree_notes_at(p.ctas, p.tiles))[cta] = note;
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// The pieces of a unit that several CTAs shared, in the order of the CTAs.  Block (c, y): the unit that CTA c begins, a warp per row.
constexpr int kFoldThreads = 256, kFoldBatch = 8;
template <bool BF16>
__global__ void __launch_bounds__(kFoldThreads) tree_fold_kernel(const __grid_constant__ TreeDecodeParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 note = __ldcg(reinterpret_cast<const int4*>(p.part_lse + tree_notes_at(p.ctas, p.tiles)) + blockIdx.x);
  if (note.x < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.Hq / p.Hkv, per = kRows * p.tiles;
  const int row0 = row0_of(p, note.x), n_rows = min((row0_of(p, note.x + 1) - row0) * group - note.z * per, per);
  const int n = note.w - (int)blockIdx.x + 1;
  for (int r = blockIdx.y * (kFoldThreads / 32) + warp; r < n_rows; r += gridDim.y * (kFoldThreads / 32)) {
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < n; i0 += kFoldBatch) {
      float4 v[kFoldBatch];
      float l[kFoldBatch];
#pragma unroll
      for (int j = 0; j < kFoldBatch; ++j) {
        l[j] = -INFINITY;
        v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + j < n) {
          const int64_t piece = (((int64_t)blockIdx.x + i0 + j) * 2 + (i0 + j == 0 ? 1 : 0)) * per + r;
          l[j] = __ldcg(p.part_lse + piece);
          v[j] = __ldcg(reinterpret_cast<const float4*>(p.part_o + piece * kD) + lane);
        }
      }
      float top = M;
#pragma unroll
      for (int j = 0; j < kFoldBatch; ++j) top = fmaxf(top, l[j]);
      const float keep = M == -INFINITY ? 0.f : fast_exp2(M - top);
      M = top;
      L *= keep;
      acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
      for (int j = 0; j < kFoldBatch; ++j) {
        if (l[j] == -INFINITY) continue;
        const float w = fast_exp2(l[j] - top);
        L += w;
        acc.x += w * v[j].x;
        acc.y += w * v[j].y;
        acc.z += w * v[j].z;
        acc.w += w * v[j].w;
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int grow = note.z * per + r, node = grow / group;
    const int64_t at = (int64_t)(row0 + node) * p.Hq + note.y * group + grow - node * group;
    *(reinterpret_cast<uint2*>(p.o + at * kD) + lane) = make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
    if (lane == 0) {
      const float lse2 = L == 0.f ? -INFINITY : M + log2f(L);
      p.lse[at] = p.lse_base2 ? lse2 : lse2 * kLn2;
    }
  }
}

using Fn = void (*)(TreeDecodeParams);

}  // namespace

TreePlan tree_plan(int B, int Hkv, int group, int max_q, int max_seq_len, int sm_count) {
  TreePlan t;
  t.tiles = (long long)group * max_q > kRows ? 2 : 1;
  const long long per = (long long)kRows * t.tiles, n_tiles = std::max((max_seq_len + kTile - 1) / kTile, 1);
  const long long units = (long long)std::max(B, 1) * Hkv * (((long long)group * std::max(max_q, 1) + per - 1) / per);
  t.whole = units <= sm_count && n_tiles <= kWholeTiles;
  t.ctas = (int)std::min<long long>(t.whole ? units : units * n_tiles, sm_count);
  return t;
}

cudaError_t launch_tree_decode(const TreeDecodeParams& p, bool pdl, cudaStream_t stream) {
  if (p.rows <= 0) return cudaSuccess;
  if (p.Hkv <= 0 || p.Hq % p.Hkv != 0 || p.tiles < 1 || p.tiles > 2 || p.ctas < 1 || p.words < 0 || p.words > kTreeMaxWords ||
      (p.box_tok != 16 && p.box_tok != 32 && p.box_tok != 64 && p.box_tok != 128) || p.page_size % p.box_tok != 0)
    return cudaErrorInvalidValue;
  Fn fn = p.is_bf16 ? (p.tiles == 1 ? (Fn)tree_decode_kernel<true, 1> : (Fn)tree_decode_kernel<true, 2>)
                    : (p.tiles == 1 ? (Fn)tree_decode_kernel<false, 1> : (Fn)tree_decode_kernel<false, 2>);
  static bool attr_set[64][4] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  const int which = (p.is_bf16 ? 2 : 0) + p.tiles - 1;
  cudaError_t e = cudaSuccess;
  if (dev >= 64 || !attr_set[dev][which]) {
    e = cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_set[dev][which] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.ctas, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, fn, p);
  if (e != cudaSuccess || p.whole) return e;
  // the fold is always chained to this launch; it waits for the whole grid before it reads a piece
  cfg.gridDim = dim3(p.ctas, 16, 1);
  cfg.blockDim = dim3(kFoldThreads, 1, 1);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, p.is_bf16 ? (Fn)tree_fold_kernel<true> : (Fn)tree_fold_kernel<false>, p);
}

}  // namespace helix
