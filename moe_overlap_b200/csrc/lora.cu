// Low-rank adapters of many requests beside a shared projection, on sm_100a.
//
//   y[m] = x[m] W^T + scale[i] (x[m] A[i]^T) B[i]^T,   i = ids[m] (-1: no adapter)
//
// The shared product is the grouped GEMM of one expert, which can take the adapters'
// second product into its accumulator; the kernels here prepare that and form the
// gradients.  Rows are taken in adapter order through a permutation, so each adapter is
// read once per block of its rows:
//   plan    perm (the rows with an adapter, by adapter, in row order), offs, and for each
//           tile of 256 rows the adapters in it and which rows are whose
//   shrink  s[p] = x[perm[p]] A[i]^T           (also dy B[i], with B read along rows)
//   expand  y[perm[p]] += scale[i] s[p] B[i]^T (also dx += scale[i] (dy B[i]) A[i]) for the
//           rows of tiles with more adapters than the shared product takes
//   grads   dB[i] = scale[i] sum_p dy[perm[p]]^T s[p]  (and dA[i])
// For the gradients and for expand s is held as two values of the inputs' type, the
// rounded one and what the rounding left: 16 bits of bf16.  fp16 has 22 bits but little
// range (dy B of gradients of 1e-5 lies below its normal numbers, where the second part is
// nothing), so s is scaled before it is split: by a power of two common to 16 rows of an
// adapter, the grads' step, which puts their largest between 2^6 and 2^14; what is lost is
// 2^-31 of that one at most.  expand undoes it by row, the grads step by step.  (x and dy
// themselves are taken as they are: the tensor cores add the products of a subnormal number
// at the place of 2^-14, so those of dy near 2^-24 keep some 14 bits, as in any product.)
// The shared product takes scale[i] s rounded to the type, like every operand of it; the sum
// with the shared part is then rounded once, where expand rounds it a second time.  A row of
// fp16 whose largest |scale[i] s| is beyond 65504 or below the normal numbers (2^-14) has no
// such operand: it is left to expand, with zeros in the product.
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/moe_overlap.h"
#include "gemm_common.cuh"
#include "host_common.h"
#include "lora.cuh"
#include "mma16.cuh"
#include "ptx.cuh"

namespace moe {
namespace lora {

constexpr int kMaxAdapters = 1024;
constexpr int kMaxRank = 128;

constexpr int kTileRows = 256;  // of the shared product
using gg::TileAdapters;

// The caller's plan buffer (int32, 16-byte aligned): what depends on the ids alone.
struct PlanView {
  TileAdapters* tile;  // [tiles]
  int32_t* taken;  // [m] whether the shared product takes the row's adapter
  int32_t* perm;   // [m]
  int32_t* offs;   // [adapters + 1]
  int32_t* base;   // {0, m}
  int32_t* queue;  // tile counters of the shared products of the forward and the backward, 0 before each
  // With fp16, per pass: whether shrink has left a row to expand (once set it stays: expand
  // then looks at `put`), the rows by place that the shared product takes, and the powers of
  // two of s and of t by blocks of 16 rows (see Range).
  int32_t* left;
  int32_t* put;  // [m]
  int32_t* exps[2];
  static int64_t tiles(int64_t m) { return (m + kTileRows - 1) / kTileRows; }
  // Entries of exps: block o / 16 of adapter i, whose rows start at place offs[i], is
  // number offs[i] / 16 + i + o / 16 (n rows make at most n / 16 + 1 blocks).
  static int64_t blocks16(int64_t m, int adapters) { return m / 16 + adapters + 1; }
  static int64_t ints(int64_t m, int adapters) {
    return tiles(m) * int64_t(sizeof(TileAdapters) / 4) + 3 * m + adapters + 6 + 2 * blocks16(m, adapters);
  }
  PlanView(void* plan, int64_t m, int adapters) {
    tile = static_cast<TileAdapters*>(plan);
    taken = reinterpret_cast<int32_t*>(tile + tiles(m));
    perm = taken + m;
    offs = perm + m;
    base = offs + adapters + 1;
    queue = base + 2;
    left = queue + 2;
    put = left + 1;
    exps[0] = put + m;
    exps[1] = exps[0] + blocks16(m, adapters);
  }
};

__device__ __forceinline__ int id_at(const void* ids, int ids64, int m, int L) {
  const int64_t v = ids64 ? static_cast<const int64_t*>(ids)[m]
                          : static_cast<int64_t>(static_cast<const int32_t*>(ids)[m]);
  return v < 0 || v >= L ? (v == -1 ? -1 : -2) : static_cast<int>(v);  // -2: a bad id
}

// Blocks 0 .. L-1 each take one adapter: they count the rows of smaller adapters (the
// segment's start) and write their own rows in order.  Blocks L .. take one row tile each:
// the adapters in it, which rows are whose, and whether the shared product takes them.
// No block depends on another and the order is always the same.  Every adapter's block reads
// all ids (from L2): nothing beside the products at tens of adapters, but 1024 of them take
// 0.05 ms more at 16384 rows and 0.6 ms at a million (64 x 64 products, with what expand
// then costs).
__global__ void __launch_bounds__(1024) plan_kernel(const void* ids, int ids64, int M, int L, PlanView plan,
                                                    int per_tile, int32_t* status) {
  let_next_kernel_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x;
  if (static_cast<int>(blockIdx.x) < L) {
    __shared__ int less[32], equal[32];
    constexpr int kBatch = 8;  // loads under way at a time
    const int i = blockIdx.x;
    const int per = ((M + 31) / 32 + 31) / 32 * 32;  // rows of a warp
    const int m0 = warp * per, m1 = min(M, m0 + per);
    int nl = 0, ne = 0;
    bool bad = false;
    for (int b = m0; b < m1; b += 32 * kBatch) {
      int v[kBatch];
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int m = b + 32 * q + lane;
        v[q] = m < m1 ? id_at(ids, ids64, m, L) : -1;
      }
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        nl += v[q] >= 0 && v[q] < i;
        ne += v[q] == i;
        bad |= v[q] == -2;
      }
    }
    if (bad && i == 0) record_status(status, MOE_ERR_INVALID_ARG);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      nl += __shfl_xor_sync(0xffffffffu, nl, o);
      ne += __shfl_xor_sync(0xffffffffu, ne, o);
    }
    if (lane == 0) less[warp] = nl, equal[warp] = ne;
    __syncthreads();
    int start = 0, at = 0, all = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      start += less[k];
      at += k < warp ? equal[k] : 0;
      all += equal[k];
    }
    if (tid == 0) {
      plan.offs[i] = start;
      if (i == L - 1) plan.offs[L] = start + all;
      if (i == 0) plan.base[0] = 0, plan.base[1] = M, plan.queue[0] = plan.queue[1] = 0, *plan.left = 0;
    }
    if (all == 0) return;
    at += start;
    for (int b = m0; b < m1; b += 32 * kBatch) {
      bool mine[kBatch];
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int m = b + 32 * q + lane;
        mine[q] = m < m1 && id_at(ids, ids64, m, L) == i;
      }
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const unsigned votes = __ballot_sync(0xffffffffu, mine[q]);
        if (mine[q]) plan.perm[at + __popc(votes & ((1u << lane) - 1u))] = b + 32 * q + lane;
        at += __popc(votes);
      }
    }
    return;
  }
  __shared__ unsigned present[kMaxAdapters / 32];  // a bit for each adapter
  __shared__ int before[kMaxAdapters / 32 + 1];
  static_assert(kMaxAdapters / 32 == 32, "one word a lane");
  const int t = blockIdx.x - L, m = t * kTileRows + tid;
  const int id = tid < kTileRows && m < M ? id_at(ids, ids64, m, L) : -1;
  if (tid < 32) present[tid] = 0;
  __syncthreads();
  if (id >= 0) atomicOr(&present[id >> 5], 1u << (id & 31));
  __syncthreads();
  if (tid < 32) {
    const int n = __popc(present[tid]);
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (tid >= o) incl += v;
    }
    before[tid] = incl - n;
    if (tid == 31) before[32] = incl;
  }
  __syncthreads();
  const int n = before[32];
  const bool take = n <= per_tile;
  TileAdapters& of = plan.tile[t];
  if (tid == 0) of.count = take ? n : 0, of.left = !take;
  if (tid >= kTileRows) return;
  const int rank = id >= 0 ? before[id >> 5] + __popc(present[id >> 5] & ((1u << (id & 31)) - 1u)) : -1;
  if (m < M) plan.taken[m] = take && id >= 0;
  if (!take) return;
  if (id >= 0) of.list[rank] = id;  // (every row of it writes the same word)
  for (int q = 0; q < n; ++q) {
    const unsigned rows = __ballot_sync(0xffffffffu, rank == q);
    if (lane == 0) of.mine[q][warp] = rows;
  }
}

// ---------------------------------------------------------- tensor-core tiles --
// All three products move far more bytes than they need arithmetic for at the ranks
// of adapters, so they run on m16n8k16 from shared memory filled by cp.async: rows
// are gathered through perm, which whole-tile TMA boxes cannot do.  Rows of shared
// memory are 16 bytes longer than a multiple of 32, so that ldmatrix meets no bank
// twice.  RP is the rank rounded up to 16, 32, 64 or 128.
constexpr int kThreads = 256;

// The sum over the cluster's CTAs, in their order, of 4 floats at this CTA's address
// `at`; every CTA's load is under way before the first is used.
__device__ __forceinline__ float4 cluster_sum4(const float* at, int parts) {
  if (parts == 1) return *reinterpret_cast<const float4*>(at);
  const uint32_t mine = smem_u32(at);
  float4 v[8];
#pragma unroll
  for (int q = 0; q < 8; ++q)
    if (q < parts)
      asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                   : "=f"(v[q].x), "=f"(v[q].y), "=f"(v[q].z), "=f"(v[q].w)
                   : "r"(mapa_shared(mine, q))
                   : "memory");
  float4 s = v[0];
#pragma unroll
  for (int q = 1; q < 8; ++q)
    if (q < parts) s.x += v[q].x, s.y += v[q].y, s.z += v[q].z, s.w += v[q].w;
  return s;
}

// Block `tile` of at most TILE rows of one adapter: its adapter (-1: no such block), first
// place and rows.  Called by a whole CTA; every warp finds it for itself.
struct Tile {
  int i, p0, rows;
};
__device__ __forceinline__ Tile find_tile(const int32_t* offs, int L, int tile, int TILE) {
  const int lane = threadIdx.x & 31;
  Tile t{-1, 0, 0};
  int before = 0;
  for (int b = 0; b < L; b += 32) {
    const int i = b + lane;
    const int o0 = i < L ? offs[i] : 0, n = i < L ? offs[i + 1] - o0 : 0;
    const int blocks = (n + TILE - 1) / TILE;
    int incl = blocks;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const int k = tile - before - (incl - blocks);  // block of this adapter
    const unsigned hit = __ballot_sync(0xffffffffu, k >= 0 && k < blocks);
    if (hit) {
      const int src = __ffs(hit) - 1;
      t.i = b + src;
      const int kk = __shfl_sync(0xffffffffu, k, src);
      const int o = __shfl_sync(0xffffffffu, o0, src), nn = __shfl_sync(0xffffffffu, n, src);
      t.p0 = o + kk * TILE;
      t.rows = min(TILE, nn - kk * TILE);
      return t;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return t;
}

// What fp16 needs beside the two parts of s (bf16 has fp32's range and needs nothing).
struct Range {
  int32_t* exps;  // of s: the powers of two that it was divided by, kNoExp where there is nothing to scale
  int32_t* put;   // [m] by place
  int32_t* left;
};
constexpr int kNoExp = -1000;
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 .. 127
// |v| if it is finite, else 0, as the bits of the float (which order as integers do).
__device__ __forceinline__ uint32_t finite_abs(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t finite_abs(const float4& v) {
  return max(max(finite_abs(v.x), finite_abs(v.y)), max(finite_abs(v.z), finite_abs(v.w)));
}
// The power of two for a block whose largest value has these bits: multiples of 8, so that
// neighbouring blocks mostly share it, leave that value between 2^6 and 2^14.  The bounds
// keep sums of such blocks within fp32; products of fp16 values reach neither of them.
__device__ __forceinline__ int exp_of(uint32_t largest) {
  if (largest == 0) return kNoExp;
  const int e = (static_cast<int>(largest >> 23) - 127 - 6) & ~7;  // (a two's complement floor)
  return min(max(e, -56), 64);
}

// shrink.  A CTA forms 128 rows x RP of s over one part of k: 4 warps of 32 rows (each
// reads all of w's tile from shared memory) for each half of a stage's columns (of the rank,
// if it is 128: all of it would be 128 sums a lane); the CTAs of a cluster
// share the rows and add their parts through distributed shared memory, in order.
// Bound by reading x once (and w once a block of 128 rows); measured 28 us for 16384 rows
// of 2048 (67 MB, rank 64) and 80 us for 16384 of 8192 (268 MB, 3.4 TB/s): the gathers'
// instructions and the barriers between stages, not memory, take the rest.
constexpr int kShrinkRows = 128;
constexpr int kShrinkCols = 64;  // of k, a stage
constexpr int kShrinkPitch = kShrinkCols * 2 + 16;

template <bool kT, int RP>
struct ShrinkCfg {
  static constexpr int kW = kT ? kShrinkCols * (RP * 2 + 16) : RP * kShrinkPitch;
  static constexpr int kStage = kShrinkRows * kShrinkPitch + kW;
  static constexpr int kStages = RP == 128 ? 3 : 4;
  static constexpr int kBytes = kStages * kStage;
  static_assert(kShrinkRows * (RP + 4) * 4 <= kBytes, "the sums reuse the stages");
};

template <typename T, bool kT, int RP>
__global__ void __launch_bounds__(kThreads, 2)
    shrink_kernel(const T* x, int64_t ldx, const T* w, int64_t sl, int64_t sr, const int32_t* perm,
                  const int32_t* offs, int L, int K, int r, int64_t part_stride, T* s, Scale scale,
                  const int32_t* taken, T* rows, Range range) {
  using C = ShrinkCfg<kT, RP>;
  extern __shared__ __align__(128) char smem[];
  constexpr bool kScaled = std::is_same<T, __half>::value;
  __shared__ int row_of[kShrinkRows];  // -1: not the shared product's
  [[maybe_unused]] __shared__ uint32_t largest[kShrinkRows / 16];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  wait_for_previous_kernel();
  let_next_kernel_start();
  const Tile t = find_tile(offs, L, blockIdx.x, kShrinkRows);
  if (t.i < 0) return;  // the same in every CTA of the cluster
  const float c = scale.of(t.i);
  if (tid < t.rows) {
    const int row = perm[t.p0 + tid];
    row_of[tid] = taken[row] ? row : -1;
  }
  if (kScaled && tid < kShrinkRows / 16) largest[tid] = 0;
  const int parts = gridDim.y, part = blockIdx.y;
  const int cols = ((K + parts - 1) / parts + kShrinkCols - 1) / kShrinkCols * kShrinkCols;
  const int k0 = min(K, part * cols), k1 = min(K, k0 + cols);
  const int steps = (k1 - k0 + kShrinkCols - 1) / kShrinkCols;
  const T* wi = w + t.i * sl;
  // What this thread copies: a 16-byte piece of 4 rows of x and of some rows of w, at
  // pointers that move on by a stage each time (rows that are not there stay at their
  // base and copy nothing).
  constexpr int kRowSteps = kThreads / 8, kXCopies = kShrinkRows / kRowSteps;
  constexpr int kWPieces = kT ? RP / 8 : kShrinkCols / 8, kWRows = kT ? kShrinkCols : RP;
  constexpr int kWCopies = (kWRows * kWPieces + kThreads - 1) / kThreads;
  const int piece = (tid & 7) * 8;
  const T* xp[kXCopies];
  uint32_t x_there = 0, w_there = 0;
#pragma unroll
  for (int q = 0; q < kXCopies; ++q) {
    const int m = tid / 8 + kRowSteps * q;
    const bool there = m < t.rows;
    xp[q] = x + (there ? perm[t.p0 + m] * ldx : 0) + k0 + piece;
    x_there |= uint32_t(there) << q;
  }
  const T* wp[kWCopies];
#pragma unroll
  for (int q = 0; q < kWCopies; ++q) {
    const int e = tid + q * kThreads, row = e / kWPieces, c = e % kWPieces * 8;
    const bool there = row < kWRows && (kT ? c : row) < r;
    wp[q] = wi + (there ? (kT ? int64_t(k0 + row) * sr + c : row * sr + k0 + c) : 0);
    w_there |= uint32_t(there) << q;
  }
  const int64_t w_step = kT ? kShrinkCols * sr : kShrinkCols;
  int ck = k0, at = 0;  // the column and the stage of the next fetch
  auto fetch = [&]() {
    if (ck < k1) {
      const uint32_t xs = smem_u32(smem) + at * C::kStage + tid / 8 * kShrinkPitch + piece * 2;
      const uint32_t ws = smem_u32(smem) + at * C::kStage + kShrinkRows * kShrinkPitch;
      const bool k_in = ck + piece < k1;
#pragma unroll
      for (int q = 0; q < kXCopies; ++q) {
        copy_async_16(xs + kRowSteps * q * kShrinkPitch, xp[q], k_in && (x_there >> q & 1));
        xp[q] += kShrinkCols;
      }
#pragma unroll
      for (int q = 0; q < kWCopies; ++q) {
        const int e = tid + q * kThreads, row = e / kWPieces, c = e % kWPieces;
        const bool in = (w_there >> q & 1) && (kT ? ck + row < k1 : k_in);
        if (row < kWRows) copy_async_16(ws + row * (kT ? RP * 2 + 16 : kShrinkPitch) + c * 16, wp[q], in);
        wp[q] += w_step;
      }
      ck += kShrinkCols;
      if (++at == C::kStages) at = 0;
    }
    copies_commit();
  };
  constexpr bool kByRank = RP == 128;
  constexpr int kRanks = kByRank ? RP / 2 : RP, kDeep = kByRank ? kShrinkCols : kShrinkCols / 2;
  float acc[2][kRanks / 8][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < kRanks / 8; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[m][n][q] = 0.0f;
#pragma unroll
  for (int q = 0; q < C::kStages - 1; ++q) fetch();
  const int mg = warp & 3, kg = warp >> 2, n_first = kByRank ? kg * kRanks : 0;
  const bool busy = mg * 32 < t.rows;  // a warp without rows only copies
  for (int step = 0, stage = 0; step < steps; ++step, stage = stage + 1 == C::kStages ? 0 : stage + 1) {
    copies_wait<C::kStages - 2>();
    __syncthreads();
    fetch();
    const uint32_t xs = smem_u32(smem) + stage * C::kStage;
    const uint32_t ws = xs + kShrinkRows * kShrinkPitch;
    if (!busy) continue;
#pragma unroll
    for (int q = 0; q < kDeep; q += 16) {
      const int kk = kByRank ? q : kg * kDeep + q;
      uint32_t a[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
        ldmatrix_x4<false>(a[m], xs + (mg * 32 + m * 16 + (lane & 15)) * kShrinkPitch +
                                     (kk + (lane >> 4) * 8) * 2);
#pragma unroll
      for (int n = 0; n < kRanks / 8; n += 2) {
        uint32_t b[4];
        if constexpr (kT)
          ldmatrix_x4<true>(b, ws + (kk + (lane & 15)) * (RP * 2 + 16) + (n_first / 8 + n + (lane >> 4)) * 16);
        else
          ldmatrix_x4<false>(b, ws + (n_first + n * 8 + (lane >> 4) * 8 + (lane & 7)) * kShrinkPitch +
                                    (kk + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          mma<T>(acc[m][n], a[m], b[0], b[1]);
          mma<T>(acc[m][n + 1], a[m], b[2], b[3]);
        }
      }
    }
  }
  copies_wait<0>();
  __syncthreads();
  constexpr int kPitch = RP + 4;
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int half = 0; half < (kByRank ? 1 : 2); ++half) {  // the second half's warps add to the first's
    if (kByRank || kg == half)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < kRanks / 8; ++n)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float2* at = reinterpret_cast<float2*>(sums + (mg * 32 + m * 16 + (lane >> 2) + 8 * q) * kPitch +
                                                   n_first + n * 8 + (lane & 3) * 2);
            float2 v = make_float2(acc[m][n][2 * q], acc[m][n][2 * q + 1]);
            if (half == 1) v.x += at->x, v.y += at->y;
            *at = v;
          }
    if (!kByRank && half == 0) __syncthreads();
  }
  if (parts > 1)
    cluster_sync_all();
  else
    __syncthreads();
  const int share = kShrinkRows / parts;  // rows that this CTA finishes
  if constexpr (kScaled) {
    // The totals replace this CTA's sums in the rows that it alone finishes (a warp's 32
    // quads lie in one block of 16 rows), then they are scaled and split.
    constexpr int kLanes = RP / 4;  // of a row
    for (int e = tid; e < share * kLanes; e += kThreads) {
      const int m = part * share + e / kLanes, j = e % kLanes * 4;
      uint32_t top = 0;
      if (m < t.rows && j < r) {
        const float4 v = cluster_sum4(sums + m * kPitch + j, parts);
        *reinterpret_cast<float4*>(sums + m * kPitch + j) = v;
        top = finite_abs(v);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) atomicMax(&largest[m / 16], top);
    }
    __syncthreads();
    const int first = offs[t.i], block0 = first / 16 + t.i + (t.p0 - first) / 16;
    for (int e = tid; e < share * kLanes; e += kThreads) {
      const int m = part * share + e / kLanes, j = e % kLanes * 4;
      const bool there = m < t.rows && j < r;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (there) v = *reinterpret_cast<const float4*>(sums + m * kPitch + j);
      const float4 op = make_float4(c * v.x, c * v.y, c * v.z, c * v.w);
      uint32_t top = there ? finite_abs(op) : 0u;  // the row's largest
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const bool fits = top == 0 || (top >= __float_as_uint(0x1p-14f) && top <= __float_as_uint(65504.0f));
      if (!there) continue;
      const int x2 = exp_of(largest[m / 16]);
      const float f = x2 == kNoExp ? 1.0f : exp2i(-x2);
      T hi[4], lo[4];
      split(v.x * f, hi, lo), split(v.y * f, hi + 1, lo + 1), split(v.z * f, hi + 2, lo + 2);
      split(v.w * f, hi + 3, lo + 3);
      T* out = s + int64_t(t.p0 + m) * r + j;
      *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(hi);
      *reinterpret_cast<uint2*>(out + part_stride) = *reinterpret_cast<const uint2*>(lo);
      const int row = row_of[m];
      if (row >= 0) {
        T o[4] = {from_f<T>(op.x), from_f<T>(op.y), from_f<T>(op.z), from_f<T>(op.w)};
        if (!fits) o[0] = o[1] = o[2] = o[3] = from_f<T>(0.0f);
        *reinterpret_cast<uint2*>(rows + int64_t(row) * r + j) = *reinterpret_cast<const uint2*>(o);
      }
      if (j == 0) {
        range.put[t.p0 + m] = row >= 0 && fits;
        if (row >= 0 && !fits) *range.left = 1;  // (every writer the same)
        if (m % 16 == 0) range.exps[block0 + m / 16] = x2;
      }
    }
  } else {
    for (int e = tid; e < share * (RP / 4); e += kThreads) {
      const int m = part * share + e / (RP / 4), j = e % (RP / 4) * 4;
      if (m >= t.rows || j >= r) continue;
      const float4 v = cluster_sum4(sums + m * kPitch + j, parts);
      T hi[4], lo[4];
      split(v.x, hi, lo), split(v.y, hi + 1, lo + 1), split(v.z, hi + 2, lo + 2), split(v.w, hi + 3, lo + 3);
      T* out = s + int64_t(t.p0 + m) * r + j;
      *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(hi);
      *reinterpret_cast<uint2*>(out + part_stride) = *reinterpret_cast<const uint2*>(lo);
      const int row = row_of[m];
      if (row >= 0) {
        const T o[4] = {from_f<T>(c * v.x), from_f<T>(c * v.y), from_f<T>(c * v.z), from_f<T>(c * v.w)};
        *reinterpret_cast<uint2*>(rows + int64_t(row) * r + j) = *reinterpret_cast<const uint2*>(o);
      }
    }
  }
  if (parts > 1) cluster_sync_all();  // no CTA leaves while another reads its sums
}

// expand.  A CTA holds 64 rows of s in registers (both parts) and runs over blocks of
// 128 columns: 4 groups of 16 rows x 2 halves of 64 columns, one per warp.  Bound by
// reading and writing y; y's 16-byte pieces and w's rows of the next block are loaded
// under the products of this one.  For w in rows of n the columns are placed so that a
// lane's results of 4 column tiles are 8 neighbours; read along n they go through a
// patch of shared memory for that.  Measured 114 us for 16384 rows of 8192 at rank 64
// (537 MB, 4.7 TB/s); 3 us when the shared product has taken every row.
constexpr int kExpandRows = 64;
constexpr int kExpandCols = 128;
constexpr int kPatchPitch = 36;  // floats

template <bool kT, int RP>
struct ExpandCfg {
  static constexpr int kW = kT ? RP * (kExpandCols * 2 + 16) : kExpandCols * (RP * 2 + 16);
  static constexpr int kPatch = kT ? 8 * 16 * kPatchPitch * 4 : 0;
  static constexpr int kBytes = 2 * kW + kPatch;
};

template <typename T, bool kT, int RP>
__global__ void __launch_bounds__(kThreads, 2)
    expand_kernel(const T* s, int64_t part_stride, const T* w, int64_t sl, int64_t sr,
                  Scale scale, const int32_t* perm, const int32_t* offs, const int32_t* taken, Range range,
                  const TileAdapters* tile, int tiles, int splits, int L, int N, int r, T* y, int64_t ldy) {
  using C = ExpandCfg<kT, RP>;
  extern __shared__ __align__(128) char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, q4 = lane & 3;
  wait_for_previous_kernel();
  let_next_kernel_start();
  // Usually the shared product has taken every row.
  constexpr bool kScaled = std::is_same<T, __half>::value;
  bool any = kScaled && *range.left != 0;
  for (int q = tid; q < tiles; q += kThreads) any |= tile[q].left != 0;
  if (!__syncthreads_or(any)) return;
  const int mg = warp & 3, half = warp >> 2;
  for (int unit = blockIdx.x;; unit += gridDim.x) {
  const Tile t = find_tile(offs, L, unit / splits, kExpandRows);
  if (t.i < 0) return;
  const int first = unit % splits * kExpandCols;
  const float c = scale.of(t.i);
  float cu[2] = {c, c};
  if constexpr (kScaled) {  // these 16 rows' power of two
    const int o0 = offs[t.i], o = t.p0 - o0 + mg * 16;
    const int x2 = mg * 16 < t.rows ? range.exps[o0 / 16 + t.i + o / 16] : kNoExp;
    if (x2 != kNoExp) cu[0] = cu[1] = c * exp2i(x2);
  }
  T* yrow[2];  // rows mg*16 + g8 and + 8; null for those that the shared product has taken
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int m = mg * 16 + g8 + 8 * u, row = m < t.rows ? perm[t.p0 + m] : -1;
    const bool done = row >= 0 && (kScaled ? range.put[t.p0 + m] : taken[row]) != 0;
    yrow[u] = row >= 0 && !done ? y + row * ldy + half * 64 + q4 * 8 : nullptr;
  }
  if (!__syncthreads_or(yrow[0] != nullptr || yrow[1] != nullptr)) continue;
  const T* wi = w + t.i * sl;
  const int step = splits * kExpandCols;
  auto fetch_w = [&](int n0, int buf) {
    if (n0 < N) {
      const uint32_t ws = smem_u32(smem) + buf * C::kW;
      constexpr int kPieces = RP * kExpandCols / 8 / kThreads;
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        const int e = tid + q * kThreads;
        if constexpr (kT) {
          const int j = e / (kExpandCols / 8), n = e % (kExpandCols / 8) * 8;
          const bool in = j < r && n0 + n < N;
          copy_async_16(ws + j * (kExpandCols * 2 + 16) + n * 2, in ? wi + j * sr + n0 + n : w, in);
        } else {
          const int n = e / (RP / 8), j = e % (RP / 8) * 8;
          // column 8 q + 2 t + o of a group of 32 goes to row 8 t + 2 q + o
          const int at = (n & ~31) + ((n >> 1) & 3) * 8 + ((n >> 3) & 3) * 2 + (n & 1);
          const bool in = j < r && n0 + n < N;
          copy_async_16(ws + at * (RP * 2 + 16) + j * 2, in ? wi + (n0 + n) * sr + j : w, in);
        }
      }
    }
    copies_commit();
  };
  fetch_w(first, 0);
  const int ncol = half * 64 + q4 * 8;  // this lane's first column of a block; + 32 for the second
  auto fetch_y = [&](int n0, uint4(&v)[2][2]) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (yrow[u] != nullptr && n0 + ncol + g * 32 < N)
          v[g][u] = *reinterpret_cast<const uint4*>(yrow[u] + n0 + g * 32);
  };
  uint4 yv[2][2], yn[2][2];
  fetch_y(first, yv);
  // A fragments straight from s: rows mg*16 + g8 and + 8, pairs of columns.
  uint32_t a[2][RP / 16][4];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int m = mg * 16 + g8 + 8 * u;
#pragma unroll
    for (int k = 0; k < RP / 16; ++k)
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int j = k * 16 + v * 8 + q4 * 2;
        const bool in = m < t.rows && j < r;
        const T* at = s + int64_t(t.p0 + m) * r + j;
        a[0][k][u + 2 * v] = in ? *reinterpret_cast<const uint32_t*>(at) : 0u;
        a[1][k][u + 2 * v] = in ? *reinterpret_cast<const uint32_t*>(at + part_stride) : 0u;
      }
  }
  int buf = 0;
  for (int n0 = first; n0 < N; n0 += step) {
    fetch_w(n0 + step, buf ^ 1);
    fetch_y(n0 + step, yn);
    copies_wait<1>();
    __syncthreads();
    const uint32_t ws = smem_u32(smem) + buf * C::kW;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float acc[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[n][q] = 0.0f;
      const int col = half * 64 + g * 32;
#pragma unroll
      for (int k = 0; k < RP / 16; ++k)
#pragma unroll
        for (int n = 0; n < 4; n += 2) {
          uint32_t b[4];
          if constexpr (kT)
            ldmatrix_x4<true>(b, ws + (k * 16 + (lane & 15)) * (kExpandCols * 2 + 16) +
                                     (col + (n + (lane >> 4)) * 8) * 2);
          else
            ldmatrix_x4<false>(b, ws + (col + n * 8 + (lane >> 4) * 8 + (lane & 7)) * (RP * 2 + 16) +
                                      (k * 16 + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            mma<T>(acc[n], a[part][k], b[0], b[1]);
            mma<T>(acc[n + 1], a[part][k], b[2], b[3]);
          }
        }
      float add[2][8];  // this lane's 8 neighbouring columns of its two rows
      if constexpr (kT) {
        float* patch = reinterpret_cast<float*>(smem + 2 * C::kW) + warp * 16 * kPatchPitch;
        __syncwarp();
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            *reinterpret_cast<float2*>(patch + (g8 + 8 * u) * kPatchPitch + n * 8 + q4 * 2) =
                make_float2(acc[n][2 * u], acc[n][2 * u + 1]);
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int v = 0; v < 2; ++v)
            *reinterpret_cast<float4*>(&add[u][4 * v]) =
                *reinterpret_cast<const float4*>(patch + (g8 + 8 * u) * kPatchPitch + q4 * 8 + 4 * v);
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q) add[q >> 1][2 * n + (q & 1)] = acc[n][q];
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (yrow[u] == nullptr || n0 + ncol + g * 32 >= N) continue;
        T* v = reinterpret_cast<T*>(&yv[g][u]);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = from_f<T>(to_f(v[q]) + cu[u] * add[u][q]);
        *reinterpret_cast<uint4*>(yrow[u] + n0 + g * 32) = yv[g][u];
      }
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int u = 0; u < 2; ++u) yv[g][u] = yn[g][u];
    buf ^= 1;
  }
  copies_wait<0>();
  }
}

// grads.  A CTA forms 128 MT columns of z x RP of one adapter's gradient over one part
// of its rows, 32 at a time: z^T by ldmatrix.trans as the 16-row side, s as the
// 8-column side.  The CTAs of a cluster take the parts of the rows and add their sums
// through distributed shared memory, in order.  Bound by reading z once, at rank 64 by the
// products of both parts of s as well: measured 175 us for dA [8, 64, 2048] and dB [8, 8192,
// 64] of 16384 rows (335 MB).
constexpr int kGradRows = 32;

template <int RP>
struct GradCfg {
  static constexpr int MT = RP == 128 ? 1 : 2;  // 16-column tiles of z a warp
  static constexpr int kCols = 128 * MT;
  static constexpr int kZPitch = kCols * 2 + 16, kSPitch = RP * 2 + 16;
  static constexpr int kStage = kGradRows * (kZPitch + 2 * kSPitch);
  static constexpr int kStages = 4;
  static constexpr int kSums = (kCols + 4) * (RP + 4) * 4;
  static constexpr int kBytes = kStages * kStage > kSums ? kStages * kStage : kSums;
};

// One gradient: of rows z [m, n] and the low-rank rows s, into g of [n, rank] for each
// adapter, or [rank, n].
template <typename T>
struct GradOf {
  const T *s, *z;
  int64_t ldz;
  int n;
  T* g;
  const int32_t* exps;  // fp16: s's powers of two
};

template <typename T, bool kT, int RP>
__device__ __forceinline__ void grad_block(char* smem, const GradOf<T>& of, int block, int parts, int64_t part_stride,
                                           Scale scale, const int32_t* perm, const int32_t* offs, int r) {
  using C = GradCfg<RP>;
  constexpr int MT = C::MT;
  const T *s = of.s, *z = of.z;
  const int64_t ldz = of.ldz, gl = int64_t(of.n) * r, gr = kT ? of.n : r;
  const int n = of.n;
  T* g = of.g;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int part = blockIdx.x % parts, n0 = block * C::kCols, i = blockIdx.y;
  const int o0 = offs[i], rows = offs[i + 1] - o0;
  const int share = ((rows + parts - 1) / parts + kGradRows - 1) / kGradRows * kGradRows;
  const int p0 = min(rows, part * share), p1 = min(rows, p0 + share);
  const int steps = (p1 - p0 + kGradRows - 1) / kGradRows;
  constexpr int kPieces = C::kCols / 8;  // 16-byte pieces of a row of z
  constexpr int kCopies = kGradRows * kPieces / kThreads;
  const int zc = tid % kPieces * 8;
  int next_row[kCopies];  // perm's entries for the next fetch: known before they are used
  auto look_up = [&](int step) {
#pragma unroll
    for (int q = 0; q < kCopies; ++q) {
      const int p = p0 + step * kGradRows + tid / kPieces + q * (kThreads / kPieces);
      next_row[q] = p < p1 && n0 + zc < n ? perm[o0 + p] : -1;
    }
  };
  look_up(0);
  // s: pieces of both parts, at pointers that move on by 32 rows.
  constexpr int kSPieces = RP / 8, kSCopies = (2 * kGradRows * kSPieces + kThreads - 1) / kThreads;
  const T* sp[kSCopies];
#pragma unroll
  for (int q = 0; q < kSCopies; ++q) {
    const int e = tid + q * kThreads, half = e / (kGradRows * kSPieces), f = e % (kGradRows * kSPieces);
    const int j = f % kSPieces * 8;
    sp[q] = s + (j < r && half < 2 ? half * part_stride + int64_t(o0 + p0 + f / kSPieces) * r + j : 0);
  }
  // fp16: the powers of two of a step's two blocks of 16 rows, known a step ahead.  The sums
  // are held divided by the last block's, `unit`: a block with another one changes it in all
  // of them first, which is exact and seldom (multiples of 8), and loses nothing of small
  // rows behind large ones.
  constexpr bool kScaled = std::is_same<T, __half>::value;
  [[maybe_unused]] int unit = kNoExp, next_exp[2] = {kNoExp, kNoExp};
  auto look_up_exps = [&](int step) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int o = p0 + step * kGradRows + 16 * q;
      next_exp[q] = o < p1 ? of.exps[o0 / 16 + i + o / 16] : kNoExp;
    }
  };
  if constexpr (kScaled) look_up_exps(0);
  int step_f = 0, at = 0;  // the step and the stage of the next fetch
  auto fetch = [&]() {
    if (step_f < steps) {
      const uint32_t zs = smem_u32(smem) + at * C::kStage;
      const uint32_t ss = zs + kGradRows * C::kZPitch;
      const int p = p0 + step_f * kGradRows;
#pragma unroll
      for (int q = 0; q < kCopies; ++q) {
        const int m = tid / kPieces + q * (kThreads / kPieces);
        const bool in = next_row[q] >= 0;
        copy_async_16(zs + m * C::kZPitch + zc * 2, z + (in ? next_row[q] * ldz + n0 + zc : 0), in);
      }
      ++step_f;
      look_up(step_f);
#pragma unroll
      for (int q = 0; q < kSCopies; ++q) {
        const int e = tid + q * kThreads, half = e / (kGradRows * kSPieces), f = e % (kGradRows * kSPieces);
        const int m = f / kSPieces, j = f % kSPieces;
        const bool in = p + m < p1 && j * 8 < r;
        if (half < 2) copy_async_16(ss + (half * kGradRows + m) * C::kSPitch + j * 16, sp[q], in);
        sp[q] += kGradRows * r;
      }
      if (++at == C::kStages) at = 0;
    }
    copies_commit();
  };
  float acc[MT][RP / 8][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int k = 0; k < RP / 8; ++k)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[m][k][q] = 0.0f;
#pragma unroll
  for (int q = 0; q < C::kStages - 1; ++q) fetch();
  for (int step = 0, stage = 0; step < steps; ++step, stage = stage + 1 == C::kStages ? 0 : stage + 1) {
    copies_wait<C::kStages - 2>();
    __syncthreads();
    fetch();
    const uint32_t zs = smem_u32(smem) + stage * C::kStage;
    const uint32_t ss = zs + kGradRows * C::kZPitch;
    [[maybe_unused]] const int exps[2] = {next_exp[0], next_exp[1]};
    if constexpr (kScaled) look_up_exps(step + 1);
#pragma unroll
    for (int kk = 0; kk < kGradRows; kk += 16) {
      if constexpr (kScaled) {
        const int x2 = exps[kk / 16];
        if (x2 != unit && x2 != kNoExp) {
          if (unit != kNoExp) {
            const float f = exp2i(unit - x2);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int k = 0; k < RP / 8; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[m][k][q] *= f;
          }
          unit = x2;
        }
      }
      uint32_t a[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
        ldmatrix_x4<true>(a[m], zs + (kk + (lane & 7) + (lane >> 4) * 8) * C::kZPitch +
                                    ((warp * MT + m) * 16 + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
      for (int k = 0; k < RP / 8; k += 2)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t b[4];
          ldmatrix_x4<true>(b, ss + (half * kGradRows + kk + (lane & 15)) * C::kSPitch +
                                   (k + (lane >> 4)) * 16);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma<T>(acc[m][k], a[m], b[0], b[1]);
            mma<T>(acc[m][k + 1], a[m], b[2], b[3]);
          }
        }
    }
  }
  copies_wait<0>();
  __syncthreads();
  // The sums lie as the gradient does: [column][rank], or [rank][column] with kT.
  constexpr int kPitch = kT ? C::kCols + 4 : RP + 4;
  float* sums = reinterpret_cast<float*>(smem);
  const float f = kScaled && unit != kNoExp ? exp2i(unit) : 1.0f;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int k = 0; k < RP / 8; ++k)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = (warp * MT + m) * 16 + (lane >> 2) + 8 * (q >> 1), j = k * 8 + (lane & 3) * 2 + (q & 1);
        sums[kT ? j * kPitch + col : col * kPitch + j] = f * acc[m][k][q];
      }
  if (parts > 1)
    cluster_sync_all();
  else
    __syncthreads();
  const float c = scale.of(i);
  // Four neighbours of a row at a time; the CTAs take the rows in turn.
  constexpr int kRows = kT ? RP : C::kCols, kQuads = (kT ? C::kCols : RP) / 4;
  for (int e = tid; e < kRows / parts * kQuads; e += kThreads) {
    const int row = e / kQuads * parts + part, at = e % kQuads * 4;
    if (kT ? row >= r || n0 + at >= n : n0 + row >= n || at >= r) continue;
    const float4 v = cluster_sum4(sums + row * kPitch + at, parts);
    const T o[4] = {from_f<T>(c * v.x), from_f<T>(c * v.y), from_f<T>(c * v.z), from_f<T>(c * v.w)};
    T* out = g + i * gl + (kT ? row * gr + n0 + at : (n0 + row) * gr + at);
    *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(o);
  }
  if (parts > 1) cluster_sync_all();
}

// dA and dB in one launch: the first blocks_a blocks of columns are dA's.  Blocks and their
// parts share the grid's x, the one direction that takes any number of them.
template <typename T, int RP>
__global__ void __launch_bounds__(kThreads, 2)
    grad_kernel(GradOf<T> a, GradOf<T> b, int blocks_a, int parts, int64_t part_stride, Scale scale,
                const int32_t* perm, const int32_t* offs, int r, int32_t* queue) {
  extern __shared__ __align__(128) char smem[];
  wait_for_previous_kernel();
  let_next_kernel_start();
  const int block = blockIdx.x / parts;
  // the shared product before is done with its counter: 0 again for another pass
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *queue = 0;
  if (block < blocks_a)
    grad_block<T, true, RP>(smem, a, block, parts, part_stride, scale, perm, offs, r);
  else
    grad_block<T, false, RP>(smem, b, block - blocks_a, parts, part_stride, scale, perm, offs, r);
}

template <auto kern, typename... A>
int launch(dim3 grid, dim3 cluster, int smem, cudaStream_t stream, A... args) {
  if (!allow_shared_memory<kern>(smem)) return MOE_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  // Set up beside the kernel before.  Each waits for that one's end and only then lets
  // the next start, so that a kernel starts with all but its predecessor complete (the
  // shared product relies on it).
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster.x;
  attr[1].val.clusterDim.y = cluster.y;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster.x * cluster.y > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

// Calls fn(T(), transposed, RP) with the compile-time values for this call.
template <typename Fn>
int dispatch(int dtype, bool transposed, int rank, Fn fn) {
  auto by_rank = [&](auto t, auto tr) {
    if (rank <= 16) return fn(t, tr, std::integral_constant<int, 16>());
    if (rank <= 32) return fn(t, tr, std::integral_constant<int, 32>());
    if (rank <= 64) return fn(t, tr, std::integral_constant<int, 64>());
    return fn(t, tr, std::integral_constant<int, 128>());
  };
  auto by_layout = [&](auto t) {
    return transposed ? by_rank(t, std::true_type()) : by_rank(t, std::false_type());
  };
  return dtype == MOE_DTYPE_BF16 ? by_layout(__nv_bfloat16()) : by_layout(__half());
}

// The most blocks of `tile` rows that m rows of `adapters` adapters can make.
inline int64_t most_tiles(int64_t m, int adapters, int tile) {
  const int64_t t = (m + tile - 1) / tile + adapters;
  return t < m ? t : m;
}
// A power of two up to 8 that keeps blocks * parts at most `most` and gives each part
// at least `least` of `length`.
inline int cluster_parts(int64_t blocks, int64_t most, int64_t length, int64_t least) {
  int parts = 1;
  while (parts < 8 && blocks * parts * 2 <= most && length / (parts * 2) >= least) parts *= 2;
  return parts;
}

// The current device's SMs, for the rules below.
inline int device_sms(int* sms) {
  int dev;
  DeviceInfo info;
  const int rc = current_device_info(&dev, &info);
  if (rc == MOE_OK) *sms = info.sm_count;
  return rc;
}

// s = x w^T by adapter, w in rows of k (transposed: in rows of the rank); scale s also
// by row, for the shared product.
int shrink(const void* x, int64_t ldx, Weights w, bool transposed, Scale scale, const PlanView& plan, int dtype,
           int64_t m, int64_t k, int adapters, int rank, void* s, void* rows, int32_t* exps,
           cudaStream_t stream) {
  int sms;
  if (const int rc = device_sms(&sms); rc != MOE_OK) return rc;
  return dispatch(dtype, transposed, rank, [&](auto t, auto tr, auto rp) {
    using T = decltype(t);
    constexpr bool kT = decltype(tr)::value;
    constexpr int RP = decltype(rp)::value;
    const unsigned tiles = static_cast<unsigned>(most_tiles(m, adapters, kShrinkRows));
    // Few rows leave half of the SMs to the shared product, which starts at once on those
    // (4096 rows of 2048 x 2048, a step: 104.8 us, and 111.5 with all SMs taken); many take
    // two CTAs an SM (16384 rows: 1048 us, and 1098 with one part).
    const unsigned parts = cluster_parts(tiles, int(tiles) <= sms / 2 ? sms / 2 : 2 * sms, k, 256);
    return launch<&shrink_kernel<T, kT, RP>>(dim3(tiles, parts), dim3(1, parts),
                  ShrinkCfg<kT, RP>::kBytes, stream, static_cast<const T*>(x), ldx,
                  static_cast<const T*>(w.p), w.stride_l, w.stride_row, plan.perm, plan.offs, adapters,
                  static_cast<int>(k), rank, m * rank, static_cast<T*>(s), scale, plan.taken,
                  static_cast<T*>(rows), Range{exps, plan.put, plan.left});
  });
}

// y += scale s w^T for the rows that the shared product has left, w in rows of the rank
// (transposed: in rows of n).
int expand(const void* s, Weights w, bool transposed, Scale scale, const PlanView& plan, int dtype,
           int64_t m, int64_t n, int adapters, int rank, int32_t* exps, void* y, int64_t ldy,
           cudaStream_t stream) {
  int sms;
  if (const int rc = device_sms(&sms); rc != MOE_OK) return rc;
  return dispatch(dtype, transposed, rank, [&](auto t, auto tr, auto rp) {
    using T = decltype(t);
    constexpr bool kT = decltype(tr)::value;
    constexpr int RP = decltype(rp)::value;
    const int64_t blocks = (n + kExpandCols - 1) / kExpandCols;
    // Two CTAs an SM; work for about four times as many, if every row were left.
    const int64_t places = 2 * sms, tiles = most_tiles(m, adapters, kExpandRows);
    const int64_t want = (4 * places + tiles - 1) / tiles;
    const int splits = static_cast<int>(want < blocks ? want : blocks);
    const int64_t units = tiles * splits;
    return launch<&expand_kernel<T, kT, RP>>(dim3(static_cast<unsigned>(units < places ? units : places)),
                  dim3(1, 1), ExpandCfg<kT, RP>::kBytes, stream, static_cast<const T*>(s),
                  m * rank, static_cast<const T*>(w.p), w.stride_l, w.stride_row, scale, plan.perm,
                  plan.offs, plan.taken, Range{exps, plan.put, plan.left}, plan.tile, static_cast<int>(PlanView::tiles(m)), splits, adapters,
                  static_cast<int>(n), rank, static_cast<T*>(y), ldy);
  });
}

// da [adapters, rank, k] = scale t^T x and db [adapters, n, rank] = scale dy^T s by
// adapter; a null one is not formed.
int grads(const void* t, const void* x, int64_t ldx, int64_t k, void* da, const void* s, const void* dy,
          int64_t lddy, int64_t n, void* db, Scale scale, const PlanView& plan, int dtype, int64_t m,
          int adapters, int rank, cudaStream_t stream) {
  int sms;
  if (const int rc = device_sms(&sms); rc != MOE_OK) return rc;
  return dispatch(dtype, false, rank, [&](auto tt, auto, auto rp) {
    using T = decltype(tt);
    constexpr int RP = decltype(rp)::value;
    using C = GradCfg<RP>;
    const int blocks_a = da != nullptr ? static_cast<int>((k + C::kCols - 1) / C::kCols) : 0;
    const int blocks = blocks_a + (db != nullptr ? static_cast<int>((n + C::kCols - 1) / C::kCols) : 0);
    // Parts of an adapter's rows, as many as leave about four CTAs for each of the two places on
    // an SM, since adapters' rows are uneven.  The rule knows the adapters' average only: where
    // many columns and adapters leave one part, a single adapter with most of the rows is
    // summed by its column blocks alone.
    const unsigned parts = cluster_parts(int64_t(blocks) * adapters, 4 * 2 * sms, m / adapters, 64);
    const GradOf<T> a{static_cast<const T*>(t), static_cast<const T*>(x), ldx, static_cast<int>(k),
                      static_cast<T*>(da), plan.exps[1]};
    const GradOf<T> b{static_cast<const T*>(s), static_cast<const T*>(dy), lddy, static_cast<int>(n),
                      static_cast<T*>(db), plan.exps[0]};
    return launch<&grad_kernel<T, RP>>(dim3(parts * static_cast<unsigned>(blocks), adapters), dim3(parts, 1),
                                       C::kBytes, stream, a, b, blocks_a, static_cast<int>(parts), m * rank, scale,
                                       static_cast<const int32_t*>(plan.perm),
                                       static_cast<const int32_t*>(plan.offs), rank, plan.queue + 1);
  });
}

}  // namespace lora
}  // namespace moe

using namespace moe;

namespace {
bool dims_ok(int32_t dtype, int64_t m, int64_t k, int64_t n, int32_t adapters, int32_t rank) {
  const int64_t most = INT32_MAX / 2;
  return (dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16) && m >= 0 && m <= most && k >= 8 &&
         k % 8 == 0 && k <= most && n >= 8 && n % 8 == 0 && n <= most && adapters >= 1 &&
         adapters <= lora::kMaxAdapters && rank >= 8 && rank % 8 == 0 && rank <= lora::kMaxRank;
}
// Rows of `width` at 16-byte starts; of several adapters, one behind another.
bool rows_ok(const void* p, int64_t ld, int64_t width) {
  return p != nullptr && aligned16(p) && ld >= width && ld % 8 == 0;
}
bool weights_ok(lora::Weights w, int64_t rows, int64_t width, int32_t adapters) {
  return rows_ok(w.p, w.stride_row, width) &&
         (adapters == 1 || (w.stride_l % 8 == 0 && w.stride_l >= (rows - 1) * w.stride_row + width));
}
// y = x w^T, w(k, n) at the given strides, with the adapters' second product of the rows
// that it takes.
int shared_product(const void* x, int64_t ldx, const void* w, int64_t stride_k, int64_t stride_n, void* y,
                   int64_t ldy, const lora::PlanView& plan, lora::Weights second, const void* rows,
                   int64_t m, int64_t k, int64_t n, int adapters, int rank, int dtype, int32_t* queue,
                   int32_t* status, cudaStream_t stream) {
  int dev;
  DeviceInfo info;
  const int rc = current_device_info(&dev, &info);
  if (rc != MOE_OK) return rc;
  const gg::Adapters extra{rows, plan.tile, second.p, second.stride_l, second.stride_row, rank, adapters};
  return gg::grouped_gemm_launch(x, ldx, w, 0, stride_k, stride_n, y, ldy, plan.base, 0, m, k, n, 1, dtype,
                                 MOE_ACT_NONE, info.sm_count, queue != nullptr, queue, nullptr, nullptr, nullptr, 0, status,
                                 stream, nullptr, nullptr, force_single_sm_kernel() ? nullptr : &extra);
}
// Adapters that the shared product takes in a tile of rows; none on the 1-SM kernel.
int per_tile(int rank) { return force_single_sm_kernel() ? 0 : gg::Adapters::most(rank); }
// Whether expand may have rows to do: of tiles with more adapters than that, or, with fp16,
// out of the type's range.
bool may_leave_rows(int adapters, int rank, int dtype) {
  return adapters > per_tile(rank) || dtype == MOE_DTYPE_F16;
}
int64_t low_bytes(int64_t m, int32_t rank) { return 4 * m * rank; }
// The caller's buffer: x A^T by adapter and dy B by adapter (two parts each), the shared
// product's operand by row, the plan.
struct Buffers {
  char *s, *t, *rows, *plan;
  int64_t bytes;
  Buffers(void* kept, int64_t m, int32_t adapters, int32_t rank) {
    const int64_t low = low_bytes(m, rank);
    s = static_cast<char*>(kept);
    t = s + low;
    rows = t + low;
    plan = rows + low / 2;
    bytes = 2 * low + low / 2 + 4 * lora::PlanView::ints(m, adapters);
  }
};
}  // namespace

extern "C" int64_t moe_lora_kept_bytes(int64_t m, int32_t adapters, int32_t rank) {
  if (!dims_ok(MOE_DTYPE_BF16, m, 8, 8, adapters, rank)) return -1;
  return Buffers(nullptr, m, adapters, rank).bytes;
}

extern "C" int32_t moe_lora_forward(const void* x, int64_t ldx, const void* weight, int64_t ldw,
                                    const void* lora_a, int64_t a_stride_l, int64_t a_stride_row,
                                    const void* lora_b, int64_t b_stride_l, int64_t b_stride_row,
                                    const void* ids, int32_t ids_int64, const float* scale,
                                    float scale_all, int32_t dtype, int64_t m, int64_t k, int64_t n,
                                    int32_t adapters, int32_t rank, int32_t for_backward, void* y,
                                    int64_t ldy, void* kept, int32_t* status, void* stream) {
  const lora::Weights a{lora_a, a_stride_l, a_stride_row}, b{lora_b, b_stride_l, b_stride_row};
  if (!dims_ok(dtype, m, k, n, adapters, rank) || kept == nullptr || !aligned16(kept) ||
      !rows_ok(weight, ldw, k) || !weights_ok(a, rank, k, adapters) || !weights_ok(b, n, rank, adapters) ||
      (m > 0 && (!rows_ok(x, ldx, k) || !rows_ok(y, ldy, n) || ids == nullptr)))
    return MOE_ERR_INVALID_ARG;
  const lora::Scale sc{scale, scale_all};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int sms = 0;
  if (m > 0)
    if (const int rc = lora::device_sms(&sms); rc != MOE_OK) return rc;
  if (!for_backward && m > 0 && lora::takes_few_rows(m, k, n, rank, sms))
    return lora::forward_few_rows(x, ldx, weight, ldw, a, b, ids, ids_int64, sc, dtype,
                                  static_cast<int>(m), static_cast<int>(k), static_cast<int>(n), adapters,
                                  rank, y, ldy, static_cast<float*>(kept), status, st);
  const Buffers buf(kept, m, adapters, rank);
  const lora::PlanView plan(buf.plan, m, adapters);
  lora::plan_kernel<<<static_cast<unsigned>(adapters + lora::PlanView::tiles(m)), 1024, 0, st>>>(
      ids, ids_int64, static_cast<int>(m), adapters, plan, per_tile(rank), status);
  if (cudaGetLastError() != cudaSuccess) return MOE_ERR_CUDA;
  if (m == 0) return MOE_OK;
  int rc = lora::shrink(x, ldx, a, false, sc, plan, dtype, m, k, adapters, rank, buf.s, buf.rows, plan.exps[0], st);
  if (rc == MOE_OK)
    rc = shared_product(x, ldx, weight, 1, ldw, y, ldy, plan, b, buf.rows, m, k, n, adapters, rank, dtype, plan.queue,
                        status, st);
  if (rc == MOE_OK && may_leave_rows(adapters, rank, dtype))
    rc = lora::expand(buf.s, b, false, sc, plan, dtype, m, n, adapters, rank, plan.exps[0], y, ldy, st);
  return rc;
}

extern "C" int32_t moe_lora_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                     const void* weight, int64_t ldw, const void* lora_a,
                                     int64_t a_stride_l, int64_t a_stride_row, const void* lora_b,
                                     int64_t b_stride_l, int64_t b_stride_row, const float* scale,
                                     float scale_all, int32_t dtype, int64_t m, int64_t k, int64_t n,
                                     int32_t adapters, int32_t rank, void* kept, void* dx, int64_t lddx,
                                     void* da, void* db, int32_t* status, void* stream) {
  const lora::Weights a{lora_a, a_stride_l, a_stride_row}, b{lora_b, b_stride_l, b_stride_row};
  if (!dims_ok(dtype, m, k, n, adapters, rank) || kept == nullptr || !aligned16(kept) ||
      !rows_ok(weight, ldw, k) || !weights_ok(a, rank, k, adapters) || !weights_ok(b, n, rank, adapters) ||
      (da != nullptr && !aligned16(da)) || (db != nullptr && !aligned16(db)) ||
      (m > 0 && (!rows_ok(dy, lddy, n) || !rows_ok(x, ldx, k) || (dx != nullptr && !rows_ok(dx, lddx, k)))))
    return MOE_ERR_INVALID_ARG;
  const Buffers buf(kept, m, adapters, rank);
  const lora::PlanView plan(buf.plan, m, adapters);
  const lora::Scale sc{scale, scale_all};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = MOE_OK;
  if (m > 0 && (dx != nullptr || da != nullptr))
    rc = lora::shrink(dy, lddy, b, true, sc, plan, dtype, m, n, adapters, rank, buf.t, buf.rows, plan.exps[1], st);
  if (rc == MOE_OK && m > 0 && dx != nullptr) {
    rc = shared_product(dy, lddy, weight, ldw, 1, dx, lddx, plan, a, buf.rows, m, n, k, adapters, rank, dtype,
                        da != nullptr || db != nullptr ? plan.queue + 1 : nullptr, status, st);
    if (rc == MOE_OK && may_leave_rows(adapters, rank, dtype))
      rc = lora::expand(buf.t, a, true, sc, plan, dtype, m, k, adapters, rank, plan.exps[1], dx, lddx, st);
  }
  if (rc == MOE_OK && (da != nullptr || db != nullptr))
    rc = lora::grads(buf.t, x, ldx, k, da, buf.s, dy, lddy, n, db, sc, plan, dtype, m, adapters, rank, st);
  return rc;
}
