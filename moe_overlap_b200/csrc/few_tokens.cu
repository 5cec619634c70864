// The routed-experts layer for a few tokens on sm_100a: gate, top-k, up-projection
// with exact GELU, down-projection and weighted sum.
//
//   z = x Wg^T + bias;  p = softmax(z);  idx = the k largest z (ties: lower id);
//   w = p[idx] (/ their sum);
//   h[t,j] = gelu(x[t] W1[idx]^T);  out[t] = sum_j w[t,j] (h[t,j] W2[idx]^T)
//
// (the routed path of src/train_moe_baseline.py:315-441 at decode batch sizes).
// A slot with expert -1 adds nothing; a token without any expert gets zeros.
// Sums are fp32 (the gate's fp64); h is held as two values of the input type, the rounded
// one and what the rounding left, since it is the operand of a second tensor-core product:
// 16 bits of bf16; of fp16 22 bits, but not below 2^-25, and up to 131008 (an fp16 h of its
// own ends at 65504).  The output is rounded once.
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/moe_overlap.h"
#include "host_common.h"
#include "mma16.cuh"
#include "ptx.cuh"

namespace moe {
namespace few {

constexpr int kMaxTokens = 128;
constexpr int kMaxWidth = 1 << 30;  // of hidden and ffn: a column and a stage behind it fit in an int
constexpr int kMaxE = 256;
constexpr int kMaxK = 16;
constexpr int kWarps = 8;

// Dot product of two rows of `n` elements (a multiple of 8, 16-byte aligned) over one
// warp.  A product of two bf16 or fp16 values is exact in fp32 (of bf16 within fp32's
// range); the sum is fp64.
template <typename T>
__device__ __forceinline__ double warp_dot(const T* a, const T* b, int n, int lane) {
  double s = 0;
#pragma unroll 4
  for (int i = lane * 8; i < n; i += 256) {
    const uint4 ua = *reinterpret_cast<const uint4*>(a + i);
    const uint4 ub = *reinterpret_cast<const uint4*>(b + i);
    const T* pa = reinterpret_cast<const T*>(&ua);
    const T* pb = reinterpret_cast<const T*>(&ub);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += static_cast<double>(to_f(pa[j]) * to_f(pb[j]));
  }
  return warp_sum(s);
}

// The k largest of a token's E logits (fp64, in shared memory) by one warp, in
// descending order with ties to the lower id, and their softmax weights.  A NaN or
// +inf logit makes every probability NaN: then ids 0..k-1 with NaN weights, as a
// stable sort of all-equal values gives.
__device__ __forceinline__ void warp_topk(const double* z, int E, int k, bool renorm, int lane,
                                          int64_t* idx_out, float* w_out) {
  constexpr int kPer = kMaxE / 32;
  double v[kPer];
  double m = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + 32 * i;
    v[i] = e < E ? z[e] : -INFINITY;
    bad |= e < E && !(v[i] < INFINITY);
    m = fmax(m, v[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
  bad = __any_sync(0xffffffffu, bad) || !(m > -INFINITY);
  if (bad) {
    if (lane < k) {
      idx_out[lane] = lane;
      w_out[lane] = __int_as_float(0x7fc00000);
    }
    return;
  }
  // The exponent's argument is a difference of fp64 logits, rounded once to fp32.
  float s = 0.0f;
  // Order-preserving words for the search: a larger word is a larger logit (+0 and -0
  // are one); 0 is below every logit's word and marks no candidate.
  uint64_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    key[i] = 0;
    if (lane + 32 * i < E) {
      s += expf(static_cast<float>(v[i] - m));
      const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v[i] + 0.0));
      key[i] = (b >> 63) ? ~b : b | (1ull << 63);
    }
  }
  s = warp_sum(s);
  double my_z = 0.0;
  int my_e = 0;
  for (int j = 0; j < k; ++j) {
    uint64_t best = key[0];
    int be = lane;
#pragma unroll
    for (int i = 1; i < kPer; ++i)
      if (key[i] > best) best = key[i], be = lane + 32 * i;
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(best >> 32));
    const uint32_t lo = __reduce_max_sync(
        0xffffffffu, static_cast<uint32_t>(best >> 32) == hi ? static_cast<uint32_t>(best) : 0u);
    const bool mine = best == ((static_cast<uint64_t>(hi) << 32) | lo);
    be = static_cast<int>(__reduce_min_sync(0xffffffffu, mine ? static_cast<uint32_t>(be) : 0xffffffffu));
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + 32 * i == be) key[i] = 0;
    if (lane == j) my_e = be;
  }
  if (lane < k) my_z = z[my_e];
  const float p = lane < k ? expf(static_cast<float>(my_z - m)) / s : 0.0f;
  const float sum = renorm ? warp_sum(p) : 1.0f;
  if (lane < k) {
    idx_out[lane] = my_e;
    w_out[lane] = p / sum;
  }
}

// One cluster of 8 CTAs a token: CTA r sums the logits of experts r, r + 8, ..., its
// warps split over those experts and, when they are few, over parts of hidden; the
// first CTA gathers the logits and takes the top k.  Also zeroes the counters of the
// experts' kernel, which is allowed to start at once and waits for this one's end.
constexpr int kGateCluster = 8;

template <typename T>
__global__ void __cluster_dims__(kGateCluster, 1, 1) __launch_bounds__(32 * kWarps)
    gate_kernel(const T* x, int64_t ldx, const T* rw, int64_t ldr, const float* bias, int H, int E,
                int k, int renorm, int64_t* idx, float* w, int32_t* count, int n_count) {
  __shared__ double z[kMaxE];
  __shared__ double partial[kMaxE / kGateCluster][kWarps];
  let_next_kernel_start();
  cluster_arrive();  // this CTA is there; the first one's memory is written only when it is
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = static_cast<int>(cluster_ctarank()), t = blockIdx.x / kGateCluster;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < n_count; i += 32 * kWarps) count[i] = 0;
  const int mine = (E - rank + kGateCluster - 1) / kGateCluster;  // experts of this CTA (may be 0)
  const int parts = mine > 0 && mine < kWarps ? kWarps / mine : 1;
  const int cols = ((H + parts - 1) / parts + 7) / 8 * 8;
  for (int u = warp; u < mine * parts; u += kWarps) {
    const int i = u / parts, c0 = (u % parts) * cols;
    const int n = min(cols, H - c0);  // <= 0: an empty part
    const double d = warp_dot(x + t * ldx + c0, rw + int64_t(rank + i * kGateCluster) * ldr + c0, n, lane);
    if (lane == 0) partial[i][u % parts] = d;
  }
  __syncthreads();
  cluster_wait();
  if (threadIdx.x < mine) {
    const int e = rank + static_cast<int>(threadIdx.x) * kGateCluster;
    double d = 0;
    for (int i = 0; i < parts; ++i) d += partial[threadIdx.x][i];
    if (bias != nullptr) d += static_cast<double>(bias[e]);
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&z[e]), 0)), "d"(d)
                 : "memory");
  }
  cluster_sync_all();
  if (rank == 0 && warp == 0)
    warp_topk(z, E, k, renorm != 0, lane, idx + int64_t(t) * k, w + int64_t(t) * k);
}

// ------------------------------------------------------------ the experts --
// One persistent kernel streams the weights of the experts taken, once for each group of at
// most 8 J of an expert's slots; an expert's later groups find them in L2 for the most part.
// A work item is BM rows of W1[e] (all of hidden) for one group of at most 8 J slots
// of expert e, or BM rows of W2[e] (one of KS parts of ffn) for such a group.  Items
// are taken from a ticket counter, all of W1's before any of W2's; the items of W2
// wait (bounded) until their group's h is complete.  Whoever holds an earlier ticket
// is running and waits for nothing later, so the waits end whatever else the GPU
// does, and no grid-wide barrier is needed.
//
// Warp 0 fetches weights: TMA boxes of BM rows x 64 columns into a ring of stages of
// 16 KB.  The weights do not depend on h, so the ring runs ahead into W2 while h is
// still being finished.  Up to four warps copy the slots' columns of the same stage beside
// them (rows of x picked by token, or rows of h; one warp's instructions bound
// many slots: 215 us of 46 tokens' top-8 of 9 x 1712 x 6320, 200 by four).  Two sets of 8 warps
// multiply, on items in turn, so that one set's sums, stores and fences (several
// microseconds' worth of latency an item) pass under the other's products, or (SHARE) on
// half of an item's slots each: a stage is R tiles of 16 rows x C = 8/R slices of 64
// columns, one (tile, slice) per warp of a set, m16n8k16 with the weights as the 16-row side and the slots as the 8-column side.
// (tcgen05's 128-row tiles would leave too few items for 148 SMs at one token, and
// at a few slots an expert the tensor work is a few percent of the time.)  The order of k
// inside a slice is free, so lane (g, q) takes the 16 contiguous columns 16q.. of its
// rows and of its slot: both come by conflict-free 16-byte shared loads.
//
// Bound at a few slots an expert by reading the weights of the experts taken.  Gate and
// experts together, measured: 16 tokens, 16 experts of 2048 x 8192, top-2: 140-146 us,
// 6.5-6.7 TB/s; 64 tokens of the same 173-178 us, 6.0-6.2 TB/s; one token of 2048 x 4096: 28.3 us,
// of which some 15 read weights and the rest is the chain from the gate to the last sum.
// At many slots an expert (41: 46 tokens, top-8 of 9 x 1712 x 6320, 179 us) by the slots'
// way through shared memory and registers once a row block: DRAM is at 28 % then, the
// shared-memory pipe at 53 %, the tensor pipe at 28 %.
constexpr int kConsumers = 8;
constexpr int kSets = 2;         // of consumers
// Warps that copy slots: more than their rows need only add arrivals to every stage (16
// tokens, top-2 of 16 x 1024 x 2048: 43 us with one, 46 with four).
constexpr int copy_warps(int J, bool share) { return share ? 4 : J == 1 ? 1 : 2; }
constexpr int threads(int J, bool share) { return 32 * (1 + copy_warps(J, share) + kSets * kConsumers); }
constexpr int kStageBytes = 16 * 1024;
constexpr int kRedStride = 20;  // floats between slots in the reduction buffer: no bank conflicts
constexpr int kMaxSlots = kMaxTokens * kMaxK;
constexpr int kQueue = 8;

// Shared memory of one variant.  A stage's slots: 8 J rows of 64 C columns, twice (h
// comes in two parts).
template <int R, int J>
struct Cfg {
  static constexpr int BM = 16 * R, C = kConsumers / R, BKS = 64 * C, NT = 8 * J;
  static constexpr int kSlotBytes = NT * BKS * 2;
  static constexpr int kFull = kStageBytes + 2 * kSlotBytes;
  static constexpr int kRed = C > 1 ? kSets * kConsumers * NT * kRedStride * 4 : 0;
  static constexpr int kStages = (200 * 1024 - kRed) / kFull;
  static constexpr int kBytes = kStages * kFull + kRed;
};

__host__ __device__ constexpr int max_groups(int J, int E) { return E + kMaxSlots / (8 * J); }

struct Params {
  const void* x;
  int64_t ldx;
  const int64_t* idx;
  const float* w;
  void* out;
  int64_t ldo;
  void* h;         // [2][slots][F]: h in slot order by expert, rounded, and what the rounding left
  float* part;     // [KS * C][slots][H]
  int32_t* count;  // ticket, then per group its finished W1 items, then per 16 rows of H its finished parts
  int32_t* status;
  int T, H, F, E, k, KS, part_cols;  // W2's items: KS parts of F, of part_cols columns (see parts_of)
};

struct Plan {  // in shared memory; every CTA derives the same one from idx
  int n_groups, n_slots;
  int16_t expert_of_slot[kMaxSlots];  // -1: none
  uint16_t slot_at[kMaxSlots];        // slots ordered by expert
  uint16_t pos_of[kMaxSlots];         // place of a slot in that order, 0xffff: none
};

struct Ctrl {
  uint64_t full[12], empty[12], qfull[kQueue], qempty[kQueue], turn[kSets], sums[kSets];
  int item[kQueue];
  int abort;  // a wait ran out: every role leaves
};

// The slots by expert and the groups of at most NT of them: grp holds
// expert << 16 | place of the group's first slot.
__device__ __forceinline__ void build_plan(const Params& p, int NT, int block, Plan* pl, int* grp, int* cnt,
                                           int* grp_first) {
  const int tid = threadIdx.x, S = p.T * p.k;
  for (int i = tid; i < S; i += block) {
    const int64_t e = p.idx[i];
    if (e < -1 || e >= p.E) record_status(p.status, MOE_ERR_INVALID_ARG);
    pl->expert_of_slot[i] = (e >= 0 && e < p.E) ? static_cast<int16_t>(e) : int16_t(-1);
  }
  for (int e = tid; e < p.E; e += block) cnt[e] = 0;
  __syncthreads();
  if (tid < 32) {
    // Each slot's rank among its expert's, 32 slots at a time in slot order.
    for (int b = 0; b < S; b += 32) {
      const int i = b + tid, e = i < S ? pl->expert_of_slot[i] : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      const int before = e >= 0 ? cnt[e] : 0;
      if (i < S) pl->pos_of[i] = static_cast<uint16_t>(before + __popc(same & ((1u << tid) - 1u)));
      __syncwarp();
      if (e >= 0 && (same >> tid) == 1u) cnt[e] = before + __popc(same);
      __syncwarp();
    }
    int run_s = 0, run_g = 0;  // prefix sums over the experts: slots and groups
    for (int b = 0; b < p.E; b += 32) {
      const int e = b + tid;
      const int c = e < p.E ? cnt[e] : 0, g = (c + NT - 1) / NT;
      int is = c, ig = g;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int vs = __shfl_up_sync(0xffffffffu, is, o), vg = __shfl_up_sync(0xffffffffu, ig, o);
        if (tid >= o) {
          is += vs;
          ig += vg;
        }
      }
      if (e < p.E) {
        cnt[e] = run_s + is - c;
        grp_first[e] = run_g + ig - g;
      }
      run_s += __shfl_sync(0xffffffffu, is, 31);
      run_g += __shfl_sync(0xffffffffu, ig, 31);
    }
    if (tid == 0) {
      pl->n_slots = run_s;
      pl->n_groups = run_g;
    }
  }
  __syncthreads();
  for (int i = tid; i < S; i += block) {
    const int e = pl->expert_of_slot[i], rank = pl->pos_of[i];
    if (e < 0) {
      pl->pos_of[i] = 0xffff;
      continue;
    }
    const int at = cnt[e] + rank;
    if (rank % NT == 0) grp[grp_first[e] + rank / NT] = (e << 16) | at;
    pl->slot_at[at] = static_cast<uint16_t>(i);
    pl->pos_of[i] = static_cast<uint16_t>(at);
  }
  __syncthreads();
}

// One work item, decoded from its ticket.
struct Item {
  bool down;
  int g, blk, ks, c0, c1;  // group, row block, part of ffn, its columns [c0, c1)
};

template <typename T, int R, int J, bool SHARE>
__global__ void __launch_bounds__(threads(J, SHARE), 1)
    experts_kernel(const __grid_constant__ CUtensorMap map1, const __grid_constant__ CUtensorMap map2,
                   const __grid_constant__ Params p) {
  using K = Cfg<R, J>;
  constexpr int BM = K::BM, C = K::C, BKS = K::BKS, NT = K::NT, kStages = K::kStages;
  constexpr int kSliceBytes = BM * 128;
  static_assert(!SHARE || (C == 1 && J % kSets == 0), "whole tiles of 8 slots a set");
  constexpr int kCopyWarps = copy_warps(J, SHARE), kFirstConsumer = 1 + kCopyWarps;
  constexpr int kThreads = threads(J, SHARE);
  constexpr int JS = SHARE ? J / kSets : J;                         // tiles of 8 slots of a warp
  constexpr int kWarpsOn = SHARE ? kSets * kConsumers : kConsumers;  // on an item
  extern __shared__ char smem_raw[];
  char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // Stages' weights, then their slots, then two reduction buffers.
  char* slots = base + kStages * kStageBytes;
  float* red = reinterpret_cast<float*>(slots + kStages * 2 * K::kSlotBytes);
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(base + K::kBytes);
  Plan* plan = reinterpret_cast<Plan*>(ctrl + 1);
  int* grp = reinterpret_cast<int*>(plan + 1);
  int* cnt = grp + max_groups(J, p.E);
  int* grp_first = cnt + p.E;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&ctrl->full[s]), 1 + 32 * kCopyWarps);
      mbar_init(smem_u32(&ctrl->empty[s]), kWarpsOn);
    }
    for (int s = 0; s < kSets; ++s) {
      mbar_init(smem_u32(&ctrl->turn[s]), kConsumers);
      mbar_init(smem_u32(&ctrl->sums[s]), kConsumers);
    }
    for (int s = 0; s < kQueue; ++s) {
      mbar_init(smem_u32(&ctrl->qfull[s]), 1);
      mbar_init(smem_u32(&ctrl->qempty[s]), kCopyWarps + kSets * kConsumers);
    }
    ctrl->abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map1);
    tma_prefetch_desc(&map2);
  }
  wait_for_previous_kernel();  // the gate's idx, w and counters
  int ticket = 0;  // the fetching thread's first, on its way while the plan is made
  if (tid == 0) ticket = atomicAdd(p.count, 1);
  build_plan(p, NT, kThreads, plan, grp, cnt, grp_first);
  const int G = plan->n_groups, S = plan->n_slots;
  const int FB = (p.F + BM - 1) / BM, HB = (p.H + BM - 1) / BM;
  if (G == 0) {  // no slot is routed: zeros
    T* out = static_cast<T*>(p.out);
    for (int64_t i = blockIdx.x * kThreads + tid; i < int64_t(p.T) * p.H; i += gridDim.x * kThreads)
      out[(i / p.H) * p.ldo + i % p.H] = from_f<T>(0.0f);
    return;
  }
  const int up_items = G * FB, items = up_items + G * HB * p.KS;
  int* ready = p.count + 1;
  int* done = ready + G;
  auto decode = [&](int item) {
    Item it;
    it.down = item >= up_items;
    const int q = it.down ? item - up_items : item, per = it.down ? HB * p.KS : FB;
    it.g = q / per;
    const int r = q - it.g * per;
    it.blk = it.down ? r / p.KS : r;
    it.ks = it.down ? r - it.blk * p.KS : 0;
    it.c0 = it.ks * p.part_cols;
    it.c1 = it.down ? min(it.c0 + p.part_cols, p.F) : p.H;
    return it;
  };
  // A warp whose wait has run out (or another's has) leaves; no one waits for it unbounded.
  volatile int* abort_flag = &ctrl->abort;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_wait(smem_u32(bar), parity, abort_flag)) return true;
    give_up(abort_flag, p.status, MOE_ERR_TIMEOUT);
    return false;
  };
  // Until a counter that other CTAs raise has come to `n`.
  auto wait_count = [&](const int* count, int n) {
    const long long t0 = clock64();
    while (ld_acquire_gpu(count) < n)
      if (*abort_flag || clock64() - t0 > kWaitBudgetCycles) {
        give_up(abort_flag, p.status, MOE_ERR_TIMEOUT);
        return false;
      }
    return true;
  };
  // Takes the queue's next item; -1 at the end, -2 when the wait ran out.
  auto pop = [&](int n) {
    const int slot = n % kQueue;
    if (!__all_sync(0xffffffffu, wait(&ctrl->qfull[slot], (n / kQueue) & 1))) return -2;
    const int item = ctrl->item[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&ctrl->qempty[slot]));
    return item;
  };

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int next = ticket;
      for (int n = 0;; ++n) {
        const int item = next;
        const bool end = item >= items;
        if (!end) next = atomicAdd(p.count, 1);
        const int slot = n % kQueue;
        if (!wait(&ctrl->qempty[slot], ((n / kQueue) & 1) ^ 1)) return;
        ctrl->item[slot] = end ? -1 : item;
        mbar_arrive(smem_u32(&ctrl->qfull[slot]));
        if (end) return;
        const Item it = decode(item);
        const int e = grp[it.g] >> 16;
        const CUtensorMap* map = it.down ? &map2 : &map1;
        for (int c = it.c0; c < it.c1; c += BKS) {
          const uint32_t full = smem_u32(&ctrl->full[stage]);
          if (!wait(&ctrl->empty[stage], phase ^ 1)) return;
          mbar_arrive_expect_tx(full, kStageBytes);
          const uint32_t dst = smem_u32(base + stage * kStageBytes);
#pragma unroll
          for (int i = 0; i < C; ++i)
            tma_load_3d(dst + i * kSliceBytes, map, full, c + 64 * i, it.blk * BM, e);
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
      }
    }
    return;
  }

  const T* x = static_cast<const T*>(p.x);
  T* h = static_cast<T*>(p.h);
  T* h_lo = h + int64_t(p.T) * p.k * p.F;
  if (warp < kFirstConsumer) {
    // A stage's slots: row nn of slice s at (s NT + nn) * 128, its 16-byte pieces
    // XOR-ed with nn & 7 like the weights' TMA swizzle.
    constexpr int kPieces = BKS / 8;              // of 16 bytes in a row
    constexpr int kPasses = (NT * kPieces / 32 + kCopyWarps - 1) / kCopyWarps;
    const int first = (warp - 1) * 32 + lane;     // its pieces: this one and every 32 kCopyWarps-th
    constexpr int kNext = 32 * kCopyWarps;
    uint32_t off[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int nn = (first + kNext * i) / kPieces, piece = (first + kNext * i) % kPieces;
      off[i] = ((piece >> 3) * NT + nn) * 128 + (((piece & 7) ^ (nn & 7)) << 4);
    }
    const int piece8 = lane % kPieces * 8;  // (32 is a multiple of kPieces: the same in every pass)
    int stage = 0;
    uint32_t phase = 0;
    for (int n = 0;; ++n) {
      const int item = pop(n);
      if (item < 0) return copies_wait_all();
      const Item it = decode(item);
      const int pos0 = grp[it.g] & 0xffff;
      const int rows = (it.g + 1 < G ? (grp[it.g + 1] & 0xffff) : S) - pos0;
      // (in a down item) this group's h, complete and visible to this thread
      if (it.down && !__all_sync(0xffffffffu, wait_count(ready + it.g, FB * kWarpsOn))) return copies_wait_all();
      const T* src[kPasses];
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int nn = (first + kNext * i) / kPieces;
        src[i] = nullptr;
        if (nn < rows)
          src[i] = (it.down ? h + int64_t(pos0 + nn) * p.F
                            : x + (plan->slot_at[pos0 + nn] / p.k) * p.ldx) +
                   piece8;
      }
      for (int c = it.c0; c < it.c1; c += BKS) {
        const uint32_t full = smem_u32(&ctrl->full[stage]);
        if (!__all_sync(0xffffffffu, wait(&ctrl->empty[stage], phase ^ 1))) return copies_wait_all();
        const uint32_t dst = smem_u32(slots + stage * 2 * K::kSlotBytes);
        const bool in = c + piece8 < it.c1;
        const int from = in ? c : it.c0;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          if (i * kNext / kPieces >= rows) break;
          if (src[i] != nullptr) {
            copy_async_16(dst + off[i], src[i] + from, in);
            if (it.down) copy_async_16(dst + off[i] + K::kSlotBytes, src[i] + from + (h_lo - h), in);
          }
        }
        copies_arrive(full);
        if (++stage == kStages) stage = 0, phase ^= 1;
      }
    }
  }

  const int set = (warp - kFirstConsumer) / kConsumers, cw = (warp - kFirstConsumer) % kConsumers;
  const int rt = cw % R, cs = cw / R, g8 = lane >> 2, q4 = lane & 3;
  const uint32_t a_base = smem_u32(base) + cs * kSliceBytes + (rt * 16 + g8) * 128;
  const int s0 = SHARE ? set * 8 * JS : 0;  // this set's first slot of a group
  const uint32_t b_base = smem_u32(slots) + (cs * NT + s0 + g8) * 128;
  const uint32_t off0 = ((2 * q4) ^ g8) * 16, off1 = ((2 * q4 + 1) ^ g8) * 16;
  int stage = 0;
  uint32_t phase = 0;
  [[maybe_unused]] uint32_t sums_parity = 0;
  for (int n = 0;; ++n) {
    const int item = pop(n);
    if (item == -1) break;
    if (item < 0) return;
    const Item it = decode(item);
    if (!SHARE && n % kSets != set) {  // the other set's item: past its stages
      stage += (it.c1 - it.c0 + BKS - 1) / BKS;
      while (stage >= kStages) stage -= kStages, phase ^= 1;
      continue;
    }
    // The other set has used every stage before this item's: a parity wait on a stage
    // is only sound within one turn of the ring.
    if (!SHARE && !__all_sync(0xffffffffu, wait(&ctrl->turn[set], ((n / kSets) & 1) ^ (set == 0)))) return;
    const int pos0 = grp[it.g] & 0xffff;
    const int rows = (it.g + 1 < G ? (grp[it.g + 1] & 0xffff) : S) - pos0;
    // Two sums of every output, so that no product waits for the one before it (a stage's
    // products are a chain of latencies otherwise); added at the end.
    float acc[JS][4], acc2[JS][4];
#pragma unroll
    for (int j = 0; j < JS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = acc2[j][i] = 0.0f;

    // A stage with NJ tiles of 8 slots (what is in slots behind the group's stays in their
    // sums, which nobody reads), of x or of both parts of h.
    auto multiply = [&](auto nj, auto parts) {
      constexpr int NJ = decltype(nj)::value, P = decltype(parts)::value;
      uint32_t a[2][8];  // rows g8 and g8 + 8, 16 columns each
      const uint32_t sa = a_base + stage * kStageBytes;
      ld_shared_v4(sa + off0, &a[0][0]);
      ld_shared_v4(sa + off1, &a[0][4]);
      ld_shared_v4(sa + 1024 + off0, &a[1][0]);
      ld_shared_v4(sa + 1024 + off1, &a[1][4]);
#pragma unroll
      for (int part = 0; part < P; ++part) {
        uint32_t v[NJ][8];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint32_t sb = b_base + stage * 2 * K::kSlotBytes + part * K::kSlotBytes + j * 1024;
          ld_shared_v4(sb + off0, &v[j][0]);
          ld_shared_v4(sb + off1, &v[j][4]);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            mma<T>(s & 1 ? acc2[j] : acc[j], a[0][2 * s], a[1][2 * s], a[0][2 * s + 1], a[1][2 * s + 1],
                   v[j][2 * s], v[j][2 * s + 1]);
      }
    };
    for (int c = it.c0; c < it.c1; c += BKS) {
      if (!__all_sync(0xffffffffu, wait(&ctrl->full[stage], phase))) return;
      using std::integral_constant;
      if (JS > 1 && rows > s0 + 8) {
        it.down ? multiply(integral_constant<int, JS>(), integral_constant<int, 2>())
                : multiply(integral_constant<int, JS>(), integral_constant<int, 1>());
      } else if (rows > s0) {
        it.down ? multiply(integral_constant<int, 1>(), integral_constant<int, 2>())
                : multiply(integral_constant<int, 1>(), integral_constant<int, 1>());
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctrl->empty[stage]));
      if (++stage == kStages) stage = 0, phase ^= 1;
    }

    if (!SHARE && lane == 0) mbar_arrive(smem_u32(&ctrl->turn[set ^ 1]));
#pragma unroll
    for (int j = 0; j < JS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] += acc2[j][i];

    if (!it.down) {
      auto put_h = [&](int nn, int row, float v) {
        const float a = 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f));
        const int64_t at = int64_t(pos0 + nn) * p.F + row;
        split(a, h + at, h_lo + at);
      };
      if constexpr (C == 1) {
#pragma unroll
        for (int j = 0; j < JS; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int nn = s0 + j * 8 + 2 * q4 + (i & 1), row = it.blk * BM + rt * 16 + g8 + 8 * (i >> 1);
            if (nn < rows && row < p.F) put_h(nn, row, acc[j][i]);
          }
      } else {  // the C column slices' sums, through shared memory
        float* rb = red + (set * kConsumers + cw) * (NT * kRedStride);
#pragma unroll
        for (int j = 0; j < JS; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            rb[(j * 8 + 2 * q4 + (i & 1)) * kRedStride + g8 + 8 * (i >> 1)] = acc[j][i];
        const uint32_t bar = smem_u32(&ctrl->sums[set]);
        if (!__all_sync(0xffffffffu, warps_sync(bar, sums_parity, abort_flag)))
          return give_up(abort_flag, p.status, MOE_ERR_TIMEOUT);
        const float* rs = red + set * kConsumers * (NT * kRedStride);
        for (int o = cw * 32 + lane; o < BM * rows; o += 32 * kConsumers) {
          const int m = o % BM, nn = o / BM, row = it.blk * BM + m;
          float v = 0.0f;
#pragma unroll
          for (int i = 0; i < C; ++i)
            v += rs[(i * R + m / 16) * (NT * kRedStride) + nn * kRedStride + m % 16];
          if (row < p.F) put_h(nn, row, v);
        }
        if (!__all_sync(0xffffffffu, warps_sync(bar, sums_parity, abort_flag)))  // the buffer is free again
          return give_up(abort_flag, p.status, MOE_ERR_TIMEOUT);
      }
      __syncwarp();
      if (lane == 0) red_release_gpu(ready + it.g, 1);
      continue;
    }

    // This warp's part of 16 rows of W2.
    const int row16 = it.blk * BM + rt * 16;
    if (row16 >= p.H) continue;
    float* part = p.part + (int64_t(it.ks * C + cs) * p.T * p.k + pos0) * p.H + row16;
#pragma unroll
    for (int j = 0; j < JS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int nn = s0 + j * 8 + 2 * q4 + (i & 1), m = g8 + 8 * (i >> 1);
        if (nn < rows && row16 + m < p.H) part[int64_t(nn) * p.H + m] = acc[j][i];
      }
    __syncwarp();
    if (lane == 0) red_release_gpu(done + it.blk * R + rt, 1);
  }

  // The weighted sums over the slots and their parts, in a fixed order: every warp of
  // the grid takes blocks of 16 columns x 8 tokens.  The items are all taken by now, by
  // CTAs that run, so the waits for their parts end.
  const int t_groups = (p.T + 7) / 8, units = (p.H + 15) / 16 * t_groups;
  const int parts = p.KS * C, terms = p.k * parts;
  const int64_t part_stride = int64_t(p.T) * p.k * p.H;
  for (int u = (warp - kFirstConsumer) * gridDim.x + blockIdx.x; u < units; u += kSets * kConsumers * gridDim.x) {
    const int blk16 = u / t_groups, t = u % t_groups * 8 + (lane >> 2);
    const int col = blk16 * 16 + (lane & 3) * 4;  // 4 columns of one token a lane (H: a multiple of 8)
    if (!wait_count(done + blk16, G * parts * (kWarpsOn / kConsumers))) return;
    if (t >= p.T || col >= p.H) continue;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int j = 0, i = 0;
    for (int b = 0; b < terms; b += 8) {  // 8 loads under way at a time
      float4 y[8];
      float wt[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        y[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        wt[q] = 0.0f;
        const int pos = b + q < terms ? plan->pos_of[t * p.k + j] : 0xffff;
        if (pos != 0xffff) {
          y[q] = __ldcg(reinterpret_cast<const float4*>(p.part + i * part_stride + int64_t(pos) * p.H + col));
          wt[q] = p.w[t * p.k + j];
        }
        if (++i == parts) i = 0, ++j;
      }
#pragma unroll
      for (int q = 0; q < 8; ++q)
        v[0] += wt[q] * y[q].x, v[1] += wt[q] * y[q].y, v[2] += wt[q] * y[q].z, v[3] += wt[q] * y[q].w;
    }
    T o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = from_f<T>(v[q]);
    *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + t * p.ldo + col) = *reinterpret_cast<const uint2*>(o);
  }
}

// The parts of F in W2's items: about 2048 columns each, wider ones when there are many slots (then
// there are many groups, and the parts' sums cost more than their balance gains), in whole
// stages of `stage` columns.  No part is empty: the consumers that skip an item count its
// stages from its columns, so the number of parts follows from their rounded width.
struct Parts {
  int n, cols;
};
inline Parts parts_of(int F, int64_t S, int stage) {
  const int64_t fine = (F + 2047) / 2048, most = S < 1 || S >= 1024 ? 1 : 1024 / S;
  const int64_t n = fine < most ? fine : most;
  const int64_t cols = ((F + n - 1) / n + stage - 1) / stage * stage;
  return {static_cast<int>((F + cols - 1) / cols), static_cast<int>(cols)};
}
// Column slices of a stage, and its columns, with row blocks of 16 R.
constexpr int slices(int R) { return kConsumers / R; }
constexpr int stage_cols(int R) { return 64 * slices(R); }
constexpr int kWideR = 8, kNarrowR = 2;  // what launch() chooses between

struct Workspace {
  int64_t part, count, total;
  Workspace(int T, int H, int F, int E, int k) {
    const int64_t S = int64_t(T) * k;
    part = (S * F * 4 + 15) / 16 * 16;
    // Each part's slices have sums of their own.
    const int wide = parts_of(F, S, stage_cols(kWideR)).n * slices(kWideR);
    const int narrow = parts_of(F, S, stage_cols(kNarrowR)).n * slices(kNarrowR);
    count = part + (S * H * 4 * (wide > narrow ? wide : narrow) + 15) / 16 * 16;
    total = count + 4 * (int64_t(1) + max_groups(1, E) + (H + 15) / 16);
  }
  int64_t count_bytes() const { return total - count; }
};

template <typename T, int R, int J, bool SHARE>
int launch_experts(Params p, const void* w1, int64_t w1_se, int64_t w1_sr, const void* w2,
                   int64_t w2_se, int64_t w2_sr, bool after_gate, int sms, cudaStream_t s) {
  using K = Cfg<R, J>;
  static_assert(K::BKS == stage_cols(R) && K::C == slices(R) && (R == kWideR || R == kNarrowR), "the workspace's");
  const Parts parts = parts_of(p.F, int64_t(p.T) * p.k, K::BKS);
  p.KS = parts.n, p.part_cols = parts.cols;
  CUtensorMap m1, m2;
  const CUtensorMapDataType dt = std::is_same<T, __nv_bfloat16>::value
                                     ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint32_t box[3] = {64, K::BM, 1};
  const uint64_t d1[3] = {uint64_t(p.H), uint64_t(p.F), uint64_t(p.E)};
  const uint64_t d2[3] = {uint64_t(p.F), uint64_t(p.H), uint64_t(p.E)};
  const uint64_t s1[2] = {uint64_t(w1_sr) * 2, uint64_t(p.E > 1 ? w1_se : w1_sr * p.F) * 2};
  const uint64_t s2[2] = {uint64_t(w2_sr) * 2, uint64_t(p.E > 1 ? w2_se : w2_sr * p.H) * 2};
  int rc = encode_tiled(&m1, dt, 3, w1, d1, s1, box);
  if (rc == MOE_OK) rc = encode_tiled(&m2, dt, 3, w2, d2, s2, box);
  if (rc != MOE_OK) return rc;
  constexpr int kFixed = 1024 + K::kBytes + int(sizeof(Ctrl)) + int(sizeof(Plan));
  const int smem = kFixed + 4 * (max_groups(J, p.E) + 2 * p.E);
  constexpr int kMost = kFixed + 4 * (max_groups(J, kMaxE) + 2 * kMaxE);
  static_assert(K::kStages <= 12 && kMost <= 227 * 1024, "shared memory");
  constexpr auto kern = &experts_kernel<T, R, J, SHARE>;
  if (!allow_shared_memory<kern>(kMost)) return MOE_ERR_CUDA;
  // No more CTAs than there can be items: every slot in a group of its own.
  const int64_t most = int64_t(p.T) * p.k * ((p.F + K::BM - 1) / K::BM + (p.H + K::BM - 1) / K::BM * p.KS);
  const int grid = static_cast<int>(most < sms ? most : sms);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads(J, SHARE));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute early{};  // set up beside the gate's kernel
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = after_gate ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, m1, m2, p) == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

template <typename T>
int launch(Params p, const void* rw, int64_t ldr, const float* bias, const void* w1, int64_t w1_se,
           int64_t w1_sr, const void* w2, int64_t w2_se, int64_t w2_sr, int renorm, int64_t* idx,
           float* w, void* ws, int sms, cudaStream_t s) {
  const Workspace lay(p.T, p.H, p.F, p.E, p.k);
  p.idx = idx;
  p.w = w;
  p.h = ws;
  p.part = reinterpret_cast<float*>(static_cast<char*>(ws) + lay.part);
  p.count = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + lay.count);
  if (rw != nullptr) {
    gate_kernel<T><<<p.T * kGateCluster, 32 * kWarps, 0, s>>>(
        static_cast<const T*>(p.x), p.ldx, static_cast<const T*>(rw), ldr, bias, p.H, p.E, p.k, renorm,
        idx, w, p.count, static_cast<int>(lay.count_bytes() / 4));
    if (cudaGetLastError() != cudaSuccess) return MOE_ERR_CUDA;
  } else if (cudaMemsetAsync(p.count, 0, lay.count_bytes(), s) != cudaSuccess) {
    return MOE_ERR_CUDA;
  }
  auto go = [&](auto r, auto j, auto share) {
    return launch_experts<T, decltype(r)::value, decltype(j)::value, decltype(share)::value>(p, w1, w1_se, w1_sr, w2, w2_se, w2_sr,
                                                                     rw != nullptr, sms, s);
  };
  using std::integral_constant;
  // Blocks of 128 rows need no sums across warps and fetch each slot's columns once for
  // all 8 warps; a few slots' few experts make too few of them for every SM and get blocks
  // of 32 rows.  Measured with 32 and 128 rows, experts x hidden x ffn: one token's 2 slots
  // of 16 x 2048 x 4096 28.6 and 32.8 us; 8 tokens' 16 of 8 x 512 x 1024 18.7 and 20.5; 16
  // tokens' 32 of 8 x 4096 x 1024 49.6 and 44.0; 128 tokens' 256 of it 168 and 76.
  const int64_t S = int64_t(p.T) * p.k, groups = S < p.E ? S : p.E;
  const bool narrow = S <= 16 && groups * ((p.F + 127) / 128) < sms;
  // With 16 slots or more an expert both sets of consumers take an item, 16 of its 32 slots
  // each, so that the weights go by half as often; but no set's sums pass under the other's
  // products then, which wants long items and enough of them.  128 tokens, top-2 of 8 x 2048 x
  // 8192: 168 us, 199 with 16 slots an item; 62 tokens, top-6 of 12 x 600 x 7888 126 and 111;
  // 32 tokens, top-2 of 2 x 2048 x 2048 45 and 37.
  if (p.T > 8 && S >= 16 * int64_t(p.E) && p.H >= 1024 && groups * ((p.F + 127) / 128) >= sms / 2)
    return go(integral_constant<int, kWideR>(), integral_constant<int, 4>(), std::true_type());
  if (p.T > 8) return go(integral_constant<int, kWideR>(), integral_constant<int, 2>(), std::false_type());
  // No expert has more than 8 slots, unless it is repeated.
  return narrow ? go(integral_constant<int, kNarrowR>(), integral_constant<int, 1>(), std::false_type())
                : go(integral_constant<int, kWideR>(), integral_constant<int, 1>(), std::false_type());
}

}  // namespace few
}  // namespace moe

namespace {
bool sizes_ok(int32_t num_tokens, int32_t hidden, int32_t ffn, int32_t num_experts, int32_t topk) {
  using namespace moe::few;
  return num_tokens >= 0 && num_tokens <= kMaxTokens && hidden >= 8 && hidden % 8 == 0 && hidden <= kMaxWidth &&
         ffn >= 8 && ffn % 8 == 0 && ffn <= kMaxWidth && num_experts >= 1 && num_experts <= kMaxE &&
         topk >= 1 && topk <= kMaxK && topk <= num_experts;
}
bool rows_ok(const void* p, int64_t ld, int64_t width) {
  return p != nullptr && moe::aligned16(p) && ld >= width && ld % 8 == 0;
}
}  // namespace

extern "C" int64_t moe_few_tokens_workspace(int32_t num_tokens, int32_t hidden, int32_t ffn,
                                            int32_t num_experts, int32_t topk) {
  if (!sizes_ok(num_tokens, hidden, ffn, num_experts, topk)) return -1;
  return moe::few::Workspace(num_tokens, hidden, ffn, num_experts, topk).total;
}

extern "C" int32_t moe_few_tokens_parts(int32_t num_tokens, int32_t ffn, int32_t num_experts, int32_t topk,
                                        int32_t narrow, int32_t* part_cols) {
  using namespace moe::few;
  if (!sizes_ok(num_tokens, 8, ffn, num_experts, topk) || part_cols == nullptr) return -1;
  const Parts parts = parts_of(ffn, int64_t(num_tokens) * topk, stage_cols(narrow != 0 ? kNarrowR : kWideR));
  *part_cols = parts.cols;
  return parts.n;
}

extern "C" int32_t moe_few_tokens(const void* x, int64_t ldx, const void* router_w, int64_t ldr,
                                  const float* router_bias, const void* w1, int64_t w1_stride_e,
                                  int64_t w1_stride_row, const void* w2, int64_t w2_stride_e,
                                  int64_t w2_stride_row, int32_t dtype, int32_t num_tokens,
                                  int32_t hidden, int32_t ffn, int32_t num_experts, int32_t topk,
                                  int32_t renormalize, int64_t* topk_idx, float* topk_weights,
                                  void* out, int64_t ldo, void* workspace, int64_t workspace_bytes,
                                  int32_t* status, void* stream) {
  if (!sizes_ok(num_tokens, hidden, ffn, num_experts, topk) ||
      (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16))
    return MOE_ERR_INVALID_ARG;
  if (num_tokens == 0) return MOE_OK;
  if (!rows_ok(x, ldx, hidden) || !rows_ok(out, ldo, hidden) || !rows_ok(w1, w1_stride_row, hidden) ||
      !rows_ok(w2, w2_stride_row, ffn) || (router_w != nullptr && !rows_ok(router_w, ldr, hidden)) ||
      (num_experts > 1 && (w1_stride_e < w1_stride_row * ffn || w1_stride_e % 8 != 0 ||
                           w2_stride_e < w2_stride_row * hidden || w2_stride_e % 8 != 0)) ||
      topk_idx == nullptr || topk_weights == nullptr || workspace == nullptr ||
      !moe::aligned16(workspace))
    return MOE_ERR_INVALID_ARG;
  if (workspace_bytes < moe_few_tokens_workspace(num_tokens, hidden, ffn, num_experts, topk))
    return MOE_ERR_CAPACITY;
  int dev;
  moe::DeviceInfo info;
  const int rc = moe::current_device_info(&dev, &info);
  if (rc != MOE_OK) return rc;
  if (info.major != 10) return MOE_ERR_UNSUPPORTED;
  moe::few::Params p{};
  p.x = x, p.ldx = ldx, p.out = out, p.ldo = ldo, p.status = status;
  p.T = num_tokens, p.H = hidden, p.F = ffn, p.E = num_experts, p.k = topk;
  auto fn = dtype == MOE_DTYPE_BF16 ? &moe::few::launch<__nv_bfloat16> : &moe::few::launch<__half>;
  return fn(p, router_w, ldr, router_bias, w1, w1_stride_e, w1_stride_row, w2, w2_stride_e,
            w2_stride_row, renormalize, topk_idx, topk_weights, workspace, info.sm_count,
            static_cast<cudaStream_t>(stream));
}
