// The adapters' projection for few rows (decode batches) on sm_100a, in two kernels:
// low[m] = x[m] A[i]^T  and  y[m] = x[m] W^T + scale[i] low[m] B[i]^T.
//
// The shared weight is the traffic: it is read once for 64 rows, and the second kernel
// starts beside the first and has its first weights under way while `low` is formed; only
// its epilogue waits for it.  The adapters' products are a few thousand products an output
// block and run on the CUDA cores in fp32, so y is rounded once.  Both kernels, measured:
// 1 row of 2048 x 2048 at rank 16 8.2 us (launch latency), 1 row of 2048 x 8192 11.9 us
// (2.8 TB/s; a cuBLAS product alone 10.3), 64 rows of it with 32 adapters 22 us.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/moe_overlap.h"
#include "host_common.h"
#include "lora.cuh"
#include "mma16.cuh"
#include "ptx.cuh"

namespace moe {
namespace lora {
namespace few {

__device__ __forceinline__ int id_at(const void* ids, int ids64, int m, int L) {
  const int64_t v = ids64 ? static_cast<const int64_t*>(ids)[m]
                          : static_cast<int64_t>(static_cast<const int32_t*>(ids)[m]);
  return v < 0 || v >= L ? (v == -1 ? -1 : -2) : static_cast<int>(v);  // -2: a bad id
}

// One warp an element of low: a row of x and a row of A, 16 bytes a lane at a time.
constexpr int kLowWarps = 4;

template <typename T>
__global__ void __launch_bounds__(32 * kLowWarps)
    low_kernel(const T* x, int64_t ldx, const T* a, int64_t sl, int64_t sr, const void* ids, int ids64,
               int L, int K, int r, float* low, int32_t* status) {
  let_next_kernel_start();
  const int lane = threadIdx.x & 31, m = blockIdx.y, j = blockIdx.x * kLowWarps + (threadIdx.x >> 5);
  const int i = id_at(ids, ids64, m, L);
  if (i == -2 && j == 0 && lane == 0) record_status(status, MOE_ERR_INVALID_ARG);
  if (i < 0 || j >= r) return;
  const T* xr = x + m * ldx;
  const T* ar = a + i * sl + j * sr;
  float s = 0.0f;
#pragma unroll 8
  for (int c = lane * 8; c < K; c += 256) {
    const uint4 ux = *reinterpret_cast<const uint4*>(xr + c);
    const uint4 ua = *reinterpret_cast<const uint4*>(ar + c);
    const T* px = reinterpret_cast<const T*>(&ux);
    const T* pa = reinterpret_cast<const T*>(&ua);
#pragma unroll
    for (int q = 0; q < 8; ++q) s += to_f(px[q]) * to_f(pa[q]);
  }
  s = warp_sum(s);
  if (lane == 0) low[m * r + j] = s;
}

// Warp 0 brings the weight by TMA, BM = 16 R rows x 64 C columns (16 KB) a stage, and the
// same columns of x's rows beside it (rows behind the last are zeros); warps 1-8
// multiply, one (16-row tile, 64-column slice) each, weights as the 16-row side of m16n8k16, x's rows as its 8-column
// side.  The order of k inside a slice is free: lane (g, q) takes the 16 contiguous
// columns 16q.. of its rows, so both operands come by 16-byte conflict-free loads.
constexpr int kConsumers = 8;
constexpr int kThreads = 32 * (1 + kConsumers);
constexpr int kStageBytes = 16 * 1024;
constexpr int kRedStride = 20;

template <typename T>
__device__ __forceinline__ float dot8(const uint4& u, const float4& l0, const float4& l1) {
  const T* p = reinterpret_cast<const T*>(&u);
  return to_f(p[0]) * l0.x + to_f(p[1]) * l0.y + to_f(p[2]) * l0.z + to_f(p[3]) * l0.w + to_f(p[4]) * l1.x +
         to_f(p[5]) * l1.y + to_f(p[6]) * l1.z + to_f(p[7]) * l1.w;
}

template <int R, int J>
struct Cfg {
  static constexpr int BM = 16 * R, C = kConsumers / R, BKS = 64 * C, NT = 8 * J;
  static constexpr int kSlotBytes = NT * BKS * 2;
  static constexpr int kRed = kConsumers * NT * kRedStride * 4;
  static constexpr int kStages = (200 * 1024 - kRed) / (kStageBytes + kSlotBytes);
  static constexpr int kBytes = kStages * (kStageBytes + kSlotBytes) + kRed;
  static_assert(kStages >= 3 && kStages <= 12, "stages");
};

struct Ctrl {
  uint64_t full[12], empty[12];
  int abort;  // a wait ran out: no other waits any more
  int id[64];
  float scale[64];
};

template <typename T, int R, int J>
__global__ void __launch_bounds__(kThreads, 1)
    project_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                   const T* b, int64_t sl, int64_t sr, const void* ids, int ids64, Scale scale, const float* low, int L, int M, int K,
                   int N, int r, T* y, int64_t ldy, int32_t* status) {
  using Q = Cfg<R, J>;
  constexpr int BM = Q::BM, C = Q::C, BKS = Q::BKS, NT = Q::NT, kStages = Q::kStages;
  constexpr int kSliceBytes = BM * 128;
  extern __shared__ char smem_raw[];
  char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* slots = base + kStages * kStageBytes;
  float* red = reinterpret_cast<float*>(slots + kStages * Q::kSlotBytes);
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(base + Q::kBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&ctrl->full[s]), 1);
      mbar_init(smem_u32(&ctrl->empty[s]), kConsumers);
    }
    ctrl->abort = 0;
    fence_mbar_init();
  }
  const int mb = blockIdx.y * NT, Mt = min(NT, M - mb);  // this CTA's rows of x
  for (int m = tid; m < Mt; m += kThreads) {
    const int i = id_at(ids, ids64, mb + m, L);
    ctrl->id[m] = i;
    ctrl->scale[m] = i >= 0 ? scale.of(i) : 0.0f;
  }
  __syncthreads();
  const int blocks = (N + BM - 1) / BM;
  int stage = 0;
  uint32_t phase = 0;
  volatile int* abort_flag = &ctrl->abort;

  if (warp == 0) {
    if (lane == 0) {
      for (int blk = blockIdx.x; blk < blocks; blk += gridDim.x)
        for (int c = 0; c < K; c += BKS) {
          const uint32_t full = smem_u32(&ctrl->full[stage]);
          if (!mbar_wait(smem_u32(&ctrl->empty[stage]), phase ^ 1, abort_flag))
            return give_up(abort_flag, status, MOE_ERR_TIMEOUT);
          mbar_arrive_expect_tx(full, kStageBytes + Q::kSlotBytes);
          const uint32_t dst = smem_u32(base + stage * kStageBytes);
          const uint32_t xdst = smem_u32(slots + stage * Q::kSlotBytes);
#pragma unroll
          for (int i = 0; i < C; ++i) {
            tma_load_2d(dst + i * kSliceBytes, &wmap, full, c + 64 * i, blk * BM);
            tma_load_2d(xdst + i * NT * 128, &xmap, full, c + 64 * i, mb);
          }
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
    }
    return;
  }
  const int cw = warp - 1, rt = cw % R, cs = cw / R, g8 = lane >> 2, q4 = lane & 3;
  const uint32_t a_base = smem_u32(base) + cs * kSliceBytes + (rt * 16 + g8) * 128;
  const uint32_t b_base = smem_u32(slots) + (cs * NT + g8) * 128;
  const uint32_t off0 = ((2 * q4) ^ g8) * 16, off1 = ((2 * q4 + 1) ^ g8) * 16;
  bool waited = false;
  // A thread whose wait has run out carries on with what is there, without further waits, so
  // that every warp still comes to the barriers below.
  bool failed = false;
  for (int blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    float acc[J][4];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    for (int c = 0; c < K; c += BKS) {
      if (!failed && !mbar_wait(smem_u32(&ctrl->full[stage]), phase, abort_flag)) {
        failed = true;
        give_up(abort_flag, status, MOE_ERR_TIMEOUT);
      }
      __syncwarp();
      uint32_t a[2][8];  // rows g8 and g8 + 8, 16 columns each
      const uint32_t sa = a_base + stage * kStageBytes;
      ld_shared_v4(sa + off0, &a[0][0]);
      ld_shared_v4(sa + off1, &a[0][4]);
      ld_shared_v4(sa + 1024 + off0, &a[1][0]);
      ld_shared_v4(sa + 1024 + off1, &a[1][4]);
      uint32_t v[J][8];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint32_t sb = b_base + stage * Q::kSlotBytes + j * 1024;
        ld_shared_v4(sb + off0, &v[j][0]);
        ld_shared_v4(sb + off1, &v[j][4]);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s)  // J independent sums between two products of one
#pragma unroll
        for (int j = 0; j < J; ++j)
          mma<T>(acc[j], a[0][2 * s], a[1][2 * s], a[0][2 * s + 1], a[1][2 * s + 1], v[j][2 * s],
                 v[j][2 * s + 1]);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctrl->empty[stage]));
      if (++stage == kStages) stage = 0, phase ^= 1;
    }
    float* rb = red + cw * (NT * kRedStride);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        rb[(j * 8 + 2 * q4 + (i & 1)) * kRedStride + g8 + 8 * (i >> 1)] = acc[j][i];
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (!waited) wait_for_previous_kernel();  // for `low`
    waited = true;
    const int tid_c = cw * 32 + lane;
    // At most 8 requests of low rank, or fewer of a high one, by rows of B (their latency
    // counts); more by columns of W (their loads do: 8 rows of 2048 x 8192 at rank 64 19 us
    // so and 22 by rows of B; 1 row at rank 128, 18.7 and 13.2).
    const bool by_rows = J == 1 && Mt * r <= 256;
    if (by_rows) {
      // The adapters' part is added to the first slice's sums, 512 bytes of neighbouring rows of
      // one request's B a warp, 16 bytes a lane, 2^lg lanes a row, four of those under way.
      constexpr int kTogether = 4;
      const int lg = r <= 8 ? 0 : 32 - __clz((r / 8) - 1), lanes = 1 << lg, rows = 32 >> lg;
      const int chunks = rows < BM ? BM / rows : 1, piece = lane & (lanes - 1);
      for (int u0 = cw; u0 < Mt * chunks; u0 += kTogether * kConsumers) {
        float add[kTogether];
        int at[kTogether];
        float c[kTogether];
#pragma unroll
        for (int q = 0; q < kTogether; ++q) {
          const int u = u0 + q * kConsumers, m = u / chunks, n = u % chunks * rows + (lane >> lg);
          const int i = m < Mt ? ctrl->id[m] : -1, row = blk * BM + n;
          const bool there = i >= 0 && n < BM && row < N;
          uint4 ub = make_uint4(0, 0, 0, 0);
          float4 l0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), l1 = l0;
          if (there && piece * 8 < r) {
            ub = *reinterpret_cast<const uint4*>(b + i * sl + row * sr + piece * 8);
            const float* lr = low + (mb + m) * r + piece * 8;
            l0 = *reinterpret_cast<const float4*>(lr);
            l1 = *reinterpret_cast<const float4*>(lr + 4);
          }
          add[q] = dot8<T>(ub, l0, l1);
          at[q] = there && piece == 0 ? n / 16 * (NT * kRedStride) + m * kRedStride + n % 16 : -1;
          c[q] = there ? ctrl->scale[m] : 0.0f;
        }
#pragma unroll
        for (int q = 0; q < kTogether; ++q) {
          for (int o = 1; o < lanes; o <<= 1) add[q] += __shfl_xor_sync(0xffffffffu, add[q], o);
          if (at[q] >= 0) red[at[q]] += c[q] * add[q];
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    // One column of W a thread (row n of the block) and every 256 / BM-th row of x, eight of
    // them at a time, so that their adapters' rows are under way together.
    constexpr int kStep = 32 * kConsumers / BM, kTogether = 8;
    const int n = tid_c % BM, row = blk * BM + n;
    if (row < N)
      for (int m0 = tid_c / BM; m0 < Mt; m0 += kTogether * kStep) {
        float add[kTogether];
        if (!by_rows) {
          const T* br[kTogether];
          const float* lr[kTogether];
#pragma unroll
          for (int u = 0; u < kTogether; ++u) {
            const int m = m0 + u * kStep, i = m < Mt ? ctrl->id[m] : -1;
            br[u] = i >= 0 ? b + i * sl + row * sr : nullptr;
            lr[u] = low + (mb + m) * r;
            add[u] = 0.0f;
          }
#pragma unroll 2
          for (int j = 0; j < r; j += 8) {
            uint4 ub[kTogether];
#pragma unroll
            for (int u = 0; u < kTogether; ++u)
              ub[u] = br[u] != nullptr ? *reinterpret_cast<const uint4*>(br[u] + j) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int u = 0; u < kTogether; ++u)
              if (br[u] != nullptr)
                add[u] += dot8<T>(ub[u], *reinterpret_cast<const float4*>(lr[u] + j),
                                  *reinterpret_cast<const float4*>(lr[u] + j + 4));
          }
        }
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
          const int m = m0 + u * kStep;
          if (m >= Mt) continue;
          float v = 0.0f;
#pragma unroll
          for (int i = 0; i < C; ++i)
            v += red[(i * R + n / 16) * (NT * kRedStride) + m * kRedStride + n % 16];
          if (!by_rows && ctrl->id[m] >= 0) v += ctrl->scale[m] * add[u];
          y[(mb + m) * ldy + row] = from_f<T>(v);
        }
      }
    asm volatile("bar.sync 1, 256;" ::: "memory");  // the buffer is free again
  }
}

template <typename T, int R, int J>
int project(const T* x, int64_t ldx, const void* weight, int64_t ldw, Weights b, const void* ids, int ids64,
            Scale scale, const float* low, int L, int m, int k, int n, int r, T* y, int64_t ldy,
            int32_t* status, int sms, cudaStream_t stream) {
  using Q = Cfg<R, J>;
  CUtensorMap wmap, xmap;
  const CUtensorMapDataType dt = std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t wdims[2] = {uint64_t(k), uint64_t(n)}, wstrides[1] = {uint64_t(ldw) * 2};
  const uint64_t xdims[2] = {uint64_t(k), uint64_t(m)}, xstrides[1] = {uint64_t(ldx) * 2};
  const uint32_t wbox[2] = {64, Q::BM}, xbox[2] = {64, Q::NT};
  int rc = encode_tiled(&wmap, dt, 2, weight, wdims, wstrides, wbox);
  if (rc == MOE_OK) rc = encode_tiled(&xmap, dt, 2, x, xdims, xstrides, xbox);
  if (rc != MOE_OK) return rc;
  constexpr auto kern = &project_kernel<T, R, J>;
  constexpr int kSmem = 1024 + Q::kBytes + int(sizeof(Ctrl));
  static_assert(kSmem <= 227 * 1024, "shared memory");
  if (!allow_shared_memory<kern>(kSmem)) return MOE_ERR_CUDA;
  const int blocks = (n + Q::BM - 1) / Q::BM;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks < sms ? blocks : sms, (m + Q::NT - 1) / Q::NT);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, wmap, xmap, static_cast<const T*>(b.p), b.stride_l, b.stride_row, ids,
                            ids64, scale, low, L, m, k, n, r, y, ldy, status) == cudaSuccess
             ? MOE_OK
             : MOE_ERR_CUDA;
}

// Weights with at least so many rows are taken 64 at a time.
constexpr int64_t kWide = 64 * 100;

template <typename T>
int forward(const void* x, int64_t ldx, const void* weight, int64_t ldw, Weights a, Weights b, const void* ids,
            int ids64, Scale scale, int m, int k, int n, int L, int r, void* y, int64_t ldy, float* low,
            int32_t* status, int sms, cudaStream_t stream) {
  low_kernel<T><<<dim3((r + kLowWarps - 1) / kLowWarps, m), 32 * kLowWarps, 0, stream>>>(
      static_cast<const T*>(x), ldx, static_cast<const T*>(a.p), a.stride_l, a.stride_row, ids, ids64, L, k, r,
      low, status);
  if (cudaGetLastError() != cudaSuccess) return MOE_ERR_CUDA;
  auto go = [&](auto rr, auto jj) {
    return project<T, decltype(rr)::value, decltype(jj)::value>(
        static_cast<const T*>(x), ldx, weight, ldw, b, ids, ids64, scale, low, L, m, k, n, r,
        static_cast<T*>(y), ldy, status, sms, stream);
  };
  auto by_width = [&](auto rr, auto wide) {
    using std::integral_constant;
    if (m <= 8) return go(rr, integral_constant<int, 1>());
    if (m <= 16) return go(rr, integral_constant<int, 2>());
    if (m <= 24) return go(wide, integral_constant<int, 3>());
    if (m <= 32) return go(wide, integral_constant<int, 4>());
    if (m <= 48) return go(wide, integral_constant<int, 6>());
    return go(wide, integral_constant<int, 8>());
  };
  // row_block(): the widest row blocks that still give most SMs one; with more rows of x the
  // narrow ones would leave too few stages of shared memory.
  using std::integral_constant;
  if (n >= kWide) return by_width(integral_constant<int, 4>(), integral_constant<int, 4>());
  if (n >= kWide / 2) return by_width(integral_constant<int, 2>(), integral_constant<int, 2>());
  return by_width(integral_constant<int, 1>(), integral_constant<int, 2>());
}

}  // namespace few

bool takes_few_rows(int64_t m, int64_t k, int64_t n, int rank, int sms) {
  // The rows of x and the adapters' products cost each block of W; the tensor-core path is
  // faster from about here on.  Measured, here and there, 8 adapters: 2048 x 2048, 48 rows of
  // rank 64 18.5 and 22.6 us, 64 rows 22.6 and 22.6; 512 x 1024, 32 rows of rank 128 16.5
  // and 26.4; 8192 x 1024, 48 rows of rank 16 22.6 and 24.7, 64 rows 27.0 and 24.7.
  const bool wide = n >= few::kWide;
  const int64_t rows = m < 64 ? m : 64;
  if (rows * (k + 96 * rank) >= (int64_t(1) << 19)) return false;
  // Wide weights have that epilogue on every SM.
  if (wide && rows * rank > 2048) return false;
  if (m <= 64) return true;
  // Further tiles of 64 rows read the weight again, from L2: worth it for one block an SM
  // (2048 x 2048 at rank 16, 128 rows: 12.7 and 22.0 us, 192 rows: 20.6 and 19.3), while
  // x A^T, by the CUDA cores, stays small.
  const int64_t blocks = (m + 63) / 64 * ((n + (wide ? 63 : 31)) / (wide ? 64 : 32));
  return blocks <= sms && m * rank * k <= (int64_t(1) << 25);
}

int forward_few_rows(const void* x, int64_t ldx, const void* weight, int64_t ldw, Weights a, Weights b,
                     const void* ids, int ids64, Scale scale, int dtype, int m, int k, int n, int adapters,
                     int rank, void* y, int64_t ldy, float* low, int32_t* status, cudaStream_t stream) {
  int dev;
  DeviceInfo info;
  const int rc = current_device_info(&dev, &info);
  if (rc != MOE_OK) return rc;
  if (info.major != 10) return MOE_ERR_UNSUPPORTED;
  auto fn = dtype == MOE_DTYPE_BF16 ? &few::forward<__nv_bfloat16> : &few::forward<__half>;
  return fn(x, ldx, weight, ldw, a, b, ids, ids64, scale, m, k, n, adapters, rank, y, ldy, low, status,
            info.sm_count, stream);
}

}  // namespace lora
}  // namespace moe
