// Low-rank adapters of many requests beside a shared projection, on sm_100a.
//
//   y[m] = x[m] W^T + scale[i] (x[m] A[i]^T) B[i]^T,   i = ids[m] (-1: no adapter)
//
// The shared product is the grouped GEMM of one expert; the kernels here add the
// adapters' part and form its gradients.  Rows are taken in adapter order through a
// permutation, so each adapter is read once per block of its rows:
//   plan    perm (the rows with an adapter, by adapter, in row order) and offs
//   shrink  s[p] = x[perm[p]] A[i]^T           (also dy B[i], with B read along rows)
//   expand  y[perm[p]] += scale[i] s[p] B[i]^T (also dx += scale[i] (dy B[i]) A[i])
//   grad    dB[i] = scale[i] sum_p dy[perm[p]]^T s[p]  (also dA[i])
// s is held in fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/moe_overlap.h"
#include "host_common.h"
#include "ptx.cuh"

namespace moe {
namespace lora {

constexpr int kMaxAdapters = 1024;
constexpr int kMaxRank = 128;

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return __bfloat162float(v);
  else
    return __half2float(v);
}
template <typename T>
__device__ __forceinline__ T from_f(float v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return __float2bfloat16_rn(v);
  else
    return __float2half_rn(v);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Adapter of sorted place p: the last i with offs[i] <= p.
__device__ __forceinline__ int adapter_of(const int32_t* offs, int L, int p) {
  int lo = 0, hi = L - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (offs[mid] <= p)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// One block per adapter: it counts the rows of smaller adapters (its segment's start)
// and writes its own rows in order.  No block depends on another and the order is
// always the same.
__global__ void __launch_bounds__(1024) plan_kernel(const void* ids, int ids64, int M, int L,
                                                    int32_t* perm, int32_t* offs, int32_t* base_offs,
                                                    int32_t* status) {
  __shared__ int less[32], equal[32];
  const int i = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto id_at = [&](int m) -> int {
    const int64_t v = ids64 ? static_cast<const int64_t*>(ids)[m]
                            : static_cast<int64_t>(static_cast<const int32_t*>(ids)[m]);
    if (v < -1 || v >= L) {
      if (i == 0) record_status(status, MOE_ERR_INVALID_ARG);
      return -1;
    }
    return static_cast<int>(v);
  };
  const int per = ((M + 31) / 32 + 31) / 32 * 32;  // rows of a warp
  const int m0 = warp * per, m1 = min(M, m0 + per);
  int nl = 0, ne = 0;
  for (int m = m0 + lane; m < m1; m += 32) {
    const int v = id_at(m);
    nl += v >= 0 && v < i;
    ne += v == i;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    nl += __shfl_xor_sync(0xffffffffu, nl, o);
    ne += __shfl_xor_sync(0xffffffffu, ne, o);
  }
  if (lane == 0) less[warp] = nl, equal[warp] = ne;
  __syncthreads();
  int start = 0, at = 0, all = 0;
  for (int k = 0; k < 32; ++k) {
    start += less[k];
    at += k < warp ? equal[k] : 0;
    all += equal[k];
  }
  if (threadIdx.x == 0) {
    offs[i] = start;
    if (i == L - 1) offs[L] = start + all;
    if (i == 0) base_offs[0] = 0, base_offs[1] = M;
  }
  at += start;
  for (int b = m0; b < m1; b += 32) {
    const bool mine = b + lane < m1 && id_at(b + lane) == i;
    const unsigned votes = __ballot_sync(0xffffffffu, mine);
    if (mine) perm[at + __popc(votes & ((1u << lane) - 1u))] = b + lane;
    at += __popc(votes);
  }
}

// s[p][j] = sum_k x[perm[p]][k] W_i(j, k): one warp an element.  W_i(j, k) is at
// w + i*sl + j*sr + k, or with kT at w + i*sl + k*sr + j.
template <typename T, bool kT>
__global__ void __launch_bounds__(256) shrink_kernel(const T* x, int64_t ldx, const T* w, int64_t sl,
                                                     int64_t sr, const int32_t* perm,
                                                     const int32_t* offs, int L, int K, int r, float* s) {
  const int64_t e = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, j = static_cast<int>(e % r);
  const int64_t p = e / r;
  if (p >= offs[L]) return;
  const T* xr = x + perm[p] * ldx;
  const T* wi = w + adapter_of(offs, L, static_cast<int>(p)) * sl;
  float v = 0.0f;
  for (int k = lane; k < K; k += 32) v += to_f(xr[k]) * to_f(kT ? wi[k * sr + j] : wi[j * sr + k]);
  v = warp_sum(v);
  if (lane == 0) s[p * r + j] = v;
}

// y[perm[p]][n] += scale[i] sum_j s[p][j] W_i(n, j): one thread an element.  W_i(n, j)
// is at w + i*sl + n*sr + j, or with kT at w + i*sl + j*sr + n.
template <typename T, bool kT>
__global__ void __launch_bounds__(256) expand_kernel(const float* s, const T* w, int64_t sl, int64_t sr,
                                                     const float* scale, const int32_t* perm,
                                                     const int32_t* offs, int L, int N, int r, T* y,
                                                     int64_t ldy) {
  const int n = blockIdx.y * 256 + threadIdx.x;
  const int p = blockIdx.x;
  if (p >= offs[L] || n >= N) return;
  const int i = adapter_of(offs, L, p);
  const T* wi = w + i * sl;
  float v = 0.0f;
  for (int j = 0; j < r; ++j) v += s[int64_t(p) * r + j] * to_f(kT ? wi[j * sr + n] : wi[n * sr + j]);
  T* at = y + perm[p] * ldy + n;
  *at = from_f<T>(to_f(*at) + scale[i] * v);
}

// g_i(n, j) = scale[i] sum_p s[p][j] z[perm[p]][n] over adapter i's rows (zeros without
// rows), at g + i*gl + n*gr + j, or with kT at g + i*gl + j*gr + n.
template <typename T, bool kT>
__global__ void __launch_bounds__(256) grad_kernel(const float* s, const T* z, int64_t ldz,
                                                   const float* scale, const int32_t* perm,
                                                   const int32_t* offs, int n, int r, T* g, int64_t gl,
                                                   int64_t gr) {
  const int col = blockIdx.x * 256 + threadIdx.x, j = blockIdx.y, i = blockIdx.z;
  if (col >= n) return;
  float v = 0.0f;
  for (int p = offs[i]; p < offs[i + 1]; ++p) v += s[int64_t(p) * r + j] * to_f(z[perm[p] * ldz + col]);
  g[i * gl + (kT ? j * gr + col : col * gr + j)] = from_f<T>(scale[i] * v);
}

}  // namespace lora
}  // namespace moe

using namespace moe;

namespace {
bool dims_ok(int32_t dtype, int64_t m, int64_t n, int32_t adapters, int32_t rank) {
  return (dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F16) && m >= 0 && m <= INT32_MAX / 2 && n >= 8 &&
         n % 8 == 0 && n <= INT32_MAX / 2 && adapters >= 1 && adapters <= lora::kMaxAdapters && rank >= 8 &&
         rank % 8 == 0 && rank <= lora::kMaxRank;
}
// Adapter weights: rows of `width` at 16-byte starts, one adapter after another.
bool weights_ok(const void* w, int64_t stride_l, int64_t stride_row, int64_t rows, int64_t width,
                int32_t adapters) {
  return w != nullptr && aligned16(w) && stride_row >= width && stride_row % 8 == 0 &&
         (adapters == 1 || (stride_l % 8 == 0 && stride_l >= (rows - 1) * stride_row + width));
}
bool rows_ok(const void* p, int64_t ld, int64_t width) {
  return p != nullptr && aligned16(p) && ld >= width && ld % 8 == 0;
}
int launched() { return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA; }
}  // namespace

extern "C" int32_t moe_lora_plan(const void* ids, int32_t ids_int64, int64_t m, int32_t adapters,
                                 int32_t* perm, int32_t* offs, int32_t* base_offs, int32_t* status,
                                 void* stream) {
  if (m < 0 || m > INT32_MAX / 2 || adapters < 1 || adapters > lora::kMaxAdapters || offs == nullptr ||
      base_offs == nullptr || (m > 0 && (ids == nullptr || perm == nullptr)))
    return MOE_ERR_INVALID_ARG;
  lora::plan_kernel<<<adapters, 1024, 0, static_cast<cudaStream_t>(stream)>>>(
      ids, ids_int64, static_cast<int>(m), adapters, perm, offs, base_offs, status);
  return launched();
}

extern "C" int32_t moe_lora_shrink(const void* x, int64_t ldx, const void* w, int64_t w_stride_l,
                                   int64_t w_stride_row, int32_t w_transposed, const int32_t* perm,
                                   const int32_t* offs, int32_t dtype, int64_t m, int64_t k,
                                   int32_t adapters, int32_t rank, float* s, void* stream) {
  if (!dims_ok(dtype, m, k, adapters, rank)) return MOE_ERR_INVALID_ARG;
  if (m == 0) return MOE_OK;
  if (!rows_ok(x, ldx, k) || perm == nullptr || offs == nullptr || s == nullptr || !aligned16(s) ||
      !(w_transposed ? weights_ok(w, w_stride_l, w_stride_row, k, rank, adapters)
                     : weights_ok(w, w_stride_l, w_stride_row, rank, k, adapters)))
    return MOE_ERR_INVALID_ARG;
  auto go = [&](auto t, auto tr) {
    using T = decltype(t);
    lora::shrink_kernel<T, decltype(tr)::value>
        <<<static_cast<unsigned>((m * rank + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(x), ldx, static_cast<const T*>(w), w_stride_l, w_stride_row, perm,
            offs, adapters, static_cast<int>(k), rank, s);
  };
  if (dtype == MOE_DTYPE_BF16)
    w_transposed ? go(__nv_bfloat16(), std::true_type()) : go(__nv_bfloat16(), std::false_type());
  else
    w_transposed ? go(__half(), std::true_type()) : go(__half(), std::false_type());
  return launched();
}

extern "C" int32_t moe_lora_expand(const float* s, const void* w, int64_t w_stride_l,
                                   int64_t w_stride_row, int32_t w_transposed, const float* scale,
                                   const int32_t* perm, const int32_t* offs, int32_t dtype, int64_t m,
                                   int64_t n, int32_t adapters, int32_t rank, void* y, int64_t ldy,
                                   void* stream) {
  if (!dims_ok(dtype, m, n, adapters, rank)) return MOE_ERR_INVALID_ARG;
  if (m == 0) return MOE_OK;
  if (!rows_ok(y, ldy, n) || perm == nullptr || offs == nullptr || scale == nullptr || s == nullptr ||
      !aligned16(s) ||
      !(w_transposed ? weights_ok(w, w_stride_l, w_stride_row, rank, n, adapters)
                     : weights_ok(w, w_stride_l, w_stride_row, n, rank, adapters)))
    return MOE_ERR_INVALID_ARG;
  auto go = [&](auto t, auto tr) {
    using T = decltype(t);
    lora::expand_kernel<T, decltype(tr)::value>
        <<<dim3(static_cast<unsigned>(m), static_cast<unsigned>((n + 255) / 256)), 256, 0,
           static_cast<cudaStream_t>(stream)>>>(s, static_cast<const T*>(w), w_stride_l, w_stride_row,
                                                scale, perm, offs, adapters, static_cast<int>(n), rank,
                                                static_cast<T*>(y), ldy);
  };
  if (dtype == MOE_DTYPE_BF16)
    w_transposed ? go(__nv_bfloat16(), std::true_type()) : go(__nv_bfloat16(), std::false_type());
  else
    w_transposed ? go(__half(), std::true_type()) : go(__half(), std::false_type());
  return launched();
}

extern "C" int32_t moe_lora_grad(const float* s, const void* z, int64_t ldz, const float* scale,
                                 const int32_t* perm, const int32_t* offs, int32_t dtype, int64_t m,
                                 int64_t n, int32_t adapters, int32_t rank, void* g, int64_t g_stride_l,
                                 int64_t g_stride_row, int32_t g_transposed, void* stream) {
  if (!dims_ok(dtype, m, n, adapters, rank)) return MOE_ERR_INVALID_ARG;
  if (offs == nullptr || scale == nullptr ||
      (m > 0 && (!rows_ok(z, ldz, n) || perm == nullptr || s == nullptr || !aligned16(s))) ||
      !(g_transposed ? weights_ok(g, g_stride_l, g_stride_row, rank, n, adapters)
                     : weights_ok(g, g_stride_l, g_stride_row, n, rank, adapters)))
    return MOE_ERR_INVALID_ARG;
  auto go = [&](auto t, auto tr) {
    using T = decltype(t);
    lora::grad_kernel<T, decltype(tr)::value>
        <<<dim3(static_cast<unsigned>((n + 255) / 256), rank, adapters), 256, 0,
           static_cast<cudaStream_t>(stream)>>>(s, static_cast<const T*>(z), ldz, scale, perm, offs,
                                                static_cast<int>(n), rank, static_cast<T*>(g),
                                                g_stride_l, g_stride_row);
  };
  if (dtype == MOE_DTYPE_BF16)
    g_transposed ? go(__nv_bfloat16(), std::true_type()) : go(__nv_bfloat16(), std::false_type());
  else
    g_transposed ? go(__half(), std::true_type()) : go(__half(), std::false_type());
  return launched();
}
