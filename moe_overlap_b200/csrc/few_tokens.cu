// The routed-experts layer for a few tokens on sm_100a: gate, top-k, up-projection
// with exact GELU, down-projection and weighted sum.
//
//   z = x Wg^T + bias;  p = softmax(z);  idx = the k largest z (ties: lower id);
//   w = p[idx] (/ their sum);
//   h[t,j] = gelu(x[t] W1[idx]^T);  out[t] = sum_j w[t,j] (h[t,j] W2[idx]^T)
//
// (the routed path of src/train_moe_baseline.py:315-441 at decode batch sizes).
// A slot with expert -1 adds nothing; a token without any expert gets zeros.
// Sums are fp32, h is rounded to the input type (the matrix operand of the second
// product, as in the layer's own path), the output is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/moe_overlap.h"
#include "host_common.h"
#include "ptx.cuh"

namespace moe {
namespace few {

constexpr int kMaxTokens = 128;
constexpr int kMaxE = 256;
constexpr int kMaxK = 16;
constexpr int kWarps = 8;

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value)
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

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Dot product of two rows of `n` elements (a multiple of 8, 16-byte aligned) over one
// warp; every 8 products (exact in fp32 for bf16 and fp16) are summed in Acc.
template <typename T, typename Acc>
__device__ __forceinline__ Acc warp_dot(const T* a, const T* b, int n, int lane) {
  Acc s = 0;
  for (int i = lane * 8; i < n; i += 256) {
    const uint4 ua = *reinterpret_cast<const uint4*>(a + i);
    const uint4 ub = *reinterpret_cast<const uint4*>(b + i);
    const T* pa = reinterpret_cast<const T*>(&ua);
    const T* pb = reinterpret_cast<const T*>(&ub);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += static_cast<Acc>(to_f(pa[j]) * to_f(pb[j]));
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
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 32 * i < E) s += expf(static_cast<float>(v[i] - m));
  s = warp_sum(s);
  uint32_t taken = 0;  // bit i: this lane's expert i is taken
  float my_w = 0.0f, wsum = 0.0f;
  int my_e = 0;
  for (int j = 0; j < k; ++j) {
    double best = -INFINITY;
    int be = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      if (e < E && !(taken >> i & 1u) && (be == 0x7fffffff || v[i] > best)) {
        best = v[i];
        be = e;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, best, o);
      const int oe = __shfl_xor_sync(0xffffffffu, be, o);
      if (oe != 0x7fffffff && (be == 0x7fffffff || ob > best || (ob == best && oe < be))) {
        best = ob;
        be = oe;
      }
    }
    if ((be & 31) == lane) taken |= 1u << (be >> 5);
    const float p = expf(static_cast<float>(best - m)) / s;
    wsum += p;
    if (lane == j) {
      my_w = p;
      my_e = be;
    }
  }
  if (lane < k) {
    idx_out[lane] = my_e;
    w_out[lane] = renorm ? my_w / wsum : my_w;
  }
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarps)
    gate_kernel(const T* x, int64_t ldx, const T* rw, int64_t ldr, const float* bias, int H, int E,
                int k, int renorm, int64_t* idx, float* w) {
  __shared__ double z[kMaxE];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x;
  for (int e = warp; e < E; e += kWarps) {
    const double d = warp_dot<T, double>(x + t * ldx, rw + e * ldr, H, lane);
    if (lane == 0) z[e] = bias != nullptr ? d + static_cast<double>(bias[e]) : d;
  }
  __syncthreads();
  if (warp == 0) warp_topk(z, E, k, renorm != 0, lane, idx + int64_t(t) * k, w + int64_t(t) * k);
}

__device__ __forceinline__ int slot_expert(const int64_t* idx, int slot, int E, int32_t* status) {
  const int64_t e = idx[slot];
  if (e < -1 || e >= E) {
    record_status(status, MOE_ERR_INVALID_ARG);
    return -1;
  }
  return static_cast<int>(e);
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarps)
    up_kernel(const T* x, int64_t ldx, const T* w1, int64_t w1_se, int64_t w1_sr, const int64_t* idx,
              int H, int F, int E, int k, T* h, int32_t* status) {
  const int lane = threadIdx.x & 31, f = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int slot = blockIdx.y, e = slot_expert(idx, slot, E, status);
  if (f >= F || e < 0) return;
  const float a = warp_dot<T, float>(x + (slot / k) * ldx, w1 + e * w1_se + f * w1_sr, H, lane);
  if (lane == 0)
    h[int64_t(slot) * F + f] = from_f<T>(0.5f * a * (1.0f + erff(a * 0.70710678118654752440f)));
}

template <typename T>
__global__ void __launch_bounds__(32 * kWarps)
    down_kernel(const T* h, const T* w2, int64_t w2_se, int64_t w2_sr, const int64_t* idx,
                const float* w, int H, int F, int E, int k, T* out, int64_t ldo) {
  const int lane = threadIdx.x & 31, col = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int t = blockIdx.y;
  if (col >= H) return;
  float s = 0.0f;
  for (int j = 0; j < k; ++j) {
    const int slot = t * k + j, e = slot_expert(idx, slot, E, nullptr);
    if (e >= 0)
      s += w[slot] * warp_dot<T, float>(h + int64_t(slot) * F, w2 + e * w2_se + col * w2_sr, F, lane);
  }
  if (lane == 0) out[t * ldo + col] = from_f<T>(s);
}

template <typename T>
int launch(const void* x, int64_t ldx, const void* rw, int64_t ldr, const float* bias,
           const void* w1, int64_t w1_se, int64_t w1_sr, const void* w2, int64_t w2_se,
           int64_t w2_sr, int T_, int H, int F, int E, int k, int renorm, int64_t* idx, float* w,
           void* out, int64_t ldo, void* ws, int32_t* status, cudaStream_t s) {
  const T* xt = static_cast<const T*>(x);
  if (rw != nullptr)
    gate_kernel<T><<<T_, 32 * kWarps, 0, s>>>(xt, ldx, static_cast<const T*>(rw), ldr, bias, H, E, k,
                                              renorm, idx, w);
  T* h = static_cast<T*>(ws);
  up_kernel<T><<<dim3((F + kWarps - 1) / kWarps, T_ * k), 32 * kWarps, 0, s>>>(
      xt, ldx, static_cast<const T*>(w1), w1_se, w1_sr, idx, H, F, E, k, h, status);
  down_kernel<T><<<dim3((H + kWarps - 1) / kWarps, T_), 32 * kWarps, 0, s>>>(
      h, static_cast<const T*>(w2), w2_se, w2_sr, idx, w, H, F, E, k, static_cast<T*>(out), ldo);
  return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

}  // namespace few
}  // namespace moe

namespace {
bool sizes_ok(int32_t num_tokens, int32_t hidden, int32_t ffn, int32_t num_experts, int32_t topk) {
  using namespace moe::few;
  return num_tokens >= 0 && num_tokens <= kMaxTokens && hidden >= 8 && hidden % 8 == 0 && ffn >= 8 &&
         ffn % 8 == 0 && num_experts >= 1 && num_experts <= kMaxE && topk >= 1 && topk <= kMaxK &&
         topk <= num_experts;
}
bool rows_ok(const void* p, int64_t ld, int64_t width) {
  return p != nullptr && moe::aligned16(p) && ld >= width && ld % 8 == 0;
}
}  // namespace

extern "C" int64_t moe_few_tokens_workspace(int32_t num_tokens, int32_t hidden, int32_t ffn,
                                            int32_t num_experts, int32_t topk) {
  if (!sizes_ok(num_tokens, hidden, ffn, num_experts, topk)) return -1;
  return int64_t(num_tokens) * topk * ffn * 2;
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
  auto fn = dtype == MOE_DTYPE_BF16 ? &moe::few::launch<__nv_bfloat16> : &moe::few::launch<__half>;
  return fn(x, ldx, router_w, ldr, router_bias, w1, w1_stride_e, w1_stride_row, w2, w2_stride_e,
            w2_stride_row, num_tokens, hidden, ffn, num_experts, topk, renormalize, topk_idx,
            topk_weights, out, ldo, workspace, status, static_cast<cudaStream_t>(stream));
}
