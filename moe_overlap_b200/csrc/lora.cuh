// Declarations shared by the adapters' kernels (lora.cu, lora_few.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace moe {
namespace lora {

// One number for each adapter, or one for all.
struct Scale {
  const float* each;
  float all;
  __device__ float of(int i) const { return each != nullptr ? each[i] : all; }
};

struct Weights {  // of all adapters
  const void* p;
  int64_t stride_l, stride_row;
};

// Whether a batch of which no gradient is wanted takes the kernels of lora_few.cu on a
// device of `sms` SMs.
bool takes_few_rows(int64_t m, int64_t k, int64_t n, int rank, int sms);

// y = x weight^T + scale (x a^T) b^T by row for such a batch; low: float [m][rank].
int forward_few_rows(const void* x, int64_t ldx, const void* weight, int64_t ldw, Weights a, Weights b,
                     const void* ids, int ids64, Scale scale, int dtype, int m, int k, int n, int adapters,
                     int rank, void* y, int64_t ldy, float* low, int32_t* status, cudaStream_t stream);

}  // namespace lora
}  // namespace moe
