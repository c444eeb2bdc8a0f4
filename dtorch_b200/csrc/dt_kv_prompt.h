// The tensor-core kernels of dt_kv_prompt.cu as dt_kv.cu calls them.
#pragma once

#include <cuda_runtime.h>

#include "dt_kv.cuh"

namespace dtb {

// Attention of many query rows, head_dim up to 128. lse2 (or null): [batch * kv_heads][rows], log2 of each row's sum.
int kv_prompt_attention(const KvAttnArgs& a, int code, float* lse2, cudaStream_t stream);

}  // namespace dtb
