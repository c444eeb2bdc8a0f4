// The tensor-core kernels of dt_kv_prompt.cu as dt_kv.cu calls them.
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

#include "dt_kv.cuh"

namespace dtb {

// Offsets into the workspace, and the CTAs that share the work.
struct KvPromptPlan {
    int ctas;
    size_t out, stats, list, starts, prefix, bytes;
};

struct KvColumnPlan {
    int ctas;
    size_t blocks, sums, list, starts, prefix, bytes;
};

KvPromptPlan kv_prompt_plan(int64_t batch, int64_t rows, int64_t head_dim, int sms);

// Attention of many query rows, head_dim up to 128. lse2 (or null): [batch * kv_heads][rows], log2 of each row's sum.
int kv_prompt_attention(const KvAttnArgs& a, int code, const KvPromptPlan& plan, void* workspace, float* lse2,
                        cudaStream_t stream);

KvColumnPlan kv_column_plan(int64_t batch, int64_t kv_heads, int64_t rows, int64_t head_dim, int64_t capacity, int sms);

// a.weights from the rows' log2 sums, head_dim up to 128. workspace: the plan's own bytes.
int kv_column_sums(const KvAttnArgs& a, int code, const KvColumnPlan& plan, void* workspace, const float* lse2,
                   cudaStream_t stream);

}  // namespace dtb
