// The 8-bit key/value cache over torch tensors: argument checks, output and workspace allocation, the current
// stream of the tensors' device; the work is dt_kv_* of the C ABI.
#pragma once

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include <torch/torch.h>

#include "../../../include/dtorch_b200.h"

namespace dtb {

class QuantizedKVCache {
   public:
    QuantizedKVCache(torch::Tensor key, torch::Tensor value, torch::Tensor keyScale, torch::Tensor valueScale);
    static QuantizedKVCache Empty(int64_t batch, int64_t kvHeads, int64_t capacity, int64_t headDim,
                                  torch::ScalarType dtype, int64_t block, torch::Device device);

    torch::Tensor key, value, keyScale, valueScale;
    dt_kv_cache abi;
};

// What append and attention ask of rows of tokens by themselves, of several caches at once: type, shape, place, no
// gradient.
void KVCacheCheckRows(const std::vector<const QuantizedKVCache*>& caches, const std::vector<torch::Tensor>& rows,
                      const std::vector<std::vector<int64_t>>& shapes, const std::string& where, const std::string& name);

void KVCacheAppend(const QuantizedKVCache& cache, const torch::Tensor& key, const torch::Tensor& value,
                   const torch::Tensor& lengths, const std::optional<torch::Tensor>& counts);

std::tuple<torch::Tensor, torch::Tensor> KVCacheRead(const QuantizedKVCache& cache, const torch::Tensor& lengths,
                                                     const std::optional<torch::Tensor>& first, int64_t firstAll,
                                                     int64_t count, torch::ScalarType dtype);

std::tuple<torch::Tensor, torch::Tensor> KVCacheAttention(const torch::Tensor& query, const QuantizedKVCache& cache,
                                                          const torch::Tensor& lengths,
                                                          const std::optional<torch::Tensor>& counts, bool isCausal,
                                                          double scale, const std::optional<torch::Tensor>& weights,
                                                          bool accumulate, bool wantLse);

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> KVCacheEvict(const QuantizedKVCache& cache,
                                                                     const torch::Tensor& lengths,
                                                                     const torch::Tensor& weights, int64_t budget,
                                                                     int64_t recent, const QuantizedKVCache& out);

}  // namespace dtb
