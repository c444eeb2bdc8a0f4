#include "kv_cache.h"

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

namespace dtb {

namespace {

void Check(int status, const char* where) {
    if (status == DT_OK) return;
    TORCH_CHECK_VALUE(status != DT_ERR_INVALID, where, ": ", dt_last_error_message());
    TORCH_CHECK(false, where, ": ", dt_status_string(status), " (", dt_last_error_message(), ")");
}

int Dtype(torch::ScalarType t, const char* where) {
    switch (t) {
        case torch::kBFloat16: return DT_BFLOAT16;
        case torch::kHalf: return DT_FLOAT16;
        case torch::kFloat: return DT_FLOAT32;
        default: TORCH_CHECK_TYPE(false, where, ": unsupported dtype ", t);
    }
}

// The cache's device holds everything else, and the call runs there.
void CheckPlace(const QuantizedKVCache& c, const torch::Tensor& t, const char* where, const char* name) {
    TORCH_CHECK_VALUE(t.device() == c.key.device(), where, ": ", name, " is on ", t.device(), ", the cache on ",
                      c.key.device());
}

void CheckInts(const QuantizedKVCache& c, const torch::Tensor& t, const char* where, const char* name) {
    TORCH_CHECK_VALUE(t.scalar_type() == torch::kInt && t.dim() == 1 && t.size(0) == c.abi.batch && t.is_contiguous(),
                      where, ": ", name, " must be a contiguous int32 tensor of (", c.abi.batch, ",)");
    CheckPlace(c, t, where, name);
}

void CheckNoGrad(const torch::Tensor& t, const char* where) {
    TORCH_CHECK(!(t.requires_grad() && torch::GradMode::is_enabled()), where,
                ": no backward pass through an 8-bit cache; call it under torch.no_grad()");
    TORCH_CHECK(!t._fw_grad(0).defined(), where, ": no forward-mode derivative through an 8-bit cache; pass the primal");
}

// (N, H, T, E) rows of the model's type, E contiguous.
void CheckRows(const QuantizedKVCache& c, const torch::Tensor& t, const char* where, const char* name) {
    TORCH_CHECK_TYPE(t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kHalf, where, ": ", name,
                     " must be bfloat16 or float16");
    TORCH_CHECK_VALUE(t.dim() == 4 && t.size(0) == c.abi.batch && t.size(3) == c.abi.head_dim, where, ": ", name,
                      " must be (", c.abi.batch, ", heads, tokens, ", c.abi.head_dim, ")");
    CheckPlace(c, t, where, name);
    CheckNoGrad(t, where);
}

}  // namespace

void KVCacheCheckRows(const std::vector<const QuantizedKVCache*>& caches, const std::vector<torch::Tensor>& rows,
                      const std::vector<std::vector<int64_t>>& shapes, const std::string& where, const std::string& name) {
    TORCH_CHECK_VALUE(caches.size() == rows.size() && caches.size() == shapes.size(), where, ": ", name, " is of ", rows.size(),
                      " devices, the cache of ", caches.size());
    for (size_t i = 0; i < rows.size(); ++i) {
        CheckRows(*caches[i], rows[i], where.c_str(), name.c_str());
        TORCH_CHECK_VALUE(rows[i].sizes() == at::IntArrayRef(shapes[i]), where, ": ", name, " is ", rows[i].sizes(),
                          " on one device, not ", at::IntArrayRef(shapes[i]));
    }
}

namespace {

torch::Tensor InnerContiguous(const torch::Tensor& t) { return t.stride(3) == 1 ? t : t.contiguous(); }

void CheckWeights(const QuantizedKVCache& c, const torch::Tensor& t, const char* where) {
    TORCH_CHECK_VALUE(t.scalar_type() == torch::kFloat && t.dim() == 3 && t.size(0) == c.abi.batch &&
                          t.size(1) == c.abi.kv_heads && t.size(2) == c.abi.capacity && t.is_contiguous(),
                      where, ": weights must be a contiguous float32 tensor of (", c.abi.batch, ", ", c.abi.kv_heads, ", ",
                      c.abi.capacity, ")");
    CheckPlace(c, t, where, "weights");
}

void* Stream(const torch::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

void CheckCuda(const QuantizedKVCache& c, const char* where) {
    TORCH_CHECK_VALUE(c.key.is_cuda(), where, ": the cache is on ", c.key.device(), "; it is served on cuda devices only");
}

}  // namespace

QuantizedKVCache::QuantizedKVCache(torch::Tensor k, torch::Tensor v, torch::Tensor ks, torch::Tensor vs)
    : key(std::move(k)), value(std::move(v)), keyScale(std::move(ks)), valueScale(std::move(vs)), abi{} {
    const char* w = "QuantizedKVCache";
    TORCH_CHECK_TYPE(key.scalar_type() == torch::kChar || key.scalar_type() == torch::kFloat8_e4m3fn, w,
                     ": codes must be int8 or float8_e4m3fn");
    TORCH_CHECK_VALUE(key.dim() == 4 && key.sizes() == value.sizes() && key.scalar_type() == value.scalar_type(), w,
                      ": key and value must be (batch, heads, capacity, head_dim) of one shape and type");
    TORCH_CHECK_VALUE(keyScale.scalar_type() == torch::kFloat && valueScale.scalar_type() == torch::kFloat &&
                          keyScale.dim() == 3 && keyScale.sizes() == valueScale.sizes() &&
                          keyScale.size(0) == key.size(0) && keyScale.size(1) == key.size(1),
                      w, ": scales must be float32 (batch, heads, capacity / block)");
    const int64_t capacity = key.size(2), nblocks = keyScale.size(2);
    TORCH_CHECK_VALUE(nblocks > 0 && capacity % nblocks == 0, w, ": the capacity must be a multiple of the block");
    for (const auto* t : {&key, &value, &keyScale, &valueScale}) {
        TORCH_CHECK_VALUE(t->is_contiguous() && t->device() == key.device(), w,
                          ": codes and scales must be contiguous and on one device");
    }
    abi.batch = key.size(0);
    abi.kv_heads = key.size(1);
    abi.capacity = capacity;
    abi.head_dim = key.size(3);
    abi.block = capacity / nblocks;
    abi.code = key.scalar_type() == torch::kChar ? DT_KV_INT8 : DT_KV_E4M3;
    abi.key = key.data_ptr();
    abi.value = value.data_ptr();
    abi.key_scale = keyScale.data_ptr<float>();
    abi.value_scale = valueScale.data_ptr<float>();
    size_t unused = 0;
    Check(dt_kv_evict_workspace(&abi, 0, &unused), w);  // the C ABI's own checks of the cache
}

QuantizedKVCache QuantizedKVCache::Empty(int64_t batch, int64_t kvHeads, int64_t capacity, int64_t headDim,
                                         torch::ScalarType dtype, int64_t block, torch::Device device) {
    TORCH_CHECK_VALUE(block == 32 || block == 64 || block == 128, "QuantizedKVCache: block must be 32, 64 or 128 tokens");
    TORCH_CHECK_VALUE(capacity > 0 && capacity % block == 0,
                      "QuantizedKVCache: the capacity must be a positive multiple of the block");
    const auto codes = torch::TensorOptions().dtype(dtype).device(device);
    const auto scales = torch::TensorOptions().dtype(torch::kFloat).device(device);
    TORCH_CHECK_TYPE(dtype == torch::kChar || dtype == torch::kFloat8_e4m3fn,
                     "QuantizedKVCache: codes must be int8 or float8_e4m3fn");
    return QuantizedKVCache(torch::zeros({batch, kvHeads, capacity, headDim}, codes),
                            torch::zeros({batch, kvHeads, capacity, headDim}, codes),
                            torch::zeros({batch, kvHeads, capacity / block}, scales),
                            torch::zeros({batch, kvHeads, capacity / block}, scales));
}

void KVCacheAppend(const QuantizedKVCache& c, const torch::Tensor& key, const torch::Tensor& value,
                   const torch::Tensor& lengths, const std::optional<torch::Tensor>& counts) {
    const char* w = "kv_cache_append";
    CheckRows(c, key, w, "key");
    CheckRows(c, value, w, "value");
    TORCH_CHECK_VALUE(key.sizes() == value.sizes() && key.size(1) == c.abi.kv_heads, w, ": key and value must be (",
                      c.abi.batch, ", ", c.abi.kv_heads, ", tokens, ", c.abi.head_dim, ")");
    TORCH_CHECK_TYPE(key.scalar_type() == value.scalar_type(), w, ": key and value differ in type");
    CheckInts(c, lengths, w, "lengths");
    if (counts) CheckInts(c, *counts, w, "counts");
    CheckCuda(c, w);
    const c10::cuda::CUDAGuard guard(c.key.device());
    const auto k = InnerContiguous(key), v = InnerContiguous(value);
    Check(dt_kv_append(&c.abi, k.data_ptr(), v.data_ptr(), k.size(2), k.strides().data(), v.strides().data(),
                       Dtype(k.scalar_type(), w), lengths.data_ptr<int32_t>(),
                       counts ? counts->data_ptr<int32_t>() : nullptr, Stream(c.key)),
          w);
}

std::tuple<torch::Tensor, torch::Tensor> KVCacheRead(const QuantizedKVCache& c, const torch::Tensor& lengths,
                                                     const std::optional<torch::Tensor>& first, int64_t firstAll,
                                                     int64_t count, torch::ScalarType dtype) {
    const char* w = "kv_cache_read";
    CheckInts(c, lengths, w, "lengths");
    if (first) CheckInts(c, *first, w, "first");
    TORCH_CHECK_VALUE(count >= 0, w, ": count must not be negative");
    const int code = Dtype(dtype, w);
    CheckCuda(c, w);
    const c10::cuda::CUDAGuard guard(c.key.device());
    const auto opts = torch::TensorOptions().dtype(dtype).device(c.key.device());
    auto key = torch::empty({c.abi.batch, c.abi.kv_heads, count, c.abi.head_dim}, opts);
    auto value = torch::empty_like(key);
    Check(dt_kv_read(&c.abi, lengths.data_ptr<int32_t>(), first ? first->data_ptr<int32_t>() : nullptr, firstAll, count,
                     key.data_ptr(), value.data_ptr(), code, Stream(c.key)),
          w);
    return {key, value};
}

std::tuple<torch::Tensor, torch::Tensor> KVCacheAttention(const torch::Tensor& query, const QuantizedKVCache& c,
                                                          const torch::Tensor& lengths,
                                                          const std::optional<torch::Tensor>& counts, bool isCausal,
                                                          double scale, const std::optional<torch::Tensor>& weights,
                                                          bool accumulate, bool wantLse) {
    const char* w = "kv_cache_attention";
    CheckRows(c, query, w, "query");
    TORCH_CHECK_VALUE(query.size(1) > 0 && query.size(1) % c.abi.kv_heads == 0, w, ": query heads (", query.size(1),
                      ") must be a multiple of the key heads (", c.abi.kv_heads, ")");
    CheckInts(c, lengths, w, "lengths");
    if (counts) CheckInts(c, *counts, w, "counts");
    if (weights) CheckWeights(c, *weights, w);
    CheckCuda(c, w);
    const c10::cuda::CUDAGuard guard(c.key.device());
    const auto q = InnerContiguous(query);
    const int64_t heads = q.size(1), tokens = q.size(2);
    auto out = torch::empty({c.abi.batch, heads, tokens, c.abi.head_dim}, q.options().requires_grad(false));
    torch::Tensor lse;
    if (wantLse) lse = torch::empty({c.abi.batch, heads, tokens}, out.options().dtype(torch::kFloat));
    size_t bytes = 0;
    Check(dt_kv_attention_workspace(&c.abi, heads, tokens, weights.has_value(), &bytes), w);
    const auto ws = torch::empty({static_cast<int64_t>(bytes)}, out.options().dtype(torch::kByte));
    Check(dt_kv_attention(&c.abi, q.data_ptr(), heads, tokens, q.strides().data(), Dtype(q.scalar_type(), w),
                          lengths.data_ptr<int32_t>(), counts ? counts->data_ptr<int32_t>() : nullptr,
                          static_cast<float>(scale),
                          (isCausal ? DT_KV_CAUSAL : 0) | (weights && accumulate ? DT_KV_ACCUMULATE : 0), out.data_ptr(),
                          wantLse ? lse.data_ptr<float>() : nullptr, weights ? weights->data_ptr<float>() : nullptr,
                          ws.data_ptr(), bytes, Stream(c.key)),
          w);
    return {out, lse};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> KVCacheEvict(const QuantizedKVCache& c,
                                                                     const torch::Tensor& lengths,
                                                                     const torch::Tensor& weights, int64_t budget,
                                                                     int64_t recent, const QuantizedKVCache& out) {
    const char* w = "kv_cache_evict";
    CheckInts(c, lengths, w, "lengths");
    CheckWeights(c, weights, w);
    CheckPlace(c, out.key, w, "out");
    TORCH_CHECK_VALUE(budget >= 0 && budget <= out.abi.capacity, w, ": budget must be 0..", out.abi.capacity);
    TORCH_CHECK_VALUE(recent >= 0 && recent <= budget, w, ": recent must be 0..budget");
    CheckCuda(c, w);
    const c10::cuda::CUDAGuard guard(c.key.device());
    auto outLengths = torch::empty_like(lengths);
    auto outWeights = torch::empty({c.abi.batch, c.abi.kv_heads, out.abi.capacity}, weights.options());
    auto kept = torch::empty({c.abi.batch, c.abi.kv_heads, budget}, lengths.options());
    Check(dt_kv_evict(&c.abi, &out.abi, lengths.data_ptr<int32_t>(), weights.data_ptr<float>(), budget, recent,
                      outLengths.data_ptr<int32_t>(), outWeights.data_ptr<float>(),
                      budget > 0 ? kept.data_ptr<int32_t>() : nullptr, nullptr, 0, Stream(c.key)),
          w);
    return {outLengths, outWeights, kept};
}

}  // namespace dtb
