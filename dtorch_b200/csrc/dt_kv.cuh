// Device helpers of the 8-bit key/value cache (dt_kv.cu, dt_kv_prompt.cu).
#pragma once

#include <cstdint>
#include <string>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../../include/dtorch_b200.h"
#include "dt_internal.h"

namespace dtb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Maxima of scores begin at the least finite number rather than -infinity: differences of two of them are not NaN, and a
// score of -infinity less one is -infinity.
constexpr float kNothing = -3.402823466e38f;

// What the attention kernels read. Query row r of key head h is query r / group of the sequence and query head
// h * group + r % group: rows in the order of the tokens, so the rows of a tile see nearly the same tokens.
struct KvAttnArgs {
    const uint8_t* key;
    const uint8_t* value;
    const float* key_scale;
    const float* value_scale;
    const void* query;
    const int32_t* lengths;
    const int32_t* counts;
    void* out;
    float* lse;
    float* weights;
    int64_t q_stride_n, q_stride_h, q_stride_t;
    int batch, kv_heads, head_dim, group, tokens, rows;  // rows = group * tokens
    int64_t capacity;
    int block_shift;   // log2(tokens that share a scale)
    int nblocks;       // capacity >> block_shift
    float scale_log2;  // softmax scale * log2(e)
    int causal;
    int query_bf16;
    int accumulate;
    int q_vec;  // query rows can be read 16 bytes at a time
};

// At the top of every kernel of the cache, in every thread: the next kernel of the stream may be set up from now on (it
// waits here too), and what this one reads was written by kernels that have ended. A call is several short kernels;
// this takes 1 to 2 us off each step from one to the next.
__device__ __forceinline__ void enter_kernel() {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ int kv_length(const int32_t* lengths, int n, int64_t capacity) {
    const int l = lengths[n];
    return l < 0 ? 0 : (l > capacity ? static_cast<int>(capacity) : l);
}

__device__ __forceinline__ int kv_count(const int32_t* counts, int n, int tokens) {
    if (counts == nullptr) return tokens;
    const int c = counts[n];
    return c < 0 ? 0 : (c > tokens ? tokens : c);
}

// How many tokens, from the first, query row `row` of a sequence sees.
__device__ __forceinline__ int kv_limit(const KvAttnArgs& a, int row, int len, int cnt) {
    const int t = row / a.group;
    if (row >= a.rows || t >= cnt) return 0;
    const int lim = a.causal ? len - cnt + t + 1 : len;
    return lim < 0 ? 0 : lim;
}

// A row's sum of weights, by which its outputs are divided. 0 is that of a row that sees nothing, whose outputs are 0; a row
// that sees nothing but scores of -infinity has it too, but no softmax: NaN.
__device__ __forceinline__ float row_sum(float l, bool sees) { return l == 0.0f && sees ? __int_as_float(0x7fc00000) : l; }

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}

__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// Four codes of a word to two fp16 pairs; every code is exact in fp16. SPLIT 0: pairs (0,1) and (2,3); SPLIT 1: pairs
// (0,2) and (1,3), the byte transposition that rows read through ldmatrix.trans need.
// int8: 1024 + (code + 128) is the fp16 whose low byte is code + 128; subtracting 1152 leaves the code; the transposition
// costs nothing. e4m3: the conversion instruction, which runs at the rate of a byte permutation (2 cycles a warp, measured).
template <bool E4M3, int SPLIT>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (E4M3) {
        if (SPLIT) w = prmt(w, 0u, 0x3120);
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        const uint32_t u = w ^ 0x80808080u;
        lo = hsub2(prmt(u, 0x64646464u, SPLIT ? 0x4240 : 0x4140), 0x64806480u);
        hi = hsub2(prmt(u, 0x64646464u, SPLIT ? 0x4341 : 0x4342), 0x64806480u);
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// Two 16-bit floats of a word as fp32.
__device__ __forceinline__ float2 unpack16(uint32_t w, bool bf16) {
    if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Power of two that brings a row whose largest |element| is `amax` into fp16's range, and its inverse. bf16 and fp16
// elements stay exact above 2^-38 of the row's largest, below that the error is under 2^-39 of it: the products are
// those of the model's type, and one fp16 path serves both types.
__device__ __forceinline__ void row_power(float amax, float& mul, float& inv) {
    int ex = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
    ex = ex < -100 ? -100 : ex;
    mul = __uint_as_float(static_cast<uint32_t>(127 + 13 - ex) << 23);
    inv = __uint_as_float(static_cast<uint32_t>(127 - 13 + ex) << 23);
}

// 8 N elements of a query row from element `e` on, as words of two; zeros where there is no row and behind head_dim. All
// loads are issued before any is used.
template <int N>
__device__ __forceinline__ void load_row(const KvAttnArgs& a, const uint16_t* p, int e, uint32_t* x) {
#pragma unroll
    for (int j = 0; j < 4 * N; ++j) x[j] = 0;
    if (p == nullptr) return;
    if (a.q_vec) {
#pragma unroll
        for (int c = 0; c < N; ++c)
            if (e + c * 8 < a.head_dim) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + e + c * 8));
                x[c * 4] = u.x, x[c * 4 + 1] = u.y, x[c * 4 + 2] = u.z, x[c * 4 + 3] = u.w;
            }
    } else {
#pragma unroll
        for (int j = 0; j < 4 * N; ++j)
            if (e + 2 * j < a.head_dim) x[j] = p[e + 2 * j] | (static_cast<uint32_t>(p[e + 2 * j + 1]) << 16);
    }
}

// Largest |element| of words of two.
template <int N>
__device__ __forceinline__ float row_max(const KvAttnArgs& a, const uint32_t* x) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float2 f = unpack16(x[j], a.query_bf16);
        m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
    return m;
}

// Launch of a kernel that begins with enter_kernel, behind whatever stands in the stream; in clusters of `cluster` CTAs.
template <typename... P, typename... A>
int launch_kernel(const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                  unsigned cluster, A... args) {
    // Above 48 KB with the kernel's static shared memory, of which those that take both have less than 16 KB. Per device and
    // cheap: the limit belongs to the kernel in the current context.
    if (smem > 32 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return set_error(DT_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
    }
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
    if (e != cudaSuccess) return set_error(DT_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
    return check_launch(what);
}

}  // namespace dtb
