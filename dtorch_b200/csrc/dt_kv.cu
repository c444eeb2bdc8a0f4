// The 8-bit key/value cache of include/dtorch_b200.h: append, read, attention of few query rows, eviction, and the host
// entry points.

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include <cooperative_groups.h>

#include "dt_internal.h"
#include "dt_kv.cuh"
#include "dt_kv_prompt.h"

using namespace dtb;

namespace {

// ---------------------------------------------------------------------------------------------------------------
// Quantisation
// ---------------------------------------------------------------------------------------------------------------
constexpr float kNan = __builtin_nanf("");

// amax / limit, up to the next bfloat16. amax has at most 15 significant bits, so unless the quotient is a bfloat16
// itself it is much further from one than fp32's rounding of it: the result is that of the exact quotient.
template <bool E4M3>
__device__ __forceinline__ float scale_of(float amax) {
    const float s = amax / (E4M3 ? 448.0f : 127.0f);
    return __uint_as_float((__float_as_uint(s) + 0xffffu) & 0xffff0000u);
}

// Codes of four values x / s, to nearest, ties to even, of the exact quotient. The scale has 8 significant bits and the
// values at most 15, so an exact quotient that is not half way between two codes is well away from there, and a product
// with the rounded reciprocal r (off by 2^-24 of itself, so by less than 2^-17) only has to be put back on the half way
// points that it stands for, which costs a third of a division:
//   int8: a quotient in [2^j, 2^(j+1)) that is no half way point is 2^(j-15) away from one, 2^-16 at least. Adding and
//   taking off 128 rounds to multiples of 2^-16; half way points are such multiples.
//   e4m3: half way points have 5 significant bits and others differ by 2^-13 of themselves; rounding to 18 bits restores them.
// Scales below 2^-100, whose reciprocals may not be normal, take the division.
template <bool E4M3>
__device__ __forceinline__ uint32_t pack_codes(const float* y) {
    if constexpr (E4M3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    } else {
        uint32_t q[4];  // 1.5 * 2^23 more: the integer, ties to even, in the low byte
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = __float_as_uint(y[i] + 12582912.0f);
        return prmt(prmt(q[0], q[1], 0x0040), prmt(q[2], q[3], 0x0040), 0x5410);
    }
}

template <bool E4M3>
__device__ __noinline__ uint32_t encode4_divided(float a, float b, float c, float d, float s) {
    const float y[4] = {a / s, b / s, c / s, d / s};
    return pack_codes<E4M3>(y);
}

template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(const float* x, float s, float r) {
    if (!(s >= 0x1p-100f)) return s > 0.0f ? encode4_divided<E4M3>(x[0], x[1], x[2], x[3], s) : 0;  // 0: all zero; NaN: marked
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = E4M3 ? __uint_as_float((__float_as_uint(x[i] * r) + 0x20u) & ~0x3fu)
                    : copysignf(fmaf(fabsf(x[i]), r, 128.0f) - 128.0f, x[i]);
    return pack_codes<E4M3>(y);
}

__device__ __forceinline__ float reciprocal(float s) { return s >= 0x1p-100f ? 1.0f / s : 0.0f; }

// The four codes of a word as fp32 (without the scale).
template <bool E4M3>
__device__ __forceinline__ void decode4(uint32_t w, float* v) {
    uint32_t lo, hi;
    codes_to_half<E4M3, 0>(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    v[0] = a.x;
    v[1] = a.y;
    v[2] = b.x;
    v[3] = b.y;
}

struct KvAppendArgs {
    uint8_t* codes[2];
    float* scales[2];
    const uint16_t* src[2];
    int64_t stride[2][3];
    bool vec[2];
    const int32_t* lengths;
    const int32_t* counts;
    int64_t capacity;
    int heads, head_dim, tokens, block_shift, spans;
    bool bf16;
};

constexpr int kAppendThreads = 256;

// One block of the cache (`block` tokens of a head, keys or values) per CTA: largest |x| of the new tokens, the
// block's scale, their codes; where the scale grows, the earlier tokens' codes again. The new tokens stay in registers
// between the two passes (VPT vectors of 8 elements a thread), so every element is read once. The largest |x| is
// taken on the bit patterns: it also finds infinities and NaN, which a floating maximum would drop. Bound by the chain of
// a CTA (length, tokens, largest, codes) against what six CTAs an SM have under way: 2 x 8191 tokens of 8 heads of 128,
// 101 MB in and out, 30 us, 3.4 TB/s; one token of 32 sequences 5 us.
template <bool E4M3, int VPT>
__global__ void __launch_bounds__(kAppendThreads) k_kv_append(KvAppendArgs a) {
    enter_kernel();
    const int tid = threadIdx.x;
    unsigned b = blockIdx.x;
    const int i = static_cast<int>(b % a.spans);
    b /= a.spans;
    const int kv = static_cast<int>(b & 1);
    b >>= 1;
    const int h = static_cast<int>(b % a.heads);
    const int n = static_cast<int>(b / a.heads);
    const int len = kv_length(a.lengths, n, a.capacity);
    const int cnt = kv_count(a.counts, n, a.tokens);
    const int block = 1 << a.block_shift;
    const int64_t slot = (static_cast<int64_t>(len >> a.block_shift) + i) << a.block_shift;  // first token of the block
    const int64_t end = min(min(slot + block, static_cast<int64_t>(len) + cnt), a.capacity);
    const int64_t begin = max(slot, static_cast<int64_t>(len));
    if (begin >= end) return;
    const int held = static_cast<int>(begin - slot);
    const int fresh = static_cast<int>(end - begin);
    const int cpr = a.head_dim >> 3;  // vectors of 8 elements in a row
    const size_t head = static_cast<size_t>(n) * a.heads + h;
    uint8_t* dst = a.codes[kv] + (head * a.capacity + slot) * a.head_dim;
    float* scale = a.scales[kv] + head * (a.capacity >> a.block_shift) + (slot >> a.block_shift);
    const uint16_t* src = a.src[kv] + n * a.stride[kv][0] + h * a.stride[kv][1] + (begin - len) * a.stride[kv][2];

    uint32_t x[VPT][4];
    uint32_t most = 0;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int idx = v * kAppendThreads + tid;
        x[v][0] = x[v][1] = x[v][2] = x[v][3] = 0;
        if (idx < fresh * cpr) {
            const int t = idx / cpr;
            const uint16_t* p = src + t * a.stride[kv][2] + (idx - t * cpr) * 8;
            if (a.vec[kv]) {
                const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
                x[v][0] = u.x, x[v][1] = u.y, x[v][2] = u.z, x[v][3] = u.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[v][j] = p[2 * j] | (static_cast<uint32_t>(p[2 * j + 1]) << 16);
            }
        }
    }
    const float old = held > 0 ? *scale : 0.0f;
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) most = __vmaxu2(most, x[v][j] & 0x7fff7fffu);
    most = max(most & 0xffffu, most >> 16);
    __shared__ uint32_t part[kAppendThreads / 32];
    most = __reduce_max_sync(0xffffffffu, most);
    if ((tid & 31) == 0) part[tid >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) most = max(most, part[w]);
    float s = old;
    if (most >= (a.bf16 ? 0x7f80u : 0x7c00u)) {
        s = kNan;
    } else {
        const float now = scale_of<E4M3>(unpack16(most, a.bf16).x);
        if (now > s) s = now;  // an old NaN stays
    }
    if (tid == 0) *scale = s;
    const float r = reciprocal(s);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int idx = v * kAppendThreads + tid;
        if (idx < fresh * cpr) {
            uint32_t q[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 lo = unpack16(x[v][2 * j], a.bf16);
                const float2 hi = unpack16(x[v][2 * j + 1], a.bf16);
                const float f[4] = {lo.x, lo.y, hi.x, hi.y};
                q[j] = encode4<E4M3>(f, s, r);
            }
            *reinterpret_cast<uint2*>(dst + static_cast<size_t>(held) * a.head_dim + static_cast<size_t>(idx) * 8) =
                make_uint2(q[0], q[1]);
        }
    }
    if (held > 0 && s > old) {
        for (int idx = tid; idx < held * cpr; idx += kAppendThreads) {
            uint2* p = reinterpret_cast<uint2*>(dst) + idx;
            const uint2 w = *p;
            float f[8];
            decode4<E4M3>(w.x, f);
            decode4<E4M3>(w.y, f + 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= old;
            *p = make_uint2(encode4<E4M3>(f, s, r), encode4<E4M3>(f + 4, s, r));
        }
    }
}

struct KvReadArgs {
    const uint8_t* codes[2];
    const float* scales[2];
    void* out[2];
    const int32_t* lengths;
    const int32_t* first;
    int64_t first_all, count, capacity, all_heads;
    int heads, head_dim, block_shift;
    int dtype;
};

// Vectors of 8 elements: 8 bytes of codes in, 16 or 32 bytes out. A thread keeps its column and takes every 256 /
// (vectors in a row)-th token of a head, kReadRows of them at a time: 102 MB in 28 us, 3.6 TB/s, with 16 bytes stored a
// lane (32 bytes a lane in two halves took 45).
constexpr int kReadRows = 4;

template <bool E4M3>
__global__ void __launch_bounds__(256) k_kv_read(KvReadArgs a) {
    enter_kernel();
    const int kv = blockIdx.y;
    if (a.out[kv] == nullptr) return;
    const int cpr = a.head_dim >> 3, step = 256 / cpr;
    const int r = threadIdx.x / cpr, c = threadIdx.x - r * cpr;
    if (r >= step) return;
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * step * kReadRows + r;
    for (int64_t head = blockIdx.z; head < a.all_heads; head += gridDim.z) {
        const int n = static_cast<int>(head / a.heads);
        const int len = kv_length(a.lengths, n, a.capacity);
        const int64_t first = a.first != nullptr ? a.first[n] : a.first_all;
        const uint8_t* const codes = a.codes[kv] + head * a.capacity * a.head_dim + c * 8;
        const float* const scales = a.scales[kv] + head * (a.capacity >> a.block_shift);
        uint2 w[kReadRows];
        float s[kReadRows];
#pragma unroll
        for (int u = 0; u < kReadRows; ++u) {
            const int64_t i = i0 + u * step, t = first + i;
            w[u] = make_uint2(0, 0);
            s[u] = 0.0f;
            if (i < a.count && t >= 0 && t < len) {
                w[u] = __ldg(reinterpret_cast<const uint2*>(codes + t * a.head_dim));
                s[u] = __ldg(scales + (t >> a.block_shift));
            }
        }
#pragma unroll
        for (int u = 0; u < kReadRows; ++u) {
            const int64_t i = i0 + u * step;
            if (i >= a.count) break;
            float f[8];
            decode4<E4M3>(w[u].x, f);
            decode4<E4M3>(w[u].y, f + 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= s[u];
            const int64_t at = (head * a.count + i) * cpr + c;
            if (a.dtype == DT_FLOAT32) {
                float4* o = reinterpret_cast<float4*>(a.out[kv]) + at * 2;
                o[0] = make_float4(f[0], f[1], f[2], f[3]);
                o[1] = make_float4(f[4], f[5], f[6], f[7]);
            } else {
                uint32_t q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (a.dtype == DT_BFLOAT16) {
                        const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                        q[j] = *reinterpret_cast<const uint32_t*>(&p);
                    } else {
                        q[j] = pack_half2(f[2 * j], f[2 * j + 1]);
                    }
                }
                reinterpret_cast<uint4*>(a.out[kv])[at] = make_uint4(q[0], q[1], q[2], q[3]);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Attention of few query rows (single tokens, drafts)
// ---------------------------------------------------------------------------------------------------------------
// 8 or 16 query rows of a key head against tiles of 128 tokens. The tiles of all (sequence, head, row tile) items stand
// in one list, and every CTA takes an equal stretch of it, whatever the lengths: a stretch may end one item and begin the
// next. An item inside one stretch is finished there; the others leave (running maximum, sum, unnormalised output) in
// the workspace, and k_kv_merge joins them in the order of the list.
//
// Within a CTA each of the four warps streams its own 32 tokens of every tile through shared memory with cp.async and
// keeps its own softmax state: no barrier inside the loop; the four states are joined once per item.
// Scores and outputs use mma.m16n8k16 with fp16 operands: this path is bound by reading the cache, and up to 16 rows would
// leave most of a tcgen05 tile empty. Keys and values are the 16-row operand and the query rows the 8 columns (S^T = K Q^T,
// O^T = V^T P^T), so that 8 rows, the common group of heads, fill the instruction. Which elements share a k16 step is free
// as long as queries and keys agree, so a lane takes 16 consecutive bytes of a key row, enough for four steps.
// 32 ragged sequences of up to 8192 tokens, 8 heads of 128 (268 MB): 52 us, 5.2 TB/s; with queries as the 16-row operand
// 78 us, and 89 with e4m3 codes turned by shifts and masks. What is left: two stages of 8 KB a warp, 12 warps an SM.
constexpr int kTile = 128;
constexpr int kWarpTokens = 32;
constexpr int kAttnThreads = 128;
// A weight is rounded to fp16 as 2^(x - top + 10), top the largest score of the row in the warp's slice: 11 significant
// bits down to 2^-24 of the slice's largest. What the slice's largest is to the row's goes into the value scale, in fp32.
constexpr float kShift = 10.0f;

struct KvPartials {
    float* out;     // [slot][row tile's rows][EP]
    float2* stats;  // [slot][row tile's rows]: maximum (log2), sum
    float* scores;  // [batch * kv_heads][row tile's rows][capacity] log2 scores, or null
    float* lse2;    // [batch * kv_heads][rows]: log2 of the sum of 2^score
};

// NT: column tiles of 8 query rows.
template <int EP, int NT>
struct AttnShape {
    static constexpr int kRows = 8 * NT;
    static constexpr int kChunks = EP / 16;
    static constexpr int kStages = EP == 64 ? 3 : 2;
    static constexpr int kCtas = EP == 64 ? 4 : EP == 128 ? 3 : 1;  // on an SM
    static constexpr int kSliceBytes = kWarpTokens * EP;            // keys, or values, of one warp's tokens
    static constexpr int kStageBytes = 2 * kSliceBytes;
    static constexpr int kWarpBytes = kStages * kStageBytes;
    static constexpr int kScaleBytes = 4 * kStages * 2 * 4;         // after the four warps' stages
    static constexpr int kSmem = 4 * kWarpBytes + kScaleBytes + 4 * kRows * 8 + 64;
    static constexpr int kJoin = EP + 8;  // floats between rows in the join: no two rows of a store meet in a bank
    static_assert(kWarpBytes >= kRows * kJoin * 4, "the outputs of an item's join reuse a warp's stages");
};

// Byte offset of 16-byte chunk `c` of row `r`: chunks are permuted within 128 bytes so that neither the key reads (two
// rows of four chunks a phase) nor the value reads (eight rows of one chunk) meet in a bank.
template <int EP>
__device__ __forceinline__ int swizzled(int r, int c) {
    if constexpr (EP == 64) {
        const int line = r >> 1;
        return line * 128 + (((((r & 1) << 2) | c) ^ (line & 3)) << 4);
    } else {
        const int f = ((r & 1) << 2) | ((r >> 1) & 3);
        return r * EP + ((c & ~7) << 4) + (((c & 7) ^ f) << 4);
    }
}

__device__ __forceinline__ void cp_async16(uint32_t smem, const void* gmem, bool live) {
    const int bytes = live ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(bytes) : "memory");
}

__device__ __forceinline__ void cp_async4(uint32_t smem, const void* gmem) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem), "l"(gmem) : "memory");
}

__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Address of query row `row` (of a key head) of a sequence, or null outside.
__device__ __forceinline__ const uint16_t* query_row(const KvAttnArgs& a, int n, int h, int row) {
    if (row >= a.rows) return nullptr;
    const int t = row / a.group, j = row - t * a.group;
    return static_cast<const uint16_t*>(a.query) + n * a.q_stride_n +
           static_cast<int64_t>(h * a.group + j) * a.q_stride_h + t * a.q_stride_t;
}

// The B fragments of 8 query rows as fp16: registers [kc * 8 + step * 2 + i], 64-wide span kc, fragment register i. The
// lane's row is row0 + lane / 4; the inverse of the row's power of two goes to inv[0], inv[1] for the rows 2 c and 2 c + 1
// (c = lane % 4), the columns that the lane has of an accumulator.
template <int EP>
__device__ __forceinline__ void load_query(const KvAttnArgs& a, int n, int h, int row0, uint32_t* q, float* inv) {
    const int lane = threadIdx.x & 31, c = lane & 3;
    const uint16_t* p = query_row(a, n, h, row0 + (lane >> 2));
    uint32_t x[EP / 8];
#pragma unroll
    for (int kc = 0; kc < EP / 64; ++kc) load_row<2>(a, p, kc * 64 + c * 16, x + kc * 8);
    float amax = row_max<EP / 8>(a, x);
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    float mul, mine;
    row_power(amax, mul, mine);
#pragma unroll
    for (int j = 0; j < EP / 8; ++j) {
        // words 2 s and 2 s + 1 of the lane's 16 elements are step s's k rows (2c, 2c + 1) and (2c + 8, 2c + 9)
        const float2 f = unpack16(x[j], a.query_bf16);
        q[j] = pack_half2(f.x * mul, f.y * mul);
    }
    inv[0] = __shfl_sync(0xffffffffu, mine, c * 8);
    inv[1] = __shfl_sync(0xffffffffu, mine, c * 8 + 4);
}

// The 8 x 8 matrix of 16-bit elements that the warp's words hold, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
    return d;
}

// Four fp32 of an output row in the query's type.
__device__ __forceinline__ uint2 pack_out(float4 v, float g, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x * g, v.y * g), hi = __floats2bfloat162_rn(v.z * g, v.w * g);
        return make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
    return make_uint2(pack_half2(v.x * g, v.y * g), pack_half2(v.z * g, v.w * g));
}

// Tiles of a sequence of `len` tokens: at least one, so that an empty sequence's outputs are written too.
__device__ __forceinline__ int tiles_of(int len) { return len <= 0 ? 1 : (len + kTile - 1) / kTile; }

// Position of tile `x` of the list. All threads of the warp call it; n = batch if x is behind the end.
struct TilePos {
    int n;         // sequence
    int item;      // (head, row tile) within the sequence
    int tile;      // within the item
    int64_t base;  // list position of the sequence's first tile
};

__device__ __forceinline__ TilePos find_tile(const KvAttnArgs& a, int per_seq, int64_t x) {
    const int lane = threadIdx.x & 31;
    int64_t base = 0;
    for (int n0 = 0; n0 < a.batch; n0 += 32) {
        const int n = n0 + lane;
        const int64_t mine = n < a.batch ? static_cast<int64_t>(tiles_of(kv_length(a.lengths, n, a.capacity))) * per_seq
                                         : 0;
        int64_t incl = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += o;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, base + incl > x);
        if (over != 0) {
            const int who = __ffs(over) - 1;
            const int64_t b = __shfl_sync(0xffffffffu, base + incl - mine, who);
            const int tiles = static_cast<int>(__shfl_sync(0xffffffffu, mine, who) / per_seq);
            const int64_t rem = x - b;
            return TilePos{n0 + who, static_cast<int>(rem / tiles), static_cast<int>(rem % tiles), b};
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
    return TilePos{a.batch, 0, 0, base};
}

template <bool E4M3, int EP, int NT>
__global__ void __launch_bounds__(kAttnThreads, AttnShape<EP, NT>::kCtas) k_kv_attend(KvAttnArgs a, KvPartials w, int row_tiles) {
    enter_kernel();
    using S = AttnShape<EP, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c4 = lane & 3, r4 = lane >> 2;
    uint8_t* const stages = smem + warp * S::kWarpBytes;
    float* const scales = reinterpret_cast<float*>(smem + 4 * S::kWarpBytes) + warp * S::kStages * 2;
    float2* const joined = reinterpret_cast<float2*>(smem + 4 * S::kWarpBytes + S::kScaleBytes);  // [warp][row]
    const uint32_t stages_s = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
    const uint32_t scales_s = static_cast<uint32_t>(__cvta_generic_to_shared(scales));
    const int per_seq = a.kv_heads * row_tiles;

    // this CTA's stretch of the list
    const int64_t total = find_tile(a, per_seq, INT64_MAX).base;
    const int64_t each = (total + gridDim.x - 1) / gridDim.x;
    int64_t x = each * blockIdx.x;
    const int64_t x_end = min(x + each, total);
    if (x >= x_end) return;
    TilePos pos = find_tile(a, per_seq, x);

    while (x < x_end) {
        const int n = pos.n, h = pos.item / row_tiles, rt = pos.item % row_tiles;
        const int len = kv_length(a.lengths, n, a.capacity), cnt = kv_count(a.counts, n, a.tokens);
        const int tiles = tiles_of(len);
        const int t0 = pos.tile;
        const int nt = static_cast<int>(min(static_cast<int64_t>(tiles - t0), x_end - x));
        const size_t head = static_cast<size_t>(n) * a.kv_heads + h;
        const uint8_t* const kbase = a.key + head * a.capacity * a.head_dim;
        const uint8_t* const vbase = a.value + head * a.capacity * a.head_dim;
        const float* const ks = a.key_scale + head * a.nblocks;
        const float* const vs = a.value_scale + head * a.nblocks;
        float* const scores = w.scores == nullptr ? nullptr
                                                  : w.scores + head * S::kRows * static_cast<size_t>(a.capacity);

        const auto fetch = [&](int it) {
            const int st = it % S::kStages;
            const int tok = (t0 + it) * kTile + warp * kWarpTokens;
            if (it < nt && tok < len) {
                const uint32_t ks_s = stages_s + st * S::kStageBytes, vs_s = ks_s + S::kSliceBytes;
                const size_t off = static_cast<size_t>(tok) * a.head_dim;
                if (a.head_dim == EP && tok + kWarpTokens <= len) {
                    // a whole slice is one piece of memory; a lane's rows are 32 / kChunks apart, which changes known bits
                    // of the permutation
                    constexpr int kStep = 32 / S::kChunks;
                    const int own = swizzled<EP>(lane / S::kChunks, lane % S::kChunks);
                    const uint8_t* const kp = kbase + off + lane * 16;
                    const uint8_t* const vp = vbase + off + lane * 16;
#pragma unroll
                    for (int j = 0; j < S::kChunks; ++j) {
                        const int flip = swizzled<EP>(j * kStep, 0) - j * kStep * EP;
                        const uint32_t to = (own ^ flip) + j * kStep * EP;
                        cp_async16(ks_s + to, kp + j * 512, true);
                        cp_async16(vs_s + to, vp + j * 512, true);
                    }
                } else {
#pragma unroll 1
                    for (int j = 0; j < S::kChunks; ++j) {
                        const int idx = j * 32 + lane, r = idx / S::kChunks, c = idx % S::kChunks;
                        const bool live = tok + r < len && c * 16 < a.head_dim;
                        const size_t o = live ? off + static_cast<size_t>(r) * a.head_dim + c * 16 : off;
                        cp_async16(ks_s + swizzled<EP>(r, c), kbase + o, live);
                        cp_async16(vs_s + swizzled<EP>(r, c), vbase + o, live);
                    }
                }
                if (lane < 2) {
                    const int b = tok >> a.block_shift;
                    cp_async4(scales_s + (st * 2 + lane) * 4, lane == 0 ? ks + b : vs + b);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

#pragma unroll
        for (int it = 0; it < S::kStages - 1; ++it) fetch(it);
        uint32_t q[NT][EP / 8];
        float f[NT][2];
        int lim[NT][2], least = INT_MAX;
        float o[EP / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            load_query<EP>(a, n, h, rt * S::kRows + j * 8, q[j], f[j]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f[j][i] *= a.scale_log2;
                lim[j][i] = kv_limit(a, rt * S::kRows + j * 8 + c4 * 2 + i, len, cnt);
                least = min(least, lim[j][i]);
                m[j][i] = -INFINITY;
                l[j][i] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < EP / 16; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[e][j][i] = 0.0f;
        }

        for (int it = 0; it < nt; ++it) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
            __syncwarp();
            fetch(it + S::kStages - 1);
            const int tok = (t0 + it) * kTile + warp * kWarpTokens;
            if (tok >= len) continue;
            const int st = it % S::kStages;
            const uint8_t* const kst = stages + st * S::kStageBytes;
            const float kscale = scales[st * 2], vscale = scales[st * 2 + 1];

            // scores: accumulator t of 16 tokens has tokens r4 (registers 0, 1) and r4 + 8 (2, 3), rows 2 c4 and 2 c4 + 1
            float s[2][NT][4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int j = 0; j < NT; ++j) s[t][j][0] = s[t][j][1] = s[t][j][2] = s[t][j][3] = 0.0f;
#pragma unroll
                for (int kc = 0; kc < EP / 64; ++kc) {
                    const uint4 lo = *reinterpret_cast<const uint4*>(kst + swizzled<EP>(t * 16 + r4, kc * 4 + c4));
                    const uint4 hi = *reinterpret_cast<const uint4*>(kst + swizzled<EP>(t * 16 + r4 + 8, kc * 4 + c4));
                    const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int step = 0; step < 4; ++step) {
                        uint32_t a0, a1, a2, a3;
                        codes_to_half<E4M3, 0>(wl[step], a0, a2);
                        codes_to_half<E4M3, 0>(wh[step], a1, a3);
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            mma16816(s[t][j], a0, a1, a2, a3, q[j][kc * 8 + step * 2], q[j][kc * 8 + step * 2 + 1]);
                    }
                }
            }
            const bool ragged = __any_sync(0xffffffffu, tok + kWarpTokens > least);
            bool grown = false;
            float alpha[NT][2], base[NT][2], gain[NT][2], vs[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float g = f[j][i] * kscale;
                    float top = kNothing;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float v = s[t][j][k * 2 + i] * g;
                            if (ragged && tok + t * 16 + k * 8 + r4 >= lim[j][i]) v = -INFINITY;
                            s[t][j][k * 2 + i] = v;
                            top = fmaxf(top, v);
                        }
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    // the smaller of the running and the slice's largest, to the larger
                    const bool over = top > m[j][i];
                    const float ratio = ex2(over ? m[j][i] - top : top - m[j][i]);
                    alpha[j][i] = over ? ratio : 1.0f;
                    gain[j][i] = over ? 1.0f : ratio;
                    base[j][i] = top - kShift;
                    // where nothing is seen there are no weights, and no values whatever their scale (NaN of a marked block)
                    vs[j][i] = top == kNothing ? 0.0f : vscale * gain[j][i];
                    grown |= over;
                    m[j][i] = over ? top : m[j][i];
                }
            if (scores != nullptr) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = j * 8 + c4 * 2 + i;
                        if (row >= a.rows) continue;
                        float* const sc = scores + row * static_cast<size_t>(a.capacity) + tok + r4;
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int k = 0; k < 2; ++k) sc[t * 16 + k * 8] = s[t][j][k * 2 + i];
                    }
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    l[j][0] *= alpha[j][0];
                    l[j][1] *= alpha[j][1];
#pragma unroll
                    for (int e = 0; e < EP / 16; ++e)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[e][j][i] *= alpha[j][i & 1];
                }
            }
            // weights: fp16 (11 significant bits, half a bf16 output's rounding at most), as the B operand of 16 tokens
            uint32_t p[2][NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float u[4], v[4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        u[t * 2 + k] = ex2(s[t][j][k * 2] - base[j][0]);
                        v[t * 2 + k] = ex2(s[t][j][k * 2 + 1] - base[j][1]);
                        p[t][j][k] = transpose8(pack_half2(u[t * 2 + k], v[t * 2 + k]));
                    }
                l[j][0] = fmaf((u[0] + u[1]) + (u[2] + u[3]), gain[j][0], l[j][0]);
                l[j][1] = fmaf((v[0] + v[1]) + (v[2] + v[3]), gain[j][1], l[j][1]);
            }
            // values: 8 x 8 pairs of bytes transposed on the way in; even elements are rows 0-7 of the operand, odd 8-15
            const uint32_t vst = stages_s + st * S::kStageBytes + S::kSliceBytes;
#pragma unroll
            for (int e = 0; e < EP / 16; ++e) {
                uint32_t v[4];
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                             : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                             : "r"(vst + swizzled<EP>(lane, e)));
                float acc[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_half<E4M3, 1>(v[2 * t], a0, a1);
                    codes_to_half<E4M3, 1>(v[2 * t + 1], a2, a3);
#pragma unroll
                    for (int j = 0; j < NT; ++j) mma16816(acc[j], a0, a1, a2, a3, p[t][j][0], p[t][j][1]);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[e][j][i] = fmaf(vs[j][i & 1], acc[j][i], o[e][j][i]);
            }
        }

        // join the four warps' states; a warp's stages are free once its copies have landed
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        float* const mine = reinterpret_cast<float*>(stages);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = j * 8 + c4 * 2 + i;
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[j][i] += __shfl_xor_sync(0xffffffffu, l[j][i], d);
                if (r4 == 0) joined[warp * S::kRows + r] = make_float2(m[j][i], l[j][i]);
#pragma unroll
                for (int e = 0; e < EP / 16; ++e)
                    *reinterpret_cast<float2*>(mine + r * S::kJoin + e * 16 + r4 * 2) = make_float2(o[e][j][i], o[e][j][i + 2]);
            }
        __syncthreads();
        const bool whole = nt == tiles;
        // a CTA has at most two open ends: an item that began before its stretch, and one that goes on behind it
        const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + (t0 > 0 ? 0 : 1);
        for (int idx = threadIdx.x; idx < S::kRows * (EP / 4); idx += kAttnThreads) {
            const int r = idx / (EP / 4), e = (idx % (EP / 4)) * 4, row = rt * S::kRows + r;
            if (row >= a.rows) continue;
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) mm = fmaxf(mm, joined[k * S::kRows + r].x);
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 ml = joined[k * S::kRows + r];
                const float g = ml.x == mm ? 1.0f : ex2(ml.x - mm);
                ll += ml.y * g;
                const float4 v = *reinterpret_cast<const float4*>(smem + k * S::kWarpBytes + (r * S::kJoin + e) * 4);
                acc.x = fmaf(v.x, g, acc.x);
                acc.y = fmaf(v.y, g, acc.y);
                acc.z = fmaf(v.z, g, acc.z);
                acc.w = fmaf(v.w, g, acc.w);
            }
            if (whole && ll == 0.0f) ll = row_sum(ll, kv_limit(a, row, len, cnt) > 0);
            if (!whole) {
                reinterpret_cast<float4*>(w.out)[(slot * S::kRows + r) * (EP / 4) + e / 4] = acc;
                if (e == 0) w.stats[slot * S::kRows + r] = make_float2(mm, ll);
                continue;
            }
            const int t = row / a.group, j = row - t * a.group;
            const size_t orow = (head * a.group + j) * a.tokens + t;
            if (e < a.head_dim)
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + orow * a.head_dim + e) =
                    pack_out(acc, ll == 0.0f ? 0.0f : 1.0f / ll, a.query_bf16);
            if (e == 0) {
                const float lse2 = ll == 0.0f ? -INFINITY : mm + log2f(ll) - kShift;
                if (a.lse != nullptr) a.lse[orow] = lse2 * kLn2;
                if (w.lse2 != nullptr) w.lse2[head * a.rows + row] = lse2;
            }
        }
        __syncthreads();  // the stages are written again
        x += nt;
        if (x < x_end) pos = find_tile(a, per_seq, x);
    }
}

// Joins the parts of the items that more than one CTA of k_kv_attend (of `grid` CTAs) worked on: one (item, row) per
// CTA, whose warps take every fourth part; their sums are joined in a fixed order. 55 parts of 64 rows: 12 us (31 with one
// warp a row).
template <int EP>
__global__ void __launch_bounds__(128) k_kv_merge(KvAttnArgs a, KvPartials w, int row_tiles, int tile_rows, int grid) {
    enter_kernel();
    __shared__ float parts_sum[4];
    __shared__ float parts_out[4][EP];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per_seq = a.kv_heads * row_tiles;
    const unsigned item = blockIdx.x / tile_rows;
    const int r = static_cast<int>(blockIdx.x % tile_rows);
    const int n = static_cast<int>(item / per_seq), in_seq = static_cast<int>(item % per_seq);
    const int h = in_seq / row_tiles, row = (in_seq % row_tiles) * tile_rows + r;
    if (n >= a.batch || row >= a.rows) return;
    // list position of the item's first tile
    int64_t total = 0, first = 0;
    for (int n0 = 0; n0 < a.batch; n0 += 32) {
        const int k = n0 + lane;
        int64_t t = k < a.batch ? static_cast<int64_t>(tiles_of(kv_length(a.lengths, k, a.capacity))) * per_seq : 0;
        int64_t before = k < n ? t : 0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            t += __shfl_xor_sync(0xffffffffu, t, d);
            before += __shfl_xor_sync(0xffffffffu, before, d);
        }
        total += t;
        first += before;
    }
    const int tiles = tiles_of(kv_length(a.lengths, n, a.capacity));
    first += static_cast<int64_t>(in_seq) * tiles;
    const int64_t each = (total + grid - 1) / grid;
    const int c0 = static_cast<int>(first / each), parts = static_cast<int>((first + tiles - 1) / each) - c0 + 1;
    if (parts == 1) return;
    // part k is in slot 2 (c0 + k) but for the first, which goes on behind its stretch: 2 c0 + 1
    const float2* const stats = w.stats + static_cast<size_t>(c0) * 2 * tile_rows + r;
    const float* const out = w.out + (static_cast<size_t>(c0) * 2 * tile_rows + r) * EP;
    float mm = -INFINITY;
    for (int k = lane; k < parts; k += 32) mm = fmaxf(mm, stats[static_cast<size_t>(k == 0 ? 1 : 2 * k) * tile_rows].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
    float ll = 0.0f;
    constexpr int kVec = EP / 64;  // float2 of the row a lane has
    float2 acc[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) acc[v] = make_float2(0.0f, 0.0f);
#pragma unroll 8
    for (int k = warp; k < parts; k += 4) {
        const size_t at = static_cast<size_t>(k == 0 ? 1 : 2 * k) * tile_rows;
        const float2 ml = stats[at];
        const float g = ml.x == mm ? 1.0f : ex2(ml.x - mm);
        ll += ml.y * g;
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const float2 u = reinterpret_cast<const float2*>(out + at * EP)[v * 32 + lane];
            acc[v].x = fmaf(u.x, g, acc[v].x);
            acc[v].y = fmaf(u.y, g, acc[v].y);
        }
    }
    if (lane == 0) parts_sum[warp] = ll;
#pragma unroll
    for (int v = 0; v < kVec; ++v) reinterpret_cast<float2*>(parts_out[warp])[v * 32 + lane] = acc[v];
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int k = 1; k < 4; ++k) {
        ll += parts_sum[k];
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const float2 u = reinterpret_cast<const float2*>(parts_out[k])[v * 32 + lane];
            acc[v].x += u.x;
            acc[v].y += u.y;
        }
    }
    if (ll == 0.0f)
        ll = row_sum(ll, kv_limit(a, row, kv_length(a.lengths, n, a.capacity), kv_count(a.counts, n, a.tokens)) > 0);
    const float g = ll == 0.0f ? 0.0f : 1.0f / ll;
    const int t = row / a.group, j = row - t * a.group;
    const size_t head = static_cast<size_t>(n) * a.kv_heads + h;
    const size_t orow = (head * a.group + j) * a.tokens + t;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
        const int e = (v * 32 + lane) * 2;
        if (e >= a.head_dim) continue;
        uint32_t u;
        if (a.query_bf16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(acc[v].x * g, acc[v].y * g);
            u = *reinterpret_cast<const uint32_t*>(&b);
        } else {
            u = pack_half2(acc[v].x * g, acc[v].y * g);
        }
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + orow * a.head_dim + e) = u;
    }
    if (lane == 0) {
        const float lse2 = ll == 0.0f ? -INFINITY : mm + log2f(ll) - kShift;
        if (a.lse != nullptr) a.lse[orow] = lse2 * kLn2;
        if (w.lse2 != nullptr) w.lse2[head * a.rows + row] = lse2;
    }
}

// 2^(score - lse2); 0 for a masked token.
__device__ __forceinline__ float weight_of(float score, float lse2) {
    return score == -INFINITY ? 0.0f : ex2(score - lse2);
}

// Weights from the stored scores: a thread sums four tokens' columns over the (at most 16) rows of a head. 8 rows of 8
// heads and 131071 tokens (38 MB, most of it still in L2): 9 us.
__global__ void __launch_bounds__(256, 8) k_kv_weights(KvAttnArgs a, KvPartials w, int tile_rows) {
    enter_kernel();
    const size_t head = blockIdx.y + static_cast<size_t>(gridDim.y) * blockIdx.z;
    const int n = static_cast<int>(head / a.kv_heads);
    if (n >= a.batch) return;
    const int len = kv_length(a.lengths, n, a.capacity);
    const int64_t t = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 4;
    if (t >= len) return;
    const float* sc = w.scores + head * tile_rows * static_cast<size_t>(a.capacity) + t;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    bool undefined = false;
#pragma unroll 4
    for (int r = 0; r < a.rows; ++r) {
        const float lse2 = w.lse2[head * a.rows + r];
        undefined |= lse2 != lse2;
        const float4 x = *reinterpret_cast<const float4*>(sc + r * static_cast<size_t>(a.capacity));
        v[0] += weight_of(x.x, lse2);
        v[1] += weight_of(x.y, lse2);
        v[2] += weight_of(x.z, lse2);
        v[3] += weight_of(x.w, lse2);
    }
    float* o = a.weights + head * a.capacity + t;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (t + i < len) o[i] = a.accumulate ? o[i] + v[i] : v[i];
    if (!undefined) return;
    // rows without a softmax: all that they see, scores of -infinity too
#pragma unroll 1
    for (int r = 0; r < a.rows; ++r) {
        const float lse2 = w.lse2[head * a.rows + r];
        if (lse2 == lse2) continue;
        const int lim = kv_limit(a, r, len, kv_count(a.counts, n, a.tokens));
#pragma unroll 1
        for (int i = 0; i < 4; ++i)
            if (t + i < lim) o[i] = lse2;
    }
}

// Weights of heads larger than the tensor-core kernels take: the scores are computed again, 128 tokens of a head a CTA,
// 32 a warp, with the keys in registers and the rows streamed past them 8 at a time; every token's sum stays in one
// lane's registers until the end, so there are no atomics and the order of the sum is fixed.
template <bool E4M3, int EP>
__global__ void __launch_bounds__(kAttnThreads) k_kv_column_sums(KvAttnArgs a, const float* __restrict__ lse2s, int key_tiles) {
    enter_kernel();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c4 = lane & 3, r4 = lane >> 2;
    const size_t head = blockIdx.x / key_tiles;
    const int n = static_cast<int>(head / a.kv_heads), h = static_cast<int>(head % a.kv_heads);
    const int len = kv_length(a.lengths, n, a.capacity), cnt = kv_count(a.counts, n, a.tokens);
    const int tok = static_cast<int>(blockIdx.x % key_tiles) * kTile + warp * kWarpTokens;
    if (tok >= len) return;
    const uint8_t* const kbase = a.key + (head * a.capacity + tok) * a.head_dim;
    const float kscale = a.key_scale[head * a.nblocks + (tok >> a.block_shift)];
    // Of tokens r4 + 8 k, of 256 rows at a time and in all: thousands of small weights added to one number would lose bits.
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    uint4 keys[4][EP / 64];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int kc = 0; kc < EP / 64; ++kc) {
            const int r = k * 8 + r4, e = (kc * 4 + c4) * 16;
            keys[k][kc] = tok + r < len && e < a.head_dim
                              ? *reinterpret_cast<const uint4*>(kbase + static_cast<size_t>(r) * a.head_dim + e)
                              : make_uint4(0, 0, 0, 0);
        }
    const int row_tiles = (a.rows + 7) / 8;
    for (int rt = 0; rt < row_tiles; ++rt) {
        if (rt % 32 == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                total[k] += sum[k];
                sum[k] = 0.0f;
            }
        }
        // the last row of a tile sees the most
        const int last = min(rt * 8 + 7, min(a.rows, cnt * a.group) - 1);
        if (last < rt * 8 || kv_limit(a, last, len, cnt) <= tok) continue;
        uint32_t q[EP / 8];
        float f[2], lse2[2];
        int lim[2];
        load_query<EP>(a, n, h, rt * 8, q, f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = rt * 8 + c4 * 2 + i;
            f[i] = f[i] * a.scale_log2 * kscale;
            lim[i] = kv_limit(a, row, len, cnt);
            lse2[i] = row < a.rows ? lse2s[head * a.rows + row] : 0.0f;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kc = 0; kc < EP / 64; ++kc) {
                const uint4 lo = keys[2 * t][kc], hi = keys[2 * t + 1][kc];
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int step = 0; step < 4; ++step) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_half<E4M3, 0>(wl[step], a0, a2);
                    codes_to_half<E4M3, 0>(wh[step], a1, a3);
                    mma16816(s, a0, a1, a2, a3, q[kc * 8 + step * 2], q[kc * 8 + step * 2 + 1]);
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (tok + t * 16 + k * 8 + r4 < lim[i]) sum[t * 2 + k] += ex2(s[k * 2 + i] * f[i] - lse2[i]);
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        sum[k] += total[k];
        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
        const int t = tok + k * 8 + r4;
        if (c4 == 0 && t < len) {
            float* o = a.weights + head * a.capacity + t;
            *o = a.accumulate ? *o + sum[k] : sum[k];
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------------------------------------------
struct KvEvictArgs {
    const uint8_t* src[2];
    const float* src_scale[2];
    uint8_t* dst[2];
    float* dst_scale[2];
    const int32_t* lengths;
    const float* weights;
    int32_t* kept;  // [batch * heads][budget]
    int32_t* dst_lengths;
    float* dst_weights;
    int64_t src_cap, dst_cap;
    int batch, heads, head_dim, block_shift, budget, recent, spans;
};

constexpr int kSelectThreads = 1024;

// Order of the weights as unsigned integers: NaN above everything, -0 equal to 0.
__device__ __forceinline__ uint32_t order_key(float f) {
    if (f != f) return 0xffffffffu;
    const uint32_t b = __float_as_uint(f + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sum over the CTA and the part of it before this thread.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
    }
    __syncthreads();  // earlier readers of warp_sums
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int wsum = warp_sums[lane], winc = wsum;  // 32 warps
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, winc, d);
        if (lane >= d) winc += o;
    }
    *all = __shfl_sync(0xffffffffu, winc, 31);
    return incl - v + __shfl_sync(0xffffffffu, winc - wsum, warp);
}

// Four keys from position i on; positions from `end` on do not count.
__device__ __forceinline__ void four_keys(const float* w, int i, int end, bool vec, uint32_t* key) {
    if (vec && i + 4 <= end) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(w + i));
        key[0] = order_key(v.x), key[1] = order_key(v.y), key[2] = order_key(v.z), key[3] = order_key(v.w);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) key[k] = i + k < end ? order_key(w[i + k]) : 0u;
    }
}

// Positions that stay, ascending: a radix selection of the threshold weight among the tokens before the recent ones
// (digits of 11, 11 and 10 bits, a histogram in shared memory each), then one pass that writes the positions in
// order, of those equal to the threshold the first ones. A head per cluster, whose CTAs have a part of the tokens each
// and read each other's histograms and counts. Bound by its four passes and their barriers: 8 heads of 131072 tokens 37 us
// (238 with one CTA a head), 64 heads of up to 32768 27 us.
__global__ void __launch_bounds__(kSelectThreads) k_kv_select(KvEvictArgs a, bool vec) {
    enter_kernel();
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    __shared__ int hist[2][2048];
    __shared__ int warp_sums[32];
    __shared__ int counts[2];  // of this CTA's tokens: above the threshold, and equal to it
    __shared__ uint32_t sh_digit;
    __shared__ int sh_above;
    // one CTA needs no barrier of the cluster
    const auto cluster_sync = [&] {
        if (ctas > 1) cluster.sync();
        else __syncthreads();
    };
    const int tid = threadIdx.x;
    const size_t head = blockIdx.x / ctas;
    const int n = static_cast<int>(head / a.heads);
    const int len = kv_length(a.lengths, n, a.src_cap);
    const int count = min(len, a.budget);
    const int late = min(len, a.recent);
    const int old = len - late;   // tokens that compete
    int need = count - late;      // places for them
    const float* const w = a.weights + head * a.src_cap;
    int32_t* const kept = a.kept + head * a.budget;
    const int all_threads = ctas * kSelectThreads, me = rank * kSelectThreads + tid;
    if (head % a.heads == 0 && me == 0) a.dst_lengths[n] = count;
    for (int i = count + me; i < a.budget; i += all_threads) kept[i] = -1;
    if (need == old) {
        for (int i = me; i < count; i += all_threads) kept[i] = i;
        return;
    }
    for (int i = me; i < late; i += all_threads) kept[need + i] = old + i;
    if (need == 0) return;

    const int part = ((old + ctas - 1) / ctas + 3) & ~3;
    const int begin = min(rank * part, old), end = min(begin + part, old);
    uint32_t prefix = 0, mask = 0;
    const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
    for (int i = tid; i < 2048; i += kSelectThreads) hist[0][i] = 0;
    if (tid < 2) counts[tid] = 0;
    __syncthreads();
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = shifts[pass], size = 1 << bits[pass];
        int* const mine = hist[pass & 1];
        for (int i0 = begin; i0 < end; i0 += 4 * 4 * kSelectThreads) {
            uint32_t key[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) four_keys(w, i0 + (u * kSelectThreads + tid) * 4, end, vec, key[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (i0 + u * 4 * kSelectThreads >= end) break;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = i0 + (u * kSelectThreads + tid) * 4 + k < end && (key[u][k] & mask) == prefix;
                    const uint32_t digit = (key[u][k] >> shift) & (size - 1);
                    const uint32_t live = __ballot_sync(0xffffffffu, in);
                    if (live == 0) continue;
                    const int leader = __ffs(live) - 1;
                    const uint32_t lead_digit = __shfl_sync(0xffffffffu, digit, leader);  // every lane takes part
                    // a warp whose keys agree (ties, such as tokens never attended to) adds once
                    if (__all_sync(0xffffffffu, !in || digit == lead_digit)) {
                        if ((tid & 31) == leader) atomicAdd(&mine[digit], __popc(live));
                    } else if (in) {
                        atomicAdd(&mine[digit], 1);
                    }
                }
            }
        }
        cluster_sync();
        // the other histogram was last read before this barrier
        for (int i = tid; i < 2048; i += kSelectThreads) hist[(pass + 1) & 1][i] = 0;
        // the digit at which the count from above reaches the places that are left; two bins a thread, from the top
        const int b0 = size - 1 - 2 * tid, b1 = b0 - 1;
        int h0 = 0, h1 = 0;
        for (int c = 0; c < ctas; ++c) {
            const int* const theirs = cluster.map_shared_rank(mine, c);
            h0 += b0 >= 0 ? theirs[b0] : 0;
            h1 += b1 >= 0 ? theirs[b1] : 0;
        }
        int all;
        const int above = block_scan(h0 + h1, warp_sums, &all);
        if (above < need && above + h0 >= need) {
            sh_digit = b0;
            sh_above = above;
        } else if (above + h0 < need && above + h0 + h1 >= need) {
            sh_digit = b1;
            sh_above = above + h0;
        }
        __syncthreads();
        prefix |= sh_digit << shift;
        mask |= static_cast<uint32_t>(size - 1) << shift;
        need -= sh_above;
        __syncthreads();
    }
    // all above the threshold `prefix`, and the first `need` equal to it: what the parts before this one have of each
    {
        int more = 0, ties = 0;
        for (int i0 = begin; i0 < end; i0 += 4 * kSelectThreads) {
            uint32_t key[4];
            const int i = i0 + tid * 4;
            four_keys(w, i, end, vec, key);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                more += i + k < end && key[k] > prefix;
                ties += i + k < end && key[k] == prefix;
            }
        }
        more = __reduce_add_sync(0xffffffffu, more);
        ties = __reduce_add_sync(0xffffffffu, ties);
        if ((tid & 31) == 0) {
            atomicAdd(&counts[0], more);
            atomicAdd(&counts[1], ties);
        }
    }
    cluster_sync();
    int more = 0, ties = 0;
    for (int c = 0; c < rank; ++c) {
        const int* const theirs = cluster.map_shared_rank(counts, c);
        more += theirs[0];
        ties += theirs[1];
    }
    for (int i0 = begin; i0 < end; i0 += 4 * kSelectThreads) {
        uint32_t key[4];
        const int i = i0 + tid * 4;
        four_keys(w, i, end, vec, key);
        int here = 0;  // above the threshold in the low half, equal in the high half: 4096 at most each
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < end) here += (key[k] > prefix ? 1 : 0) + (key[k] == prefix ? 0x10000 : 0);
        int all;
        const int before = block_scan(here, warp_sums, &all);
        int m = more + (before & 0xffff), t = ties + (before >> 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i + k >= end || key[k] < prefix) continue;
            if (key[k] > prefix) {
                kept[m + min(t, need)] = i + k;
                ++m;
            } else {
                if (t < need) kept[m + t] = i + k;
                ++t;
            }
        }
        more += all & 0xffff;
        ties += all >> 16;
    }
    cluster_sync();  // this CTA's counts may be read until here
}

// One block of dst, keys and values, per CTA: the kept tokens' codes come to shared memory with cp.async, all of them in
// flight together; then the largest value of each, the new scale, the codes. Bound by instructions: every code is decoded
// twice and encoded once. 8 sequences cut to 4096 tokens of 8 heads (134 MB): 46 us, 2.9 TB/s; 63 with divisions.
template <bool E4M3>
__global__ void __launch_bounds__(kAppendThreads) k_kv_gather(KvEvictArgs a) {
    enter_kernel();
    extern __shared__ __align__(16) uint8_t codes[];  // keys, then values: block * head_dim each
    const int tid = threadIdx.x;
    const int i = static_cast<int>(blockIdx.x % a.spans);
    const size_t head = blockIdx.x / a.spans;
    const int n = static_cast<int>(head / a.heads);
    const int count = min(kv_length(a.lengths, n, a.src_cap), a.budget);
    const int block = 1 << a.block_shift;
    const int slot = i << a.block_shift;
    const int live = min(block, count - slot);
    const int32_t* const kept = a.kept + head * a.budget + slot;
    __shared__ int from[128];
    __shared__ float from_scale[2][128];
    if (tid < live) from[tid] = kept[tid];
    __syncthreads();
    if (a.dst_weights != nullptr && tid < block)
        a.dst_weights[head * a.dst_cap + slot + tid] = tid < live ? a.weights[head * a.src_cap + from[tid]] : 0.0f;
    if (live <= 0) return;
    const int chunks = a.head_dim >> 4, vectors = a.head_dim >> 3, bytes = block * a.head_dim;
    // idx / vectors for idx < 2^12, vectors <= 32: the rounded reciprocal is off by less than 2^-8 of a row
    const uint32_t row_of = ((1u << 20) + vectors - 1) / vectors;
    for (int idx = tid; idx < live * chunks; idx += kAppendThreads) {
        const int t = idx / chunks, c = idx - t * chunks;
        const size_t at = (head * a.src_cap + from[t]) * a.head_dim + c * 16;
        const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(codes)) + idx * 16;
        cp_async16(to, a.src[0] + at, true);
        cp_async16(to + bytes, a.src[1] + at, true);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (tid < 2 * live) {
        const int kv = tid & 1, t = tid >> 1;
        from_scale[kv][t] = a.src_scale[kv][head * (a.src_cap >> a.block_shift) + (from[t] >> a.block_shift)];
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    __shared__ uint32_t part[2][kAppendThreads / 32];
#pragma unroll 1
    for (int kv = 0; kv < 2; ++kv) {
        const uint2* const src = reinterpret_cast<const uint2*>(codes + kv * bytes);
        uint32_t most = 0;
        for (int idx = tid; idx < live * vectors; idx += kAppendThreads) {
            const uint2 x = src[idx];
            float f[8], m = 0.0f;
            decode4<E4M3>(x.x, f);
            decode4<E4M3>(x.y, f + 4);
#pragma unroll
            for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(f[k]));
            most = max(most, __float_as_uint(m * from_scale[kv][idx * row_of >> 20]) & 0x7fffffffu);  // NaN: the largest pattern
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if ((tid & 31) == 0) part[kv][tid >> 5] = most;
    }
    __syncthreads();
#pragma unroll 1
    for (int kv = 0; kv < 2; ++kv) {
        uint32_t most = 0;
#pragma unroll
        for (int w = 0; w < kAppendThreads / 32; ++w) most = max(most, part[kv][w]);
        const float s = most >= 0x7f800000u ? kNan : scale_of<E4M3>(__uint_as_float(most));
        if (tid == 0) a.dst_scale[kv][head * (a.dst_cap >> a.block_shift) + i] = s;
        const float r = reciprocal(s);
        const uint2* const src = reinterpret_cast<const uint2*>(codes + kv * bytes);
        uint2* const dst = reinterpret_cast<uint2*>(a.dst[kv] + (head * a.dst_cap + slot) * a.head_dim);
        for (int idx = tid; idx < block * vectors; idx += kAppendThreads) {
            uint2 q = make_uint2(0, 0);
            if (idx < live * vectors) {
                const uint2 x = src[idx];
                const float sc = from_scale[kv][idx * row_of >> 20];
                float f[8];
                decode4<E4M3>(x.x, f);
                decode4<E4M3>(x.y, f + 4);
#pragma unroll
                for (int k = 0; k < 8; ++k) f[k] *= sc;
                q = make_uint2(encode4<E4M3>(f, s, r), encode4<E4M3>(f + 4, s, r));
            }
            dst[idx] = q;
        }
    }
}

// dst_weights behind the blocks that k_kv_gather writes.
__global__ void __launch_bounds__(256) k_kv_zero_tail(float* w, int64_t heads, int64_t cap, int64_t from) {
    enter_kernel();
    const int64_t tail = cap - from;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < heads * tail;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x)
        w[i / tail * cap + from + i % tail] = 0.0f;
}

// ---------------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------------
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int log2_of(int64_t v) {
    int s = 0;
    while ((int64_t{1} << s) < v) ++s;
    return s;
}

int check_cache(const dt_kv_cache* c, const char* name) {
    const std::string who = std::string(name) + ": ";
    if (c == nullptr) return set_error(DT_ERR_INVALID, who + "null cache");
    if (c->code != DT_KV_INT8 && c->code != DT_KV_E4M3) return set_error(DT_ERR_INVALID, who + "unknown code type");
    if (c->block != 32 && c->block != 64 && c->block != 128)
        return set_error(DT_ERR_INVALID, who + "block must be 32, 64 or 128 tokens");
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16 != 0)
        return set_error(DT_ERR_INVALID, who + "head_dim must be a multiple of 16 up to 256");
    if (c->batch < 0 || c->kv_heads < 1 || c->capacity < 1 || c->capacity % c->block != 0)
        return set_error(DT_ERR_INVALID, who + "capacity must be a positive multiple of block, heads at least 1");
    if (c->capacity > (int64_t{1} << 30) || c->batch > (int64_t{1} << 20) || c->kv_heads > (int64_t{1} << 16) ||
        c->batch * c->kv_heads > (int64_t{1} << 24))
        return set_error(DT_ERR_INVALID, who + "too many tokens, sequences or heads");
    if (c->batch == 0) return DT_OK;
    if (c->key == nullptr || c->value == nullptr || c->key_scale == nullptr || c->value_scale == nullptr)
        return set_error(DT_ERR_INVALID, who + "null buffer");
    if (!aligned16(c->key) || !aligned16(c->value)) return set_error(DT_ERR_INVALID, who + "codes must be 16-byte aligned");
    return DT_OK;
}

bool rows_vectorised(const void* p, const int64_t* strides) {
    return aligned16(p) && strides[0] % 8 == 0 && strides[1] % 8 == 0 && strides[2] % 8 == 0;
}

int grid_of(int64_t ctas, const char* what, unsigned* grid) {
    if (ctas > INT32_MAX) return set_error(DT_ERR_INVALID, std::string(what) + ": too many blocks");
    *grid = static_cast<unsigned>(ctas);
    return DT_OK;
}

// f(constant) for the number of vectors a thread of a block kernel holds.
template <typename F>
void with_vpt(int64_t block, int64_t head_dim, F f) {
    const int64_t vectors = block * head_dim / 8;
    if (vectors <= kAppendThreads) f(std::integral_constant<int, 1>{});
    else if (vectors <= 2 * kAppendThreads) f(std::integral_constant<int, 2>{});
    else if (vectors <= 4 * kAppendThreads) f(std::integral_constant<int, 4>{});
    else if (vectors <= 8 * kAppendThreads) f(std::integral_constant<int, 8>{});
    else f(std::integral_constant<int, 16>{});
}

// f(constant) for the padded head size of the attention kernels.
template <typename F>
int with_head_dim(int64_t head_dim, F f) {
    if (head_dim <= 64) return f(std::integral_constant<int, 64>{});
    if (head_dim <= 128) return f(std::integral_constant<int, 128>{});
    return f(std::integral_constant<int, 256>{});
}

int64_t padded_head(int64_t e) { return e <= 64 ? 64 : e <= 128 ? 128 : 256; }

// Query rows in a row tile of k_kv_attend.
int64_t tile_rows(int64_t rows) { return rows <= 8 ? 8 : 16; }

// Stored scores against computing them again, where few rows ask for weights: see k_kv_weights.
bool stores_scores(const dt_kv_cache* c, int64_t rows) {
    return rows <= 16 && c->batch * c->kv_heads * tile_rows(rows) * c->capacity * 4 <= (int64_t{1} << 30);
}

// Many rows of a head take the tensor-core kernel, whose time hardly depends on how many they are; that of the few-row
// kernel steps up with every 16, a walk of the cache each. Few-row against tensor-core kernel, in us: 8 sequences of 900 to
// 6001 tokens, 8 heads of 128: 17 rows 43 and 52, 32 rows 46 and 52, 33 rows 54 and 52, 48 rows 56 and 53, 64 rows 68 and 54;
// one of 32768: 32 rows 53 and 69, 48 rows 65 and 70, 64 rows 77 and 70; 16 of 500 to 2000, 4 heads of 64: 32 rows 28 and
// 31, 48 rows 31 and 32, 64 rows 36 and 32. They cross between 33 and 64 rows and are within 11 % of each other from 33 to
// 48; with weights likewise. Above 128 elements a head there is no tensor-core kernel.
bool many_rows(const dt_kv_cache* c, int64_t rows) { return rows > 32 && c->head_dim <= 128; }

struct AttnPlan {
    int64_t rows, row_tiles;
    bool many_rows;
    KvPromptPlan prompt;  // of many rows
    int grid;             // of few
    KvColumnPlan columns;  // weights of many rows, on tensor cores
    bool column_tiles;
    size_t out, stats, lse2, scores, bytes;  // offsets and the total (scores: or the columns' workspace)
};

int attn_plan(const dt_kv_cache* c, int64_t query_heads, int64_t tokens, bool weights, AttnPlan* p) {
    int dev = 0, sms = 0;
    int st = current_device(&dev, &sms);
    if (st != DT_OK) return st;
    const int64_t ep = padded_head(c->head_dim);
    p->rows = query_heads / c->kv_heads * tokens;
    p->row_tiles = (p->rows + tile_rows(p->rows) - 1) / tile_rows(p->rows);
    p->many_rows = many_rows(c, p->rows);
    p->grid = sms * (ep == 64 ? AttnShape<64, 1>::kCtas : ep == 128 ? AttnShape<128, 1>::kCtas : AttnShape<256, 1>::kCtas);
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    p->out = 0;
    if (p->many_rows) {
        p->prompt = kv_prompt_plan(c->batch, p->rows, c->head_dim, sms);
        p->lse2 = p->prompt.bytes;
    } else {
        const size_t parts = static_cast<size_t>(p->grid) * 2 * tile_rows(p->rows);
        p->stats = up(parts * ep * 4);
        p->lse2 = p->stats + up(parts * 8);
    }
    p->scores = p->lse2 + (weights ? up(static_cast<size_t>(c->batch) * c->kv_heads * p->rows * 4) : 0);
    p->bytes = p->scores;
    if (weights && stores_scores(c, p->rows)) {
        p->bytes += static_cast<size_t>(c->batch) * c->kv_heads * tile_rows(p->rows) * c->capacity * 4;
    } else if (weights && c->head_dim <= 128) {
        p->column_tiles = true;
        p->columns = kv_column_plan(c->batch, c->kv_heads, p->rows, c->head_dim, c->capacity, sms);
        p->bytes += p->columns.bytes;
    }
    return DT_OK;
}

template <bool E4M3, int EP, int NT>
int launch_few_rows(const KvAttnArgs& a, const KvPartials& w, const AttnPlan& p, cudaStream_t stream) {
    using S = AttnShape<EP, NT>;
    const int row_tiles = static_cast<int>(p.row_tiles);
    unsigned grid = 0;
    int st = grid_of(static_cast<int64_t>(a.batch) * a.kv_heads * row_tiles * S::kRows, "dt_kv_attention", &grid);
    if (st != DT_OK) return st;
    st = launch_kernel("dt_kv_attention", k_kv_attend<E4M3, EP, NT>, dim3(p.grid), kAttnThreads, S::kSmem, stream, 1, a, w,
                       row_tiles);
    if (st != DT_OK) return st;
    return launch_kernel("dt_kv_attention", k_kv_merge<EP>, dim3(grid), 128, 0, stream, 1, a, w, row_tiles, S::kRows, p.grid);
}

int launch_weights(const KvAttnArgs& a, const KvPartials& w, int tile_rows, cudaStream_t stream) {
    const int64_t heads = static_cast<int64_t>(a.batch) * a.kv_heads;
    const unsigned y = static_cast<unsigned>(std::min<int64_t>(heads, 32768));
    const dim3 g(static_cast<unsigned>((a.capacity + 1023) / 1024), y, static_cast<unsigned>((heads + y - 1) / y));
    return launch_kernel("dt_kv_attention", k_kv_weights, g, 256, 0, stream, 1, a, w, tile_rows);
}

template <bool E4M3, int EP>
int launch_attend(const KvAttnArgs& a, const KvPartials& w, const AttnPlan& p, void* workspace, bool weights,
                  cudaStream_t stream) {
    int st = DT_OK;
    if (p.many_rows) st = kv_prompt_attention(a, E4M3 ? DT_KV_E4M3 : DT_KV_INT8, p.prompt, workspace, w.lse2, stream);
    else if (tile_rows(p.rows) == 8) st = launch_few_rows<E4M3, EP, 1>(a, w, p, stream);
    else st = launch_few_rows<E4M3, EP, 2>(a, w, p, stream);
    if (st != DT_OK || !weights) return st;
    const int64_t heads = static_cast<int64_t>(a.batch) * a.kv_heads;
    if (w.scores != nullptr) return launch_weights(a, w, static_cast<int>(tile_rows(p.rows)), stream);
    if (p.column_tiles)
        return kv_column_sums(a, E4M3 ? DT_KV_E4M3 : DT_KV_INT8, p.columns, static_cast<char*>(workspace) + p.scores, w.lse2,
                              stream);
    const int key_tiles = static_cast<int>((a.capacity + kTile - 1) / kTile);
    unsigned grid = 0;
    st = grid_of(heads * key_tiles, "dt_kv_attention", &grid);
    if (st != DT_OK) return st;
    return launch_kernel("dt_kv_attention", k_kv_column_sums<E4M3, 256>, dim3(grid), kAttnThreads, 0, stream, 1, a, w.lse2,
                         key_tiles);
}

}  // namespace

extern "C" {

int dt_kv_append(const dt_kv_cache* cache, const void* key, const void* value, int64_t tokens,
                 const int64_t* key_strides, const int64_t* value_strides, int dtype, const int32_t* lengths,
                 const int32_t* counts, void* stream) {
    int st = check_cache(cache, "dt_kv_append");
    if (st != DT_OK) return st;
    if (dtype != DT_BFLOAT16 && dtype != DT_FLOAT16)
        return set_error(DT_ERR_INVALID, "dt_kv_append: keys and values must be bf16 or fp16");
    if (tokens < 0 || tokens > (int64_t{1} << 30)) return set_error(DT_ERR_INVALID, "dt_kv_append: bad token count");
    if (cache->batch == 0 || tokens == 0) return DT_OK;
    if (key == nullptr || value == nullptr || key_strides == nullptr || value_strides == nullptr || lengths == nullptr)
        return set_error(DT_ERR_INVALID, "dt_kv_append: null argument");
    KvAppendArgs a{};
    a.codes[0] = static_cast<uint8_t*>(cache->key);
    a.codes[1] = static_cast<uint8_t*>(cache->value);
    a.scales[0] = cache->key_scale;
    a.scales[1] = cache->value_scale;
    a.src[0] = static_cast<const uint16_t*>(key);
    a.src[1] = static_cast<const uint16_t*>(value);
    std::copy_n(key_strides, 3, a.stride[0]);
    std::copy_n(value_strides, 3, a.stride[1]);
    a.vec[0] = rows_vectorised(key, key_strides);
    a.vec[1] = rows_vectorised(value, value_strides);
    a.lengths = lengths;
    a.counts = counts;
    a.capacity = cache->capacity;
    a.heads = static_cast<int>(cache->kv_heads);
    a.head_dim = static_cast<int>(cache->head_dim);
    a.tokens = static_cast<int>(tokens);
    a.block_shift = log2_of(cache->block);
    // blocks that `tokens` tokens can touch, wherever the first falls
    a.spans = static_cast<int>(std::min((tokens + 2 * cache->block - 2) / cache->block, cache->capacity / cache->block));
    a.bf16 = dtype == DT_BFLOAT16;
    unsigned grid = 0;
    st = grid_of(cache->batch * cache->kv_heads * 2 * a.spans, "dt_kv_append", &grid);
    if (st != DT_OK) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    with_vpt(cache->block, cache->head_dim, [&](auto vpt) {
        constexpr int V = decltype(vpt)::value;
        st = launch_kernel("dt_kv_append", cache->code == DT_KV_E4M3 ? k_kv_append<true, V> : k_kv_append<false, V>, dim3(grid),
                           kAppendThreads, 0, s, 1, a);
    });
    return st;
}

int dt_kv_read(const dt_kv_cache* cache, const int32_t* lengths, const int32_t* first, int64_t first_all,
               int64_t count, void* key, void* value, int dtype, void* stream) {
    int st = check_cache(cache, "dt_kv_read");
    if (st != DT_OK) return st;
    if (dtype != DT_FLOAT32 && dtype != DT_BFLOAT16 && dtype != DT_FLOAT16)
        return set_error(DT_ERR_INVALID, "dt_kv_read: unsupported dtype");
    if (count < 0 || count > (int64_t{1} << 31)) return set_error(DT_ERR_INVALID, "dt_kv_read: bad token count");
    if (cache->batch == 0 || count == 0 || (key == nullptr && value == nullptr)) return DT_OK;
    if (lengths == nullptr) return set_error(DT_ERR_INVALID, "dt_kv_read: null lengths");
    if (!aligned16(key) || !aligned16(value)) return set_error(DT_ERR_INVALID, "dt_kv_read: outputs must be 16-byte aligned");
    KvReadArgs a{};
    a.codes[0] = static_cast<const uint8_t*>(cache->key);
    a.codes[1] = static_cast<const uint8_t*>(cache->value);
    a.scales[0] = cache->key_scale;
    a.scales[1] = cache->value_scale;
    a.out[0] = key;
    a.out[1] = value;
    a.lengths = lengths;
    a.first = first;
    a.first_all = first_all;
    a.count = count;
    a.capacity = cache->capacity;
    a.heads = static_cast<int>(cache->kv_heads);
    a.head_dim = static_cast<int>(cache->head_dim);
    a.block_shift = log2_of(cache->block);
    a.dtype = dtype;
    a.all_heads = cache->batch * cache->kv_heads;
    const int64_t rows = 256 / (cache->head_dim / 8) * kReadRows;
    const dim3 grid(static_cast<unsigned>((count + rows - 1) / rows), 2,
                    static_cast<unsigned>(std::min<int64_t>(a.all_heads, 65535)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return launch_kernel("dt_kv_read", cache->code == DT_KV_E4M3 ? k_kv_read<true> : k_kv_read<false>, grid, 256, 0, s, 1, a);
}

static int check_queries(const dt_kv_cache* cache, int64_t query_heads, int64_t tokens, const char* who) {
    int st = check_cache(cache, who);
    if (st != DT_OK) return st;
    if (query_heads < cache->kv_heads || query_heads % cache->kv_heads != 0)
        return set_error(DT_ERR_INVALID, std::string(who) + ": query heads must be a multiple of the key heads");
    if (tokens < 0 || tokens > (int64_t{1} << 30) || query_heads > (int64_t{1} << 20) ||
        query_heads / cache->kv_heads * tokens > (int64_t{1} << 30))
        return set_error(DT_ERR_INVALID, std::string(who) + ": too many queries");
    return DT_OK;
}

int dt_kv_attention_workspace(const dt_kv_cache* cache, int64_t query_heads, int64_t tokens, int with_weights,
                              size_t* bytes) {
    int st = check_queries(cache, query_heads, tokens, "dt_kv_attention_workspace");
    if (st != DT_OK) return st;
    if (bytes == nullptr) return set_error(DT_ERR_INVALID, "dt_kv_attention_workspace: null bytes");
    *bytes = 0;
    if (cache->batch == 0 || tokens == 0) return DT_OK;
    AttnPlan p{};
    st = attn_plan(cache, query_heads, tokens, with_weights != 0, &p);
    if (st == DT_OK) *bytes = p.bytes;
    return st;
}

int dt_kv_attention(const dt_kv_cache* cache, const void* query, int64_t query_heads, int64_t tokens,
                    const int64_t* query_strides, int dtype, const int32_t* lengths, const int32_t* counts,
                    float scale, int flags, void* out, float* lse, float* weights, void* workspace,
                    size_t workspace_bytes, void* stream) {
    int st = check_queries(cache, query_heads, tokens, "dt_kv_attention");
    if (st != DT_OK) return st;
    if (dtype != DT_BFLOAT16 && dtype != DT_FLOAT16)
        return set_error(DT_ERR_INVALID, "dt_kv_attention: queries must be bf16 or fp16");
    if ((flags & ~(DT_KV_CAUSAL | DT_KV_ACCUMULATE)) != 0) return set_error(DT_ERR_INVALID, "dt_kv_attention: unknown flag");
    if (!std::isfinite(scale)) return set_error(DT_ERR_INVALID, "dt_kv_attention: scale must be finite");
    if (cache->batch == 0) return DT_OK;
    if (tokens == 0) {  // no queries: nothing to add to weights, but sums of nothing to write
        if (weights == nullptr || (flags & DT_KV_ACCUMULATE) != 0) return DT_OK;
        if (lengths == nullptr) return set_error(DT_ERR_INVALID, "dt_kv_attention: null argument");
        KvAttnArgs a{};
        a.lengths = lengths;
        a.weights = weights;
        a.batch = static_cast<int>(cache->batch);
        a.kv_heads = static_cast<int>(cache->kv_heads);
        a.capacity = cache->capacity;
        return launch_weights(a, KvPartials{}, 0, static_cast<cudaStream_t>(stream));
    }
    if (query == nullptr || query_strides == nullptr || lengths == nullptr || out == nullptr)
        return set_error(DT_ERR_INVALID, "dt_kv_attention: null argument");
    if ((reinterpret_cast<uintptr_t>(out) & 15) != 0 || !aligned16(workspace))
        return set_error(DT_ERR_INVALID, "dt_kv_attention: out and workspace must be 16-byte aligned");
    AttnPlan p{};
    st = attn_plan(cache, query_heads, tokens, weights != nullptr, &p);
    if (st != DT_OK) return st;
    if (workspace == nullptr || workspace_bytes < p.bytes)
        return set_error(DT_ERR_INVALID, "dt_kv_attention: workspace too small (dt_kv_attention_workspace)");
    KvAttnArgs a{};
    a.key = static_cast<const uint8_t*>(cache->key);
    a.value = static_cast<const uint8_t*>(cache->value);
    a.key_scale = cache->key_scale;
    a.value_scale = cache->value_scale;
    a.query = query;
    a.lengths = lengths;
    a.counts = counts;
    a.out = out;
    a.lse = lse;
    a.weights = weights;
    a.q_stride_n = query_strides[0];
    a.q_stride_h = query_strides[1];
    a.q_stride_t = query_strides[2];
    a.batch = static_cast<int>(cache->batch);
    a.kv_heads = static_cast<int>(cache->kv_heads);
    a.head_dim = static_cast<int>(cache->head_dim);
    a.group = static_cast<int>(query_heads / cache->kv_heads);
    a.tokens = static_cast<int>(tokens);
    a.rows = static_cast<int>(p.rows);
    a.capacity = cache->capacity;
    a.block_shift = log2_of(cache->block);
    a.nblocks = static_cast<int>(cache->capacity >> a.block_shift);
    a.scale_log2 = scale * kLog2e;
    a.causal = (flags & DT_KV_CAUSAL) != 0;
    a.query_bf16 = dtype == DT_BFLOAT16;
    a.accumulate = (flags & DT_KV_ACCUMULATE) != 0;
    a.q_vec = rows_vectorised(query, query_strides);
    char* ws = static_cast<char*>(workspace);
    KvPartials w{};
    w.out = reinterpret_cast<float*>(ws + p.out);
    w.stats = reinterpret_cast<float2*>(ws + p.stats);
    w.lse2 = weights != nullptr ? reinterpret_cast<float*>(ws + p.lse2) : nullptr;
    w.scores = p.bytes > p.scores && !p.column_tiles ? reinterpret_cast<float*>(ws + p.scores) : nullptr;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_head_dim(cache->head_dim, [&](auto ep) {
        constexpr int EP = decltype(ep)::value;
        return cache->code == DT_KV_E4M3 ? launch_attend<true, EP>(a, w, p, workspace, weights != nullptr, s)
                                         : launch_attend<false, EP>(a, w, p, workspace, weights != nullptr, s);
    });
}

int dt_kv_evict_workspace(const dt_kv_cache* src, int64_t budget, size_t* bytes) {
    int st = check_cache(src, "dt_kv_evict_workspace");
    if (st != DT_OK) return st;
    if (bytes == nullptr || budget < 0 || budget > (int64_t{1} << 30))
        return set_error(DT_ERR_INVALID, "dt_kv_evict_workspace: bad argument");
    *bytes = static_cast<size_t>(src->batch) * src->kv_heads * budget * 4;
    return DT_OK;
}

static bool overlap(const void* p, size_t np, const void* q, size_t nq) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return a < b + nq && b < a + np;
}

int dt_kv_evict(const dt_kv_cache* src, const dt_kv_cache* dst, const int32_t* lengths, const float* weights,
                int64_t budget, int64_t recent, int32_t* dst_lengths, float* dst_weights, int32_t* kept,
                void* workspace, size_t workspace_bytes, void* stream) {
    int st = check_cache(src, "dt_kv_evict");
    if (st == DT_OK) st = check_cache(dst, "dt_kv_evict");
    if (st != DT_OK) return st;
    if (src->batch != dst->batch || src->kv_heads != dst->kv_heads || src->head_dim != dst->head_dim ||
        src->block != dst->block || src->code != dst->code)
        return set_error(DT_ERR_INVALID, "dt_kv_evict: the caches differ in batch, heads, head_dim, block or code");
    if (budget < 0 || budget > dst->capacity) return set_error(DT_ERR_INVALID, "dt_kv_evict: budget exceeds dst's capacity");
    if (recent < 0 || recent > budget) return set_error(DT_ERR_INVALID, "dt_kv_evict: recent must be 0..budget");
    if (src->batch == 0) return DT_OK;
    if (lengths == nullptr || weights == nullptr || dst_lengths == nullptr)
        return set_error(DT_ERR_INVALID, "dt_kv_evict: null argument");
    const size_t heads = static_cast<size_t>(src->batch) * src->kv_heads;
    const void* const in[4] = {src->key, src->value, src->key_scale, src->value_scale};
    const void* const to[4] = {dst->key, dst->value, dst->key_scale, dst->value_scale};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const size_t unit_i = i < 2 ? src->head_dim * src->block : 4, unit_j = j < 2 ? dst->head_dim * dst->block : 4;
            if (overlap(in[i], heads * (src->capacity / src->block) * unit_i, to[j],
                        heads * (dst->capacity / dst->block) * unit_j))
                return set_error(DT_ERR_INVALID, "dt_kv_evict: src and dst overlap");
        }
    const size_t n_src = heads * src->capacity * 4, n_dst = heads * dst->capacity * 4, n_len = src->batch * 4;
    if (overlap(lengths, n_len, dst_lengths, n_len) || (dst_weights != nullptr && overlap(weights, n_src, dst_weights, n_dst)))
        return set_error(DT_ERR_INVALID, "dt_kv_evict: lengths or weights overlap their outputs");
    if (kept == nullptr && budget > 0) {
        if (workspace == nullptr || workspace_bytes < heads * budget * 4)
            return set_error(DT_ERR_INVALID, "dt_kv_evict: workspace too small (dt_kv_evict_workspace)");
        kept = static_cast<int32_t*>(workspace);
    }
    KvEvictArgs a{};
    a.src[0] = static_cast<const uint8_t*>(src->key);
    a.src[1] = static_cast<const uint8_t*>(src->value);
    a.src_scale[0] = src->key_scale;
    a.src_scale[1] = src->value_scale;
    a.dst[0] = static_cast<uint8_t*>(dst->key);
    a.dst[1] = static_cast<uint8_t*>(dst->value);
    a.dst_scale[0] = dst->key_scale;
    a.dst_scale[1] = dst->value_scale;
    a.lengths = lengths;
    a.weights = weights;
    a.kept = kept;
    a.dst_lengths = dst_lengths;
    a.dst_weights = dst_weights;
    a.src_cap = src->capacity;
    a.dst_cap = dst->capacity;
    a.batch = static_cast<int>(src->batch);
    a.heads = static_cast<int>(src->kv_heads);
    a.head_dim = static_cast<int>(src->head_dim);
    a.block_shift = log2_of(src->block);
    a.budget = static_cast<int>(budget);
    a.recent = static_cast<int>(recent);
    a.spans = static_cast<int>((budget + src->block - 1) / src->block);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    unsigned grid = 0;
    st = grid_of(static_cast<int64_t>(heads) * a.spans, "dt_kv_evict", &grid);
    if (st != DT_OK) return st;
    // CTAs for a head: one for each 16384 tokens that it can hold, 8 at most (16 keys a thread and pass)
    unsigned ctas = 1;
    while (ctas < 8 && src->capacity > static_cast<int64_t>(ctas) * 16384) ctas *= 2;
    st = launch_kernel("dt_kv_evict", k_kv_select, dim3(static_cast<unsigned>(heads) * ctas), kSelectThreads, 0, s, ctas, a,
                       aligned16(weights));
    if (st != DT_OK) return st;
    if (grid > 0) {
        st = launch_kernel("dt_kv_evict", src->code == DT_KV_E4M3 ? k_kv_gather<true> : k_kv_gather<false>, dim3(grid),
                           kAppendThreads, static_cast<size_t>(2 * src->block * src->head_dim), s, 1, a);
        if (st != DT_OK) return st;
    }
    const int64_t written = static_cast<int64_t>(a.spans) * src->block;
    if (dst_weights != nullptr && written < dst->capacity) {
        const int64_t tail = static_cast<int64_t>(heads) * (dst->capacity - written);
        st = launch_kernel("dt_kv_evict", k_kv_zero_tail, dim3(static_cast<unsigned>(std::min<int64_t>((tail + 255) / 256, 148 * 16))),
                           256, 0, s, 1, dst_weights, static_cast<int64_t>(heads), dst->capacity, written);
    }
    return st;
}

}  // extern "C"
