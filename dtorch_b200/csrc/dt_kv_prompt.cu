// Attention of many query rows over the 8-bit key/value cache on the 5th-generation tensor cores.

#include <algorithm>
#include <cstdint>
#include <string>

#include "dt_internal.h"
#include "dt_kv.cuh"
#include "dt_kv_prompt.h"

using namespace dtb;

namespace {

// 256 query rows of a key head (two tiles of 128) against tiles of 128 tokens, one CTA per SM:
//   warps 0-3, 4-7   softmax of row tile 0, 1: a thread owns a row. It reads the row's scores from TMEM and writes its
//                    weights back as fp16 over the same columns, in two halves, each of which it reports.
//   warps 8-11       copy codes to shared memory a tile ahead (cp.async, every thread its own 16 bytes, so no barrier),
//                    turn them into fp16 (exact) and store them as tcgen05 operands (128-byte swizzle), two stages of
//                    keys and two of values.
//   warp 12          issues every product: O += P V (P from TMEM, the first half while the second is still made), then
//                    S = Q K^T of the next tokens, for one row tile and then the other, so that one is in its softmax
//                    while the tensor core works for the other.
// TMEM, 512 columns: S of both row tiles (128 each, P in the first half of each), O of both (EP each). Products run in
// the order of their issue, so a completed S also says that the O += P V before it is done.
//
// A softmax row keeps a reference instead of its exact maximum: it moves (and O is scaled, in TMEM) only when the
// maximum has grown by more than 2^3, so weights stay below 2^3 and the scaling is rare. Block scales: a key scale is
// constant over 32 columns and goes into the row's factor; a value scale, relative to a power of two above all of the
// sequence's, into the weight before it is rounded to fp16 (11 bits; 2^kPromptShift keeps values down to 2^-29 of the
// largest normal).
constexpr int kRowTile = 128;
constexpr int kTokTile = 128;
constexpr int kPromptThreads = 512;
// A softmax row holds 128 scores; the block is launched with 128 registers a thread and shares them out anew.
constexpr int kSoftmaxRegs = 200, kConvertRegs = 72, kIssueRegs = 40;
static_assert(256 * kSoftmaxRegs + 128 * kConvertRegs + 128 * kIssueRegs <= kPromptThreads * 128,
              "a sum above the launch's waits forever");
constexpr float kGrowth = 3.0f;
constexpr float kPromptShift = 12.0f;
constexpr int kScaleRing = 4;
constexpr uint64_t kWaitLimitNs = 10000000000ull;  // waits of one CTA for its own work last microseconds

template <int EP>
struct PromptShape {
    static constexpr int kPanels = EP / 64;                    // 64 fp16 = 128 bytes, a swizzled row
    static constexpr int kPanelBytes = 128 * 128;              // 128 rows
    static constexpr int kOperand = kPanels * kPanelBytes;
    static constexpr int kQuery = 0;                           // two row tiles
    static constexpr int kKeys = 2 * kOperand;                 // two stages
    static constexpr int kValues = 4 * kOperand;               // two stages
    static constexpr int kCodes = 6 * kOperand;                // a tile's codes of keys and of values, on their way
    static constexpr int kCodeBytes = 128 * EP;
    static constexpr int kScales = kCodes + 2 * kCodeBytes;    // [ring][keys, values][4]
    static constexpr int kBars = kScales + kScaleRing * 2 * 4 * 4;
    static constexpr int kSmem = kBars + 256 + 1024;           // barriers, TMEM address, flag, maxima; alignment of the base
    static constexpr int kTmemCols = EP == 64 ? 512 : 512;
};

// kPReady: [row tile][half]
enum Bar { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPReady = 10, kBarCount = 14 };

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Wait for the phase of the given parity. Bounded: when it runs out, `dead` is set, every later wait of the CTA returns
// at once, and the kernel runs to its end and marks its outputs.
__device__ __forceinline__ void mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* dead) {
    uint64_t start = 0;
    for (;;) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done || *dead) return;
        uint64_t now;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (start == 0) start = now;
        if (now - start > kWaitLimitNs) break;
    }
    *dead = 1;
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void async_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle: address and strides in units of 16 bytes; bit 46 marks the
// descriptor's version, 2 in bits 61-63 the swizzle. K-major operands repeat every 8 rows at `stride`; MN-major ones
// every 8 k rows at `stride` and every 64 elements at `leading`.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t leading, uint32_t stride) {
    return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(leading >> 4) << 16) |
           (static_cast<uint64_t>(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// One lane of a converged warp. tcgen05.mma takes its operands from uniform registers: issued behind this in a branch
// that the whole warp takes it needs few instructions; behind `if (thread == 0)` every operand is moved over first (eight
// products 800 cycles, measured, against the 512 that the tensor core takes).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// fp16 operands, fp32 accumulator, M = 128; bit 16: B is MN-major.
__device__ constexpr uint32_t instr_desc(int n, bool b_mn_major) {
    return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}

#define DT_R4(a, i) "=r"((a)[i]), "=r"((a)[(i) + 1]), "=r"((a)[(i) + 2]), "=r"((a)[(i) + 3])
#define DT_W4(a, i) "r"((a)[i]), "r"((a)[(i) + 1]), "r"((a)[(i) + 2]), "r"((a)[(i) + 3])

// 32 columns of the calling warp's 32 lanes.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : DT_R4(r, 0), DT_R4(r, 4), DT_R4(r, 8), DT_R4(r, 12), DT_R4(r, 16), DT_R4(r, 20), DT_R4(r, 24), DT_R4(r, 28)
        : "r"(addr));
}

__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        DT_W4(r, 0), DT_W4(r, 4), DT_W4(r, 8), DT_W4(r, 12), DT_W4(r, 16), DT_W4(r, 20), DT_W4(r, 24), DT_W4(r, 28)
        : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        DT_W4(r, 0), DT_W4(r, 4), DT_W4(r, 8), DT_W4(r, 12)
        : "memory");
}

__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Byte offset of 16-byte chunk `c` (8 fp16) of row `r` in an operand of 128-byte panels.
__device__ __forceinline__ uint32_t operand_offset(int r, int c) {
    return (c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// One query row to fp16 in the operand at `smem` (row `r`), scaled by a power of two; returns its inverse. `sign`
// carries the sign of the softmax scale, so that the score factor is not negative.
template <int EP>
__device__ __forceinline__ float stage_query(const KvAttnArgs& a, const uint16_t* p, uint8_t* smem, int r, float sign) {
    uint32_t x[EP / 2];
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < EP / 8; ++c) {
        const bool live = p != nullptr && c * 8 < a.head_dim;
        if (live && a.q_vec) {
            const uint4 u = *reinterpret_cast<const uint4*>(p + c * 8);
            x[c * 4] = u.x, x[c * 4 + 1] = u.y, x[c * 4 + 2] = u.z, x[c * 4 + 3] = u.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[c * 4 + j] = live ? p[c * 8 + 2 * j] | (static_cast<uint32_t>(p[c * 8 + 2 * j + 1]) << 16) : 0u;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpack16(x[c * 4 + j], a.query_bf16);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
    }
    float mul, inv;
    row_power(amax, mul, inv);
    mul *= sign;
#pragma unroll
    for (int c = 0; c < EP / 8; ++c) {
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpack16(x[c * 4 + j], a.query_bf16);
            h[j] = pack_half2(f.x * mul, f.y * mul);
        }
        *reinterpret_cast<uint4*>(smem + operand_offset(r, c)) = make_uint4(h[0], h[1], h[2], h[3]);
    }
    return inv;
}

// Place of vector `v` (16 codes) of thread `tid` in a tile of 128 tokens. Eight lanes take four neighbouring vectors of
// two rows: their halves, 16 bytes of fp16 each, then fall into eight different 16-byte columns of the swizzled panel.
template <int EP>
__device__ __forceinline__ void tile_place(int v, int tid, int& r, int& c) {
    r = (v / (EP / 64)) * 32 + (tid >> 2);
    c = (v % (EP / 64)) * 4 + (tid & 3);
}

// Codes of a tile of 128 tokens to shared memory: 16 codes a copy, EP / 16 copies a thread, each thread its own.
template <int EP>
__device__ __forceinline__ void fetch_codes(uint32_t smem, const uint8_t* base, int tok, int len, int head_dim, int tid) {
#pragma unroll
    for (int v = 0; v < EP / 16; ++v) {
        int r, c;
        tile_place<EP>(v, tid, r, c);
        const bool live = tok + r < len && c * 16 < head_dim;
        const uint8_t* const p = live ? base + static_cast<size_t>(tok + r) * head_dim + c * 16 : base;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem + (v * 128 + tid) * 16), "l"(p),
                     "r"(live ? 16 : 0)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// The thread's own codes as fp16 operand rows.
template <bool E4M3, int EP>
__device__ __forceinline__ void store_operand(uint8_t* smem, const uint8_t* codes, int tid) {
#pragma unroll
    for (int v = 0; v < EP / 16; ++v) {
        int r, c;
        tile_place<EP>(v, tid, r, c);
        const uint4 w = *reinterpret_cast<const uint4*>(codes + (v * 128 + tid) * 16);
        uint4 lo, hi;
        codes_to_half<E4M3, 0>(w.x, lo.x, lo.y);
        codes_to_half<E4M3, 0>(w.y, lo.z, lo.w);
        codes_to_half<E4M3, 0>(w.z, hi.x, hi.y);
        codes_to_half<E4M3, 0>(w.w, hi.z, hi.w);
        *reinterpret_cast<uint4*>(smem + operand_offset(r, 2 * c)) = lo;
        *reinterpret_cast<uint4*>(smem + operand_offset(r, 2 * c + 1)) = hi;
    }
}

// Pairs of fp32 in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// 32 scores of a row (span `c` of a tile) to weights: their sum in fp32, and times the value factor as 16 fp16 pairs.
// MASKED: columns from `live` on count nothing, whatever the scales there are.
template <bool MASKED>
__device__ __forceinline__ float weights_of(const uint32_t* s, float f, float vf, float down, int live, uint32_t* p) {
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        float2 x = fma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), make_float2(f, f),
                        make_float2(-down, -down));
        x.x = ex2(x.x);
        x.y = ex2(x.y);
        if (MASKED) {
            if (i >= live) x.x = 0.0f;
            if (i + 1 >= live) x.y = 0.0f;
        }
        sum = add2(sum, x);
        float2 v = mul2(x, make_float2(vf, vf));
        if (MASKED) {
            if (i >= live) v.x = 0.0f;
            if (i + 1 >= live) v.y = 0.0f;
        }
        p[i >> 1] = pack_half2(v.x, v.y);
    }
    return sum.x + sum.y;
}

template <bool E4M3, int EP>
__global__ void __launch_bounds__(kPromptThreads, 1) k_kv_prompt(KvAttnArgs a, float* lse2_out, int row_tiles) {
    using S = PromptShape<EP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
    const uint32_t base = smem_addr(smem);
    const uint32_t bars = base + S::kBars;
    float* const scales = reinterpret_cast<float*>(smem + S::kScales);
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + S::kBars + kBarCount * 8);
    volatile uint32_t* const dead = tmem_slot + 1;
    volatile float* const vmax_slot = reinterpret_cast<volatile float*>(tmem_slot + 2);  // [16]
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    // the row tiles that see the most tokens first
    const size_t head = blockIdx.x % (static_cast<unsigned>(a.batch) * a.kv_heads);
    const int rt = row_tiles - 1 - static_cast<int>(blockIdx.x / (static_cast<unsigned>(a.batch) * a.kv_heads));
    const int n = static_cast<int>(head / a.kv_heads), h = static_cast<int>(head % a.kv_heads);
    const int len = kv_length(a.lengths, n, a.capacity), cnt = kv_count(a.counts, n, a.tokens);
    const int row0 = rt * 2 * kRowTile;
    // rows are in the order of the tokens: the last live one sees the most
    const int last = min(min(row0 + 2 * kRowTile, a.rows), cnt * a.group) - 1;
    const int most = last < row0 ? 0 : kv_limit(a, last, len, cnt);
    const int tiles = (most + kTokTile - 1) / kTokTile;
    const float* const ks = a.key_scale + head * a.nblocks;
    const float* const vs = a.value_scale + head * a.nblocks;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars + (kKFull + i) * 8, 128);
            mbar_init(bars + (kKEmpty + i) * 8, 1);
            mbar_init(bars + (kVFull + i) * 8, 128);
            mbar_init(bars + (kVEmpty + i) * 8, 1);
            mbar_init(bars + (kSFull + i) * 8, 1);
            mbar_init(bars + (kPReady + i) * 8, 4);
            mbar_init(bars + (kPReady + 2 + i) * 8, 4);
        }
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(const_cast<uint32_t*>(tmem_slot))),
                     "n"(S::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // a power of two that no value scale of these tokens exceeds
    float vmax = 0.0f;
    const int nb = (most + (1 << a.block_shift) - 1) >> a.block_shift;
    for (int i = tid; i < nb; i += kPromptThreads) vmax = fmaxf(vmax, vs[i]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, d));
    if (lane == 0) vmax_slot[warp] = vmax;
    // the row tiles' queries, a row a thread
    float inv = 0.0f;
    if (warp < 8) {
        const int row = row0 + tid;
        const uint16_t* qp = nullptr;
        if (row < a.rows) {
            const int t = row / a.group, jj = row - t * a.group;
            qp = static_cast<const uint16_t*>(a.query) + n * a.q_stride_n +
                 static_cast<int64_t>(h * a.group + jj) * a.q_stride_h + t * a.q_stride_t;
        }
        inv = stage_query<EP>(a, qp, smem + S::kQuery + (tid >> 7) * S::kOperand, tid & 127,
                              a.scale_log2 < 0.0f ? -1.0f : 1.0f);
        async_proxy_fence();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    const int row_groups = row0 + kRowTile < a.rows ? 2 : 1;  // row tiles that hold rows
    constexpr uint32_t kScoreInstr = instr_desc(kTokTile, false), kOutInstr = instr_desc(EP, true);

    if (warp >= 12) {
        // ---- products ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == 12 && tiles > 0) {
            const auto scores = [&](int g, int j) {
                const uint64_t q_desc = operand_desc(base + S::kQuery + g * S::kOperand, 16, 1024);
                const uint64_t k_desc = operand_desc(base + S::kKeys + (j & 1) * S::kOperand, 16, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < EP / 16; ++k) {
                        const uint32_t off = ((k >> 2) * S::kPanelBytes + (k & 3) * 32) >> 4;
                        mma_ss(tmem + g * 128, q_desc + off, k_desc + off, kScoreInstr, k > 0);
                    }
                    tc_commit(bars + (kSFull + g) * 8);
                    if (g + 1 == row_groups) tc_commit(bars + (kKEmpty + (j & 1)) * 8);
                }
                __syncwarp();
            };
            const auto outputs = [&](int g, int j, int half) {
                const uint64_t v_desc = operand_desc(base + S::kValues + (j & 1) * S::kOperand, S::kPanelBytes, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kTokTile / 32; ++k) {
                        const int kk = half * (kTokTile / 32) + k;
                        mma_ts(tmem + 256 + g * EP, tmem + g * 128 + kk * 8, v_desc + kk * (2048 >> 4), kOutInstr,
                               j > 0 || kk > 0);
                    }
                    if (half == 1 && g + 1 == row_groups) tc_commit(bars + (kVEmpty + (j & 1)) * 8);
                    if (half == 1 && j + 1 == tiles) tc_commit(bars + (kSFull + g) * 8);
                }
                __syncwarp();
            };
            const auto await = [&](int bar, int parity) {
                mbar_wait(bars + bar * 8, parity, dead);
                __syncwarp();
                tc_fence_after();
            };
            await(kKFull, 0);
            for (int g = 0; g < row_groups; ++g) scores(g, 0);
            for (int j = 0; j < tiles; ++j) {
                const bool more = j + 1 < tiles;
                await(kVFull + (j & 1), (j >> 1) & 1);
                if (more) await(kKFull + ((j + 1) & 1), ((j + 1) >> 1) & 1);
                for (int g = 0; g < row_groups; ++g) {
                    await(kPReady + g * 2, j & 1);
                    outputs(g, j, 0);
                    await(kPReady + g * 2 + 1, j & 1);
                    outputs(g, j, 1);
                    if (more) scores(g, j + 1);
                }
            }
        }
    } else if (warp >= 8) {
        // ---- keys and values to fp16 operands ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
        const int t = tid - 256;
        const uint8_t* const kbase = a.key + head * a.capacity * a.head_dim;
        const uint8_t* const vbase = a.value + head * a.capacity * a.head_dim;
        uint8_t* const kcodes = smem + S::kCodes;
        uint8_t* const vcodes = kcodes + S::kCodeBytes;
        if (tiles > 0) {
            fetch_codes<EP>(smem_addr(kcodes), kbase, 0, len, a.head_dim, t);
            fetch_codes<EP>(smem_addr(vcodes), vbase, 0, len, a.head_dim, t);
        }
        for (int j = 0; j < tiles; ++j) {
            const int st = j & 1;
            const uint32_t free_parity = ((j >> 1) & 1) ^ 1;
            // behind the last tile nothing is fetched: every copy is of tokens < len or of no bytes
            const int next = j + 1 < tiles ? (j + 1) * kTokTile : len;
            float sc = 0.0f;
            if (t < 8) {  // the scales of the tile's four spans of 32 tokens; 0 behind the length
                const int tok = j * kTokTile + (t & 3) * 32;
                if (tok < len) sc = (t < 4 ? ks : vs)[tok >> a.block_shift];
            }
            mbar_wait(bars + (kKEmpty + st) * 8, free_parity, dead);
            if (t < 8) scales[(j % kScaleRing) * 8 + t] = sc;
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            store_operand<E4M3, EP>(smem + S::kKeys + st * S::kOperand, kcodes, t);
            async_proxy_fence();
            mbar_arrive(bars + (kKFull + st) * 8);
            fetch_codes<EP>(smem_addr(kcodes), kbase, next, len, a.head_dim, t);
            mbar_wait(bars + (kVEmpty + st) * 8, free_parity, dead);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            store_operand<E4M3, EP>(smem + S::kValues + st * S::kOperand, vcodes, t);
            async_proxy_fence();
            mbar_arrive(bars + (kVFull + st) * 8);
            fetch_codes<EP>(smem_addr(vcodes), vbase, next, len, a.head_dim, t);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        // ---- softmax of a row tile ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int g = warp >> 2;            // row tile of the two
        const int r = tid & 127;            // row of the tile = TMEM lane
        const int row = row0 + g * kRowTile + r;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_col = tmem + g * 128, o_col = tmem + 256 + g * EP;
        const uint32_t s_full = bars + (kSFull + g) * 8, p_ready = bars + (kPReady + g * 2) * 8;

        float vtop = 0.0f;
#pragma unroll
        for (int i = 0; i < kPromptThreads / 32; ++i) vtop = fmaxf(vtop, vmax_slot[i]);
        // 2^-e and 2^e with vtop < 2^e
        int ve = static_cast<int>(__float_as_uint(vtop) >> 23) - 126;
        ve = ve < -100 ? -100 : ve > 126 ? 126 : ve;
        const float v_down = __uint_as_float(static_cast<uint32_t>(127 - ve) << 23) * exp2f(kPromptShift);
        const float v_up = __uint_as_float(static_cast<uint32_t>(127 + ve) << 23) * (code_unit<E4M3>() * exp2f(-kPromptShift));

        const float factor = inv * fabsf(a.scale_log2) * code_unit<E4M3>();
        const int lim = kv_limit(a, row, len, cnt);
        float ref = -INFINITY, l = 0.0f;
        const int steps = g < row_groups ? tiles : 0;
        for (int j = 0; j < steps; ++j) {
            mbar_wait(s_full, j & 1, dead);
            __syncwarp();
            tc_fence_after();
            uint32_t s[128];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_load32(s_col + lanes + c * 32, s + c * 32);
            const float* const sc = scales + (j % kScaleRing) * 8;
            tmem_wait_load();
            const int tok = j * kTokTile;
            const bool ragged = __any_sync(0xffffffffu, tok + kTokTile > lim);
            if (ragged) {
#pragma unroll
                for (int c = 0; c < 128; ++c)
                    if (tok + c >= lim) s[c] = 0xff800000u;
            }
            float mx[8];  // two chains for each span of 32 columns
#pragma unroll
            for (int c = 0; c < 8; ++c) mx[c] = __uint_as_float(s[c * 16]);
#pragma unroll
            for (int i = 1; i < 16; ++i)
#pragma unroll
                for (int c = 0; c < 8; ++c) mx[c] = fmaxf(mx[c], __uint_as_float(s[c * 16 + i]));
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float m = fmaxf(mx[2 * c], mx[2 * c + 1]);
                if (m != -INFINITY) top = fmaxf(top, m * (factor * sc[c]));  // masked stays masked where the scale is 0
            }
            const bool grow = top > ref + kGrowth;  // also the first: ref is -infinity
            if (__any_sync(0xffffffffu, grow)) {
                const float now = grow ? top : ref;
                const float alpha = grow ? ex2(ref - now) : 1.0f;
                ref = now;
                l *= alpha;
                if (j > 0) {
#pragma unroll
                    for (int c = 0; c < EP; c += 32) {
                        uint32_t o[32];
                        tmem_load32(o_col + lanes + c, o);
                        tmem_wait_load();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_store32(o_col + lanes + c, o);
                    }
                }
            }
            const float down = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t p[16];
                const float f = factor * sc[c], vf = sc[4 + c] * v_down;
                if (ragged) l += weights_of<true>(s + c * 32, f, vf, down, lim - tok - c * 32, p);
                else l += weights_of<false>(s + c * 32, f, vf, down, 32, p);
                tmem_store16(s_col + lanes + c * 16, p);
                if (c & 1) {
                    tmem_wait_store();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_ready + (c >> 1) * 8);
                }
            }
        }
        if (steps > 0) {
            mbar_wait(s_full, tiles & 1, dead);
            __syncwarp();
            tc_fence_after();
        }
        const float inv_l = *dead ? __int_as_float(0x7fc00000) : l == 0.0f ? 0.0f : v_up / l;
        const int t = row < a.rows ? row / a.group : 0, jj = row - t * a.group;
        const size_t orow = (head * a.group + jj) * a.tokens + t;
        uint16_t* const out = static_cast<uint16_t*>(a.out) + orow * a.head_dim;
#pragma unroll
        for (int c = 0; c < EP; c += 32) {
            uint32_t o[32];
            if (steps > 0) {
                tmem_load32(o_col + lanes + c, o);
                tmem_wait_load();
            }
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
                uint32_t q[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    // a row that saw nothing: its O may be anything where no tile was computed
                    const float x = steps > 0 && l != 0.0f ? __uint_as_float(o[i + 2 * k]) * inv_l : 0.0f;
                    const float y = steps > 0 && l != 0.0f ? __uint_as_float(o[i + 2 * k + 1]) * inv_l : 0.0f;
                    if (a.query_bf16) {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
                        q[k] = *reinterpret_cast<const uint32_t*>(&b);
                    } else {
                        q[k] = pack_half2(x, y);
                    }
                }
                if (row < a.rows && c + i < a.head_dim)
                    *reinterpret_cast<uint4*>(out + c + i) = make_uint4(q[0], q[1], q[2], q[3]);
            }
        }
        if (row < a.rows) {
            const float lse2 = l == 0.0f ? -INFINITY : ref + log2f(l);
            if (a.lse != nullptr) a.lse[orow] = lse2 * kLn2;
            if (lse2_out != nullptr) lse2_out[head * a.rows + row] = lse2;
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTmemCols) : "memory");
    }
}

template <bool E4M3, int EP>
int launch(const KvAttnArgs& a, float* lse2, cudaStream_t stream) {
    using S = PromptShape<EP>;
    cudaError_t e = cudaFuncSetAttribute(k_kv_prompt<E4M3, EP>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return set_error(DT_ERR_CUDA, std::string("dt_kv_attention: ") + cudaGetErrorString(e));
    const int row_tiles = (a.rows + 2 * kRowTile - 1) / (2 * kRowTile);
    const int64_t ctas = static_cast<int64_t>(row_tiles) * a.batch * a.kv_heads;
    if (ctas > INT32_MAX) return set_error(DT_ERR_INVALID, "dt_kv_attention: too many blocks");
    k_kv_prompt<E4M3, EP><<<static_cast<unsigned>(ctas), kPromptThreads, S::kSmem, stream>>>(a, lse2, row_tiles);
    return check_launch("dt_kv_attention");
}

}  // namespace

namespace dtb {

int kv_prompt_attention(const KvAttnArgs& a, int code, float* lse2, cudaStream_t stream) {
    if (a.head_dim <= 64)
        return code == DT_KV_E4M3 ? launch<true, 64>(a, lse2, stream) : launch<false, 64>(a, lse2, stream);
    return code == DT_KV_E4M3 ? launch<true, 128>(a, lse2, stream) : launch<false, 128>(a, lse2, stream);
}

}  // namespace dtb
