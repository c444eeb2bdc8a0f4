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
//   warps 0-15       softmax: two warpgroups for each row tile, one for each half of the 128 columns; two threads share
//                    a row. They read their scores from TMEM, agree on the row's reference, and write their weights
//                    back as fp16 over columns that have been read, each half reported by itself.
//   warps 16-19      copy codes to shared memory a tile ahead (cp.async, every thread its own 16 bytes, so no barrier),
//                    turn them into fp16 (exact) and store them as tcgen05 operands (128-byte swizzle), two stages of
//                    keys and two of values.
//   warp 20          issues every product: O += P V (P from TMEM, the halves as they come), then S = Q K^T of the next
//                    tokens, for one row tile and then the other, so that one is in its softmax while the tensor core
//                    works for the other.
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
constexpr int kPromptThreads = 768;
constexpr int kConvertWarp = 16, kIssueWarp = 20;
// A softmax thread holds 64 scores; the block is launched with 80 registers a thread and shares them out anew.
constexpr int kSoftmaxRegs = 96, kConvertRegs = 64, kIssueRegs = 32;
static_assert(512 * kSoftmaxRegs + 128 * kConvertRegs + 128 * kIssueRegs <= kPromptThreads * 80,
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
    static constexpr int kTops = kBars + 256;                  // bfloat16 [parity][row tile][half][row]
    static constexpr int kSmem = kTops + 2 * 2 * 2 * 128 * 2;  // barriers, TMEM address, flag, maxima before it
    static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
    static constexpr int kTmemCols = 512;
};

// kPReady: [row tile][half]
enum Bar { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPReady = 10, kQReady = 14, kBarCount = 15 };

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

#define DT_RW4(a, i) "+r"((a)[i]), "+r"((a)[(i) + 1]), "+r"((a)[(i) + 2]), "+r"((a)[(i) + 3])

// Wait for the loads issued so far; the registers of the last are named, so that nothing uses them before.
__device__ __forceinline__ void tmem_wait_load32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : DT_RW4(r, 0), DT_RW4(r, 4), DT_RW4(r, 8), DT_RW4(r, 12), DT_RW4(r, 16), DT_RW4(r, 20), DT_RW4(r, 24),
                   DT_RW4(r, 28)::"memory");
}

__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Byte offset of 16-byte chunk `c` (8 fp16) of row `r` in an operand of 128-byte panels.
__device__ __forceinline__ uint32_t operand_offset(int r, int c) {
    return (c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// The least bfloat16 that is not below x (its upper 16 bits), and back.
__device__ __forceinline__ uint16_t round_up16(float x) {
    const uint32_t b = __float_as_uint(x);
    return static_cast<uint16_t>(((b >> 31) != 0 || b == 0x7f800000u ? b : b + 0xffffu) >> 16);
}
__device__ __forceinline__ float from16(uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }

// Barrier of two warps.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// Half a query row to fp16 in the operand at `smem` (row `r`), scaled by a power of two that it agrees on with the other
// half (`mine`, `other`: one warp of each half at the barrier `id`); returns its inverse. `sign` carries the sign of the
// softmax scale, so that the score factor is not negative.
template <int EP>
__device__ __forceinline__ float stage_query(const KvAttnArgs& a, const uint16_t* p, uint8_t* smem, int r, int half,
                                             volatile uint16_t* mine, volatile uint16_t* other, int id, float sign) {
    uint32_t x[EP / 4];
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < EP / 16; ++c) {
        const int e = half * (EP / 2) + c * 8;
        const bool live = p != nullptr && e < a.head_dim;
        if (live && a.q_vec) {
            const uint4 u = *reinterpret_cast<const uint4*>(p + e);
            x[c * 4] = u.x, x[c * 4 + 1] = u.y, x[c * 4 + 2] = u.z, x[c * 4 + 3] = u.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[c * 4 + j] = live ? p[e + 2 * j] | (static_cast<uint32_t>(p[e + 2 * j + 1]) << 16) : 0u;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpack16(x[c * 4 + j], a.query_bf16);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
    }
    *mine = round_up16(amax);
    pair_sync(id);
    float mul, inv;
    row_power(fmaxf(from16(*mine), from16(*other)), mul, inv);
    mul *= sign;
#pragma unroll
    for (int c = 0; c < EP / 16; ++c) {
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpack16(x[c * 4 + j], a.query_bf16);
            h[j] = pack_half2(f.x * mul, f.y * mul);
        }
        *reinterpret_cast<uint4*>(smem + operand_offset(r, half * (EP / 16) + c)) = make_uint4(h[0], h[1], h[2], h[3]);
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

// Pairs of fp32 in one 64-bit register: one instruction for two elements.
using Pair = unsigned long long;

__device__ __forceinline__ Pair pair_of(float x, float y) {
    Pair d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}

__device__ __forceinline__ void unpair(Pair p, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p));
}

__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// In the place that the program gives it: an exponential occupies its unit for 8 cycles, in which the warp can issue
// the arithmetic of other columns.
__device__ __forceinline__ void ex2_here(float& x) { asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(x)); }

// 32 scores of a row to weights: 16 fp16 pairs, times the value factor; adds their sum in fp32 (without the value
// factor). Columns 2 i and 2 i + 1 go through three stages, a few columns apart, so that the exponentials of some run
// beside the arithmetic of others. MASKED: columns from `live` on count nothing, whatever the scales there are.
template <bool MASKED>
__device__ __forceinline__ void weigh(const uint32_t* s, float f, float vf, float down, int live, uint32_t* p, Pair* sum) {
    constexpr int kAhead = 2, kBehind = 4;
    const Pair f2 = pair_of(f, f), vf2 = pair_of(vf, vf), down2 = pair_of(-down, -down);
    Pair x[16];
#pragma unroll
    for (int i = -kAhead; i < 16 + kBehind; ++i) {
        const int k = i + kAhead;
        if (k < 16) x[k] = fma2(pair_of(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), f2, down2);
        if (i >= 0 && i < 16) {
            float a, b;
            unpair(x[i], a, b);
            ex2_here(a);
            ex2_here(b);
            x[i] = pair_of(a, b);
        }
        const int d = i - kBehind;
        if (d >= 0) {
            float a, b;
            if (MASKED) {
                unpair(x[d], a, b);
                x[d] = pair_of(2 * d >= live ? 0.0f : a, 2 * d + 1 >= live ? 0.0f : b);
            }
            sum[d & 1] = add2(sum[d & 1], x[d]);
            unpair(mul2(x[d], vf2), a, b);
            if (MASKED) {
                if (2 * d >= live) a = 0.0f;
                if (2 * d + 1 >= live) b = 0.0f;
            }
            p[d] = pack_half2(a, b);
        }
    }
}

template <bool E4M3, int EP>
__global__ void __launch_bounds__(kPromptThreads, 1) k_kv_prompt(KvAttnArgs a, float* lse2_out, int row_tiles) {
    using S = PromptShape<EP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_addr(smem);
    const uint32_t bars = base + S::kBars;
    float* const scales = reinterpret_cast<float*>(smem + S::kScales);
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + S::kBars + kBarCount * 8);
    volatile uint32_t* const dead = tmem_slot + 1;
    volatile float* const vmax_slot = reinterpret_cast<volatile float*>(tmem_slot + 2);  // [24]
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
        mbar_init(bars + kQReady * 8, kConvertWarp);
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kConvertWarp) {
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
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    const int row_groups = row0 + kRowTile < a.rows ? 2 : 1;  // row tiles that hold rows
    constexpr uint32_t kScoreInstr = instr_desc(kTokTile, false), kOutInstr = instr_desc(EP, true);

    if (warp >= kIssueWarp) {
        // ---- products ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == kIssueWarp && tiles > 0) {
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
                        mma_ts(tmem + 256 + g * EP, tmem + g * 128 + (kk >> 1) * 32 + (kk & 1) * 8, v_desc + kk * (2048 >> 4), kOutInstr,
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
            await(kQReady, 0);
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
    } else if (warp >= kConvertWarp) {
        // ---- keys and values to fp16 operands ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
        const int t = tid - kConvertWarp * 32;
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
        // row tile, half of the columns, row, and the barrier and places shared with the row's other thread
        const int g = warp >> 3, half = (warp >> 2) & 1, r = tid & 127, row = row0 + g * kRowTile + r;
        const int pair = 1 + g * 4 + (warp & 3);
        volatile uint16_t* const tops = reinterpret_cast<volatile uint16_t*>(smem + S::kTops) + g * 256 + r;  // + parity * 512
        float factor;
        {
            const uint16_t* qp = nullptr;
            if (row < a.rows) {
                const int t = row / a.group, jj = row - t * a.group;
                qp = static_cast<const uint16_t*>(a.query) + n * a.q_stride_n +
                     static_cast<int64_t>(h * a.group + jj) * a.q_stride_h + t * a.q_stride_t;
            }
            // the places of odd tiles: the first tile's are written before the other thread has read these
            const float inv = stage_query<EP>(a, qp, smem + S::kQuery + g * S::kOperand, r, half, tops + 512 + half * 128,
                                              tops + 512 + (half ^ 1) * 128, pair, a.scale_log2 < 0.0f ? -1.0f : 1.0f);
            factor = inv * fabsf(a.scale_log2) * code_unit<E4M3>();
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + kQReady * 8);
        }
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        // this thread's columns of S; a span's weights lie over its own scores
        const uint32_t s_col = (tmem + g * 128 + half * 64) | lanes, o_col = (tmem + 256 + g * EP + half * (EP / 2)) | lanes;
        const uint32_t s_full = bars + (kSFull + g) * 8, p_ready = bars + (kPReady + g * 2 + half) * 8;
        float vtop = 0.0f;
#pragma unroll
        for (int i = 0; i < kPromptThreads / 32; ++i) vtop = fmaxf(vtop, vmax_slot[i]);
        // 2^-e and 2^e with vtop < 2^e
        int ve = static_cast<int>(__float_as_uint(vtop) >> 23) - 126;
        ve = ve < -100 ? -100 : ve > 126 ? 126 : ve;
        const float v_down = __uint_as_float(static_cast<uint32_t>(127 - ve) << 23) * exp2f(kPromptShift);
        const float v_up = __uint_as_float(static_cast<uint32_t>(127 + ve) << 23) * (code_unit<E4M3>() * exp2f(-kPromptShift));

        const int lim = kv_limit(a, row, len, cnt);
        float ref = -INFINITY, l = 0.0f;
        const int steps = g < row_groups ? tiles : 0;
        for (int j = 0; j < steps; ++j) {
            mbar_wait(s_full, j & 1, dead);
            __syncwarp();
            tc_fence_after();
            const float* const sc = scales + (j % kScaleRing) * 8 + half * 2;
            const int live = lim - j * kTokTile - half * 64;  // of these columns
            const bool ragged = __any_sync(0xffffffffu, live < 64);
            uint32_t s[32];
            float top = -INFINITY;
            // span 0 is loaded again for its weights: 32 scores fewer to hold meanwhile
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                tmem_load32(s_col + c * 32, s);
                tmem_wait_load32(s);
                uint32_t* const x = s;
                if (ragged) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c * 32 + i >= live) x[i] = 0xff800000u;
                }
                float mx[2] = {fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])),
                               fmaxf(__uint_as_float(x[2]), __uint_as_float(x[3]))};
#pragma unroll
                for (int i = 4; i < 32; i += 4) {
                    mx[0] = max3(mx[0], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                    mx[1] = max3(mx[1], __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
                }
                const float m = fmaxf(mx[0], mx[1]);
                if (m != -INFINITY) top = fmaxf(top, m * (factor * sc[c]));  // masked stays masked where the scale is 0
            }
            // the row's largest, of both halves, as bfloat16 rounded up: a reference need not be exact. The next use of
            // these places is two tiles on, behind the other thread's barrier of the next.
            const uint16_t top16 = round_up16(top);
            tops[(j & 1) * 512 + half * 128] = top16;
            pair_sync(pair);
            top = fmaxf(from16(top16), from16(tops[(j & 1) * 512 + (half ^ 1) * 128]));
            const bool grow = top > ref + kGrowth;  // also the first: ref is -infinity
            if (__any_sync(0xffffffffu, grow)) {    // the same for both warps of the pair
                const float now = grow ? top : ref;
                const float alpha = grow ? ex2(ref - now) : 1.0f;
                ref = now;
                l *= alpha;
                if (j > 0) {
#pragma unroll 1
                    for (int c = 0; c < EP / 2; c += 32) {
                        const uint32_t col = o_col + c;
                        uint32_t o[32];
                        tmem_load32(col, o);
                        tmem_wait_load32(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_store32(col, o);
                    }
                    tmem_wait_store();
                    tc_fence_before();
                    pair_sync(pair);  // the first half's weights release a product that adds to all of O
                    tc_fence_after();
                }
            }
            const float down = ref == -INFINITY ? 0.0f : ref;
            Pair sum[2] = {0, 0};
#pragma unroll
            for (int c = 1; c >= 0; --c) {
                uint32_t p[16];
                const float f = factor * sc[c], vf = sc[4 + c] * v_down;
                if (c == 0) {
                    tmem_load32(s_col, s);
                    tmem_wait_load32(s);
                }
                if (ragged) weigh<true>(s, f, vf, down, live - c * 32, p, sum);
                else weigh<false>(s, f, vf, down, 32, p, sum);
                tmem_store16(s_col + c * 32, p);
            }
            tmem_wait_store();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready);
            float sum_a, sum_b;
            unpair(add2(sum[0], sum[1]), sum_a, sum_b);
            l += sum_a + sum_b;
        }
        if (steps > 0) {
            mbar_wait(s_full, tiles & 1, dead);
            __syncwarp();
            tc_fence_after();
        }
        // the row's sum; the operands' memory is free once the last product is done (or holds none)
        volatile float* const sums = reinterpret_cast<volatile float*>(smem + S::kKeys) + g * 256 + r;
        if (steps > 0) {
            sums[half * 128] = l;
            pair_sync(pair);
            l += sums[(half ^ 1) * 128];
        }
        const float inv_l = *dead ? __int_as_float(0x7fc00000) : l == 0.0f ? 0.0f : v_up / l;
        const int t = row < a.rows ? row / a.group : 0, jj = row - t * a.group;
        const size_t orow = (head * a.group + jj) * a.tokens + t;
        uint16_t* const out = static_cast<uint16_t*>(a.out) + orow * a.head_dim;
#pragma unroll 1
        for (int c0 = 0; c0 < EP / 2; c0 += 32) {
            const int c = half * (EP / 2) + c0;  // element of the row
            uint32_t o[32];
            if (steps > 0) {
                tmem_load32(o_col + c0, o);
                tmem_wait_load32(o);
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
        if (row < a.rows && half == 0) {
            const float lse2 = l == 0.0f ? -INFINITY : ref + log2f(l);
            if (a.lse != nullptr) a.lse[orow] = lse2 * kLn2;
            if (lse2_out != nullptr) lse2_out[head * a.rows + row] = lse2;
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kConvertWarp) {
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
