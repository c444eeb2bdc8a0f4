// Attention of many query rows over the 8-bit key/value cache on the 5th-generation tensor cores.

#include <algorithm>
#include <cstdint>
#include <string>

#include "dt_internal.h"
#include "dt_kv.cuh"
#include "dt_kv_prompt.h"

using namespace dtb;

namespace {

// 256 query rows of a key head (two tiles of 128) against tiles of 128 tokens, one CTA per SM. The tiles of all
// (sequence, key head, 256 rows) items stand in one list, of which every CTA takes an equal stretch, whatever the lengths
// and however few the rows: a stretch may end one item and begin the next. An item inside one stretch is finished
// there; the others leave their parts in the workspace, and k_kv_prompt_merge joins them in the order of the list.
//   warps 0-15       softmax: two warpgroups for each row tile, one for each half of the 128 columns; two threads share
//                    a row. They read their scores from TMEM, agree on the row's reference, and write their weights
//                    back as fp16 over columns that have been read.
//   warps 16-19      copy codes to shared memory a tile ahead (cp.async, every thread its own 16 bytes, so no barrier),
//                    turn them into fp16 (exact) and store them as tcgen05 operands (128-byte swizzle), two stages of
//                    keys and two of values.
//   warp 20          issues every product: O += P V (P from TMEM), then S = Q K^T of the next tokens, for one row tile
//                    and then the other, so that one is in its softmax while the tensor core works for the other.
// TMEM, 512 columns: S of both row tiles (128 each, P in the first half of each), O of both (EP each). Products run in
// the order of their issue, so a completed S also says that the O += P V before it is done.
//
// 4096 tokens over 16384, 32 query and 8 key heads of 128, int8: 853 us, 1128 TFLOP/s, in a run of 20 calls, 70 % of a
// library product's burst rate; 985 to 1005 us, 60 %, in calls that go on for seconds, when the clock falls to what the
// power allows. Bound by the chain of each row tile (scores, softmax, weights, products: 4000 cycles, of which the tensor
// core works 1024, twice a step) and by issue slots; exponentials and products alone would take 2048.
//
// Block scales are constant over 32 columns: a key scale goes into the row's factor, a value scale into the weight before
// it is rounded to fp16. What is rounded is therefore 2^x * (value scale), and its reference is the row's largest of
// those: x plus the scale's exponent, of the tokens that the row sees. Times 2^kPromptShift it keeps 11 significant bits
// down to 2^-26 of the row's largest, whatever the sizes of values that the row does not see or gives no weight. The sum
// of the weights goes without the value scale, so it has a reference of its own, each thread's largest x. References
// move only when their maximum has grown by more than 2^3 (for the first, O is then scaled, in TMEM), which is rare.
constexpr int kRowTile = 128;
constexpr int kTokTile = 128;
constexpr int kPromptThreads = 768;
constexpr int kConvertWarp = 16, kIssueWarp = 20;
// A softmax thread holds 64 scores; the block is launched with 80 registers a thread and shares them out anew.
constexpr int kSoftmaxRegs = 96, kConvertRegs = 48, kIssueRegs = 48;
static_assert(512 * kSoftmaxRegs + 128 * kConvertRegs + 128 * kIssueRegs <= kPromptThreads * 80,
              "a sum above the launch's waits forever");
constexpr float kGrowth = 3.0f;
constexpr float kPromptShift = 12.0f;
constexpr int kScaleRing = 4;
// Exponents of value scales that count; scales of 0 and NaN have the least: their tokens do not set the reference.
constexpr int kLeastExponent = -100;
constexpr uint64_t kWaitLimitNs = 10000000000ull;  // waits of one CTA for its own work last microseconds
constexpr uint64_t kDrainLimitNs = 1000000000ull;

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
    static constexpr int kScales = kCodes + 2 * kCodeBytes;    // [ring][keys, values, values' exponents][4]
    static constexpr int kBars = kScales + kScaleRing * 3 * 4 * 4;
    static constexpr int kTops = kBars + 256;                  // a float for each softmax thread: [half][256 rows]
    static constexpr int kSmem = kTops + 2 * 128 * 8;
    static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
    static constexpr int kTmemCols = 512;
};

enum Bar { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPReady = 10, kQReady = 12, kBarCount = 13 };

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

// Wait, also with a limit, for copies or products in flight before the CTA ends, whether a wait has run out or not: they
// must not land in memory that has been given up.
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity) {
    uint64_t start, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
    do {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    } while (now - start < kDrainLimitNs);
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

// Barrier of two warps.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// Half a query row to fp16 in the operand at `smem` (row `r`), scaled by a power of two that it agrees on with the other
// half (`mine`, `other`: one warp of each half at the barrier `id`); returns its inverse. `sign` carries the sign of the
// softmax scale, so that the score factor is not negative.
template <int EP>
__device__ __forceinline__ float stage_query(const KvAttnArgs& a, const uint16_t* p, uint8_t* smem, int r, int half,
                                             volatile float* mine, volatile float* other, int id, float sign) {
    uint32_t x[EP / 4];
    load_row<EP / 16>(a, p, half * (EP / 2), x);
    const float amax = row_max<EP / 4>(a, x);
    *mine = amax;
    pair_sync(id);
    float mul, inv;
    row_power(fmaxf(amax, *other), mul, inv);
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

// A tile of 128 tokens is moved as vectors of 16 codes, EP / 16 a thread. Thread `tid` has column c = tid % 4 and row
// r = tid / 4; its vector v stands (v / panels) * 32 rows and (v % panels) * 4 columns further. So eight lanes take four
// neighbouring vectors of two rows, whose halves, 16 bytes of fp16 each, fall into eight different 16-byte columns of
// the swizzled panel; and every address is one of the thread's plus a constant.

// Codes of a tile to shared memory, each thread its own.
template <int EP>
__device__ __forceinline__ void fetch_codes(uint32_t smem, const uint8_t* base, int tok, int len, int head_dim, int tid) {
    constexpr int kPanels = EP / 64;
    const int r = tid >> 2, c = tid & 3;
    const uint32_t dst = smem + tid * 16;
    if (head_dim == EP && tok + kTokTile <= len) {
        const uint8_t* const p = base + static_cast<size_t>(tok + r) * EP + c * 16;
#pragma unroll
        for (int v = 0; v < EP / 16; ++v)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + v * 2048),
                         "l"(p + (v / kPanels) * 32 * EP + (v % kPanels) * 64)
                         : "memory");
    } else {
#pragma unroll 1
        for (int v = 0; v < EP / 16; ++v) {
            const int row = tok + r + (v / kPanels) * 32, e = (c + (v % kPanels) * 4) * 16;
            const bool live = row < len && e < head_dim;
            const uint8_t* const p = live ? base + static_cast<size_t>(row) * head_dim + e : base;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + v * 2048), "l"(p), "r"(live ? 16 : 0)
                         : "memory");
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// The thread's own codes as fp16 operand rows.
template <bool E4M3, int EP>
__device__ __forceinline__ void store_operand(uint8_t* smem, const uint8_t* codes, int tid) {
    constexpr int kPanels = EP / 64;
    const int r = tid >> 2, c = tid & 3;
    const uint8_t* const src = codes + tid * 16;
    uint8_t* const dst_lo = smem + operand_offset(r, 2 * c);
    uint8_t* const dst_hi = smem + operand_offset(r, 2 * c + 1);
#pragma unroll
    for (int v = 0; v < EP / 16; ++v) {
        const uint4 w = *reinterpret_cast<const uint4*>(src + v * 2048);
        uint4 lo, hi;
        codes_to_half<E4M3, 0>(w.x, lo.x, lo.y);
        codes_to_half<E4M3, 0>(w.y, lo.z, lo.w);
        codes_to_half<E4M3, 0>(w.z, hi.x, hi.y);
        codes_to_half<E4M3, 0>(w.w, hi.z, hi.w);
        constexpr int kRows = 32 * 128;
        const int off = (v / kPanels) * kRows + (v % kPanels) * (128 * 128);
        *reinterpret_cast<uint4*>(dst_lo + off) = lo;
        *reinterpret_cast<uint4*>(dst_hi + off) = hi;
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

__device__ __forceinline__ float min_or_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
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

constexpr int kItemRows = 2 * kRowTile;
constexpr int kItemCost = 2;    // tiles that an item costs besides its own: its queries' staging, its outputs
constexpr int kLeastTiles = 2;  // a stretch is not shorter: each part costs that too, and a join

// Tiles of 128 tokens that the rows of item `rt` of a sequence see; at least one, so that rows that see nothing are
// written too. Rows are in the order of the tokens: the last live one sees the most.
__device__ __forceinline__ int item_tiles(const KvAttnArgs& a, int rt, int len, int cnt) {
    const int last = min(min((rt + 1) * kItemRows, a.rows), cnt * a.group) - 1;
    const int most = last < rt * kItemRows ? 0 : kv_limit(a, last, len, cnt);
    return max(1, (most + kTokTile - 1) / kTokTile);
}

// Where a CTA's stretch of the list begins: an item and a tile of it, and what is left of the item's own cost before it.
// An item stands in the list as kItemCost and then its tiles; a boundary inside its cost leaves all tiles to what comes
// behind.
struct PromptStart {
    int n, h, rt, tile, lead;
};

struct PromptList {
    int64_t total;  // cost of all items
    int64_t each;   // of every stretch but the last
};

// x / y, in 32 bits where both fit: 64-bit division takes over a hundred instructions.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
    if (((x | y) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
    return x / y;
}

// Row tiles (of 128) that see a token of key tile `kt` of a sequence: all from the first of them on, as rows are in the
// order of the tokens. At least one where the tile holds tokens, so that weights nobody gives are written as 0.
__device__ __forceinline__ int key_tile_first_row(const KvAttnArgs& a, int kt, int len, int cnt) {
    if (!a.causal) return 0;
    // query i sees token t where t <= len - cnt + i
    const int64_t i = max(kt * kTokTile - (len - cnt), 0);
    const int64_t row_tiles = (a.rows + kRowTile - 1) / kRowTile;
    return static_cast<int>(min(i * a.group / kRowTile, row_tiles - 1));
}

__device__ __forceinline__ int key_tile_rows(const KvAttnArgs& a, int kt, int len, int cnt) {
    if (kt * kTokTile >= len) return 0;
    return (a.rows + kRowTile - 1) / kRowTile - key_tile_first_row(a, kt, len, cnt);
}

// Lays out a list, in one block: of (sequence, head, 256 rows) items and their key tiles, or (COLUMNS) of (sequence,
// head, 128 keys) items and their row tiles. prefix[n][i]: cost of a head's items before item i of sequence n, and of
// all of them at prefix[n][items]; base[n]: that of the sequences before n. Items behind a sequence's length have no
// entries: the last entry before them, at the count of those within, is that of all.
template <bool COLUMNS>
__global__ void __launch_bounds__(1024) k_kv_prompt_plan(KvAttnArgs a, PromptList* list, PromptStart* starts,
                                                         int64_t* prefix, int64_t* base, int row_tiles, int ctas) {
    enter_kernel();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int n = warp; n < a.batch; n += 32) {
        const int len = kv_length(a.lengths, n, a.capacity), cnt = kv_count(a.counts, n, a.tokens);
        int64_t* const out = prefix + static_cast<int64_t>(n) * (row_tiles + 1);
        int64_t done = 0;
        const int used = COLUMNS ? min((len + kTokTile - 1) / kTokTile, row_tiles) : row_tiles;
        for (int r0 = 0; r0 < used; r0 += 32) {
            const int rt = r0 + lane;
            const int tiles = rt >= used ? 0 : COLUMNS ? key_tile_rows(a, rt, len, cnt) : item_tiles(a, rt, len, cnt);
            const int64_t mine = tiles > 0 ? tiles + kItemCost : 0;
            int64_t incl = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += o;
            }
            if (rt < used) out[rt] = done + incl - mine;
            done += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) out[used] = out[row_tiles] = done;
    }
    __syncthreads();
    if (warp == 0) {
        int64_t done = 0;
        for (int n0 = 0; n0 < a.batch; n0 += 32) {
            const int n = n0 + lane;
            const int64_t mine = n < a.batch ? prefix[static_cast<int64_t>(n) * (row_tiles + 1) + row_tiles] * a.kv_heads : 0;
            int64_t incl = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += o;
            }
            if (n < a.batch) base[n] = done + incl - mine;
            done += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) {
            base[a.batch] = done;
            *list = PromptList{done, max(quotient(done + ctas - 1, ctas), static_cast<int64_t>(kLeastTiles))};
        }
    }
    __syncthreads();
    const PromptList l = *list;
    for (int b = threadIdx.x; b < ctas; b += 1024) {
        int64_t x = l.each * b;
        if (x >= l.total) continue;
        const auto find = [](const int64_t* p, int n, int64_t v) {  // the last i < n with p[i] <= v
            int lo = 0, hi = n;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (p[mid] <= v) lo = mid;
                else hi = mid;
            }
            return lo;
        };
        PromptStart s;
        s.n = find(base, a.batch, x);
        x -= base[s.n];
        const int64_t* const p = prefix + static_cast<int64_t>(s.n) * (row_tiles + 1);
        s.h = static_cast<int>(quotient(x, p[row_tiles]));
        x -= s.h * p[row_tiles];
        const int len = kv_length(a.lengths, s.n, a.capacity);
        s.rt = find(p, COLUMNS ? min((len + kTokTile - 1) / kTokTile, row_tiles) : row_tiles, x);
        const int at = static_cast<int>(x - p[s.rt]);
        s.tile = max(at - kItemCost, 0);
        s.lead = max(kItemCost - at, 0);
        starts[b] = s;
    }
}

struct PromptParts {
    float* out;             // [slot][EP / 4][256][4], unnormalised: neighbouring rows side by side
    float2* stats;          // [slot][256]: reference (log2), sum
    const PromptList* list;
    const PromptStart* starts;
    const int64_t* prefix;
    float* lse2;            // [batch * kv_heads][rows], or null
};

// An item of the list, from one of its tiles on.
struct PromptItem {
    int n, h, rt, tile, tiles;

    __device__ __forceinline__ PromptItem(const PromptParts& w, int row_tiles, const PromptStart& s)
        : n(s.n), h(s.h), rt(s.rt), tile(s.tile) {
        measure(w, row_tiles);
    }
    __device__ __forceinline__ void measure(const PromptParts& w, int row_tiles) {
        const int64_t* const p = w.prefix + static_cast<int64_t>(n) * (row_tiles + 1) + rt;
        tiles = static_cast<int>(p[1] - p[0]) - kItemCost;
    }
    // The next item that has tiles, whole; there is one. Empty items stand only behind a head's others (keys behind a
    // sequence's length), and are passed over at once.
    __device__ __forceinline__ void next(const PromptParts& w, int row_tiles, int kv_heads) {
        tile = 0;
        const int64_t* const p = w.prefix + static_cast<int64_t>(n) * (row_tiles + 1);
        if (++rt == row_tiles || p[rt] == p[row_tiles]) {
            rt = 0;
            if (++h == kv_heads) {
                h = 0;
                do ++n;
                while (w.prefix[static_cast<int64_t>(n) * (row_tiles + 1) + row_tiles] == 0);
            }
        }
        measure(w, row_tiles);
    }
};

template <bool E4M3, int EP>
__global__ void __launch_bounds__(kPromptThreads, 1) k_kv_prompt(KvAttnArgs a, PromptParts w, int row_tiles) {
    enter_kernel();
    using S = PromptShape<EP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_addr(smem);
    const uint32_t bars = base + S::kBars;
    float* const scales = reinterpret_cast<float*>(smem + S::kScales);
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + S::kBars + kBarCount * 8);
    volatile uint32_t* const dead = tmem_slot + 1;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    const PromptList list = *w.list;
    const int64_t x_begin = list.each * blockIdx.x;
    if (x_begin >= list.total) return;
    const PromptStart start = w.starts[blockIdx.x];
    const int count = static_cast<int>(min(list.each, list.total - x_begin)) - start.lead;  // cost, from the first tile on
    if (count <= 0) return;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars + (kKFull + i) * 8, 128);
            mbar_init(bars + (kKEmpty + i) * 8, 1);
            mbar_init(bars + (kVFull + i) * 8, 128);
            mbar_init(bars + (kVEmpty + i) * 8, 1);
            mbar_init(bars + (kSFull + i) * 8, 1);
            mbar_init(bars + (kPReady + i) * 8, 8);
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
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    constexpr uint32_t kScoreInstr = instr_desc(kTokTile, false), kOutInstr = instr_desc(EP, true);

    // Every role walks the same items. Stages and phases go by running counts over all of them.
    if (warp >= kIssueWarp) {
        // ---- products ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == kIssueWarp) {
            const auto await = [&](int bar, uint32_t count) {
                mbar_wait(bars + bar * 8, count & 1, dead);
                __syncwarp();
                tc_fence_after();
            };
            // c: tiles of this CTA before the one in question
            const auto scores = [&](int g, uint32_t c, bool last_group) {
                const uint64_t q_desc = operand_desc(base + S::kQuery + g * S::kOperand, 16, 1024);
                const uint64_t k_desc = operand_desc(base + S::kKeys + (c & 1) * S::kOperand, 16, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < EP / 16; ++k) {
                        const uint32_t off = ((k >> 2) * S::kPanelBytes + (k & 3) * 32) >> 4;
                        mma_ss(tmem + g * 128, q_desc + off, k_desc + off, kScoreInstr, k > 0);
                    }
                    tc_commit(bars + (kSFull + g) * 8);
                    if (last_group) tc_commit(bars + (kKEmpty + (c & 1)) * 8);
                }
                __syncwarp();
            };
            const auto outputs = [&](int g, uint32_t c, bool first_tile, bool last_tile, bool last_group) {
                const uint64_t v_desc = operand_desc(base + S::kValues + (c & 1) * S::kOperand, S::kPanelBytes, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kTokTile / 16; ++k)
                        mma_ts(tmem + 256 + g * EP, tmem + g * 128 + (k >> 1) * 32 + (k & 1) * 8, v_desc + k * (2048 >> 4),
                               kOutInstr, !first_tile || k > 0);
                    if (last_group) tc_commit(bars + (kVEmpty + (c & 1)) * 8);
                    if (last_tile) tc_commit(bars + (kSFull + g) * 8);
                }
                __syncwarp();
            };
            uint32_t c = 0, items = 0, c_group1 = 0;  // tiles, items, and tiles of row tile 1 so far
            PromptItem pos(w, row_tiles, start);
            for (int left = count;;) {
                const int steps = min(pos.tiles - pos.tile, left);
                const int groups = pos.rt * kItemRows + kRowTile < a.rows ? 2 : 1;
                await(kQReady, items);
                await(kKFull + (c & 1), c >> 1);
                scores(0, c, groups == 1);
                if (groups == 2) scores(1, c, true);
                for (int j = 0; j < steps; ++j, ++c) {
                    const bool more = j + 1 < steps;
                    await(kVFull + (c & 1), c >> 1);
                    if (more) await(kKFull + ((c + 1) & 1), (c + 1) >> 1);
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        if (g < groups) {
                            const uint32_t mine = g == 0 ? c : c_group1;
                            await(kPReady + g, mine);
                            outputs(g, c, j == 0, !more, g + 1 == groups);
                            if (more) scores(g, c + 1, g + 1 == groups);
                        }
                    }
                    c_group1 += groups - 1;
                }
                ++items;
                left -= steps + kItemCost;
                if (left <= 0) break;
                pos.next(w, row_tiles, a.kv_heads);
            }
            // the last tile's values are free when every product is done: none is in flight when the tensor memory is given up
            mbar_drain(bars + (kVEmpty + ((c - 1) & 1)) * 8, ((c - 1) >> 1) & 1);
        }
    } else if (warp >= kConvertWarp) {
        // ---- keys and values to fp16 operands ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
        const int t = tid - kConvertWarp * 32;
        uint8_t* const kcodes = smem + S::kCodes;
        uint8_t* const vcodes = kcodes + S::kCodeBytes;
        uint32_t c = 0;
        PromptItem pos(w, row_tiles, start);
        for (int left = count;;) {
            const int steps = min(pos.tiles - pos.tile, left);
            const size_t head = static_cast<size_t>(pos.n) * a.kv_heads + pos.h;
            const int len = kv_length(a.lengths, pos.n, a.capacity);
            const uint8_t* const kbase = a.key + head * a.capacity * a.head_dim;
            const uint8_t* const vbase = a.value + head * a.capacity * a.head_dim;
            const float* const sbase = (t < 4 ? a.key_scale : a.value_scale) + head * a.nblocks;
            fetch_codes<EP>(smem_addr(kcodes), kbase, pos.tile * kTokTile, len, a.head_dim, t);
            fetch_codes<EP>(smem_addr(vcodes), vbase, pos.tile * kTokTile, len, a.head_dim, t);
            for (int j = 0; j < steps; ++j, ++c) {
                const int st = c & 1;
                const uint32_t free_parity = ((c >> 1) & 1) ^ 1;
                const int tok0 = (pos.tile + j) * kTokTile;
                // behind the last tile nothing is fetched: every copy is of tokens < len or of no bytes
                const int next = j + 1 < steps ? tok0 + kTokTile : len;
                float sc = 0.0f;
                if (t < 8) {  // the scales of the tile's four spans of 32 tokens; 0 behind the length
                    const int tok = tok0 + (t & 3) * 32;
                    if (tok < len) sc = sbase[tok >> a.block_shift];
                }
                mbar_wait(bars + (kKEmpty + st) * 8, free_parity, dead);
                if (t < 8) scales[(c % kScaleRing) * 12 + t] = sc;
                if (t >= 4 && t < 8) {  // sc < 2^ex
                    const int bits = (__float_as_uint(sc) >> 23) & 255, ex = bits == 255 ? kLeastExponent : bits - 126;
                    scales[(c % kScaleRing) * 12 + t + 4] = static_cast<float>(max(ex, kLeastExponent));
                }
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
            left -= steps + kItemCost;
            if (left <= 0) break;
            pos.next(w, row_tiles, a.kv_heads);
        }
    } else {
        // ---- softmax of a row tile ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // row tile, half of the columns, row, and the barrier and places shared with the row's other thread
        const int g = warp >> 3, half = (warp >> 2) & 1, r = tid & 127;
        const int pair = 1 + g * 4 + (warp & 3);
        // What the thread hands to the row's other one: |q| and each tile's top. One place serves all: it is written again
        // only behind a completed S, which the issuing warp asked for after every warp of the row tile had reported its
        // queries or weights, and those come after its reads; and by an item's queries behind the last product of O.
        volatile float* const mine = reinterpret_cast<volatile float*>(smem + S::kTops) + half * 256 + g * 128 + r;
        volatile float* const other = reinterpret_cast<volatile float*>(smem + S::kTops) + (half ^ 1) * 256 + g * 128 + r;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        // this thread's columns of S; a span's weights lie over its own scores
        const uint32_t s_col = (tmem + g * 128 + half * 64) | lanes, o_col = (tmem + 256 + g * EP + half * (EP / 2)) | lanes;
        const uint32_t s_full = bars + (kSFull + g) * 8, p_ready = bars + (kPReady + g) * 8;
        uint32_t c = 0, phase = 0, items = 0;  // tiles, completions of S and items so far
        PromptItem pos(w, row_tiles, start);
        for (int left = count; left > 0; left > 0 ? pos.next(w, row_tiles, a.kv_heads) : (void)0) {
            const int item_steps = min(pos.tiles - pos.tile, left);
            const int len = kv_length(a.lengths, pos.n, a.capacity), cnt = kv_count(a.counts, pos.n, a.tokens);
            const size_t head = static_cast<size_t>(pos.n) * a.kv_heads + pos.h;
            const int row = pos.rt * kItemRows + g * kRowTile + r;
            const bool live_group = pos.rt * kItemRows + g * kRowTile < a.rows;
            float factor;
            {
                const uint16_t* qp = nullptr;
                const int t = row / a.group, jj = row - t * a.group;
                if (row < a.rows)
                    qp = static_cast<const uint16_t*>(a.query) + pos.n * a.q_stride_n +
                         static_cast<int64_t>(pos.h * a.group + jj) * a.q_stride_h + t * a.q_stride_t;
                const float inv = stage_query<EP>(a, qp, smem + S::kQuery + g * S::kOperand, r, half, mine, other, pair,
                                                  a.scale_log2 < 0.0f ? -1.0f : 1.0f);
                factor = inv * fabsf(a.scale_log2);
                tc_fence_before();  // the reads of O of the item before
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(bars + kQReady * 8);
            }
            int live = kv_limit(a, row, len, cnt) - pos.tile * kTokTile - half * 64;  // of this thread's columns

            // largest x of this thread's columns, and of the row's x + exponent of the value scale, as references
            float ref = -INFINITY, out_ref = -INFINITY, l = 0.0f;
            const int steps = live_group ? item_steps : 0;
            for (int j = 0; j < steps; ++j) {
                mbar_wait(s_full, phase & 1, dead);
                ++phase;
                __syncwarp();
                tc_fence_after();
                const float* const sc = scales + ((c + j) % kScaleRing) * 12 + half * 2;
                const bool ragged = __any_sync(0xffffffffu, live < 64);
                uint32_t s[32], s0[32];
                float top = kNothing, out_top = kNothing;
                // span 0 is loaded again for its weights: 32 scores fewer to hold meanwhile
                tmem_load32(s_col, s0);
                tmem_load32(s_col + 32, s);
                tmem_wait_load32(s0);
                tmem_wait_load32(s);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t* const v = k == 0 ? s0 : s;
                    if (ragged) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (k * 32 + i >= live) v[i] = 0xff800000u;
                    }
                    float mx[2] = {fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1])),
                                   fmaxf(__uint_as_float(v[2]), __uint_as_float(v[3]))};
#pragma unroll
                    for (int i = 4; i < 32; i += 4) {
                        mx[0] = max3(mx[0], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                        mx[1] = max3(mx[1], __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
                    }
                    const float m = fmaxf(mx[0], mx[1]);
                    const float x = m * (factor * sc[k]);  // NaN (a masked span where the scale is 0) is passed over
                    top = fmaxf(top, x);
                    out_top = fmaxf(out_top, x + sc[8 + k]);
                }
                // the row's largest, of both halves, in fp32: large scores leave a 16-bit float's step no room above it
                *mine = out_top;
                pair_sync(pair);
                out_top = fmaxf(out_top, *other);
                const bool grow = top > ref + kGrowth, out_grow = out_top > out_ref + kGrowth;  // the first too
                if (__any_sync(0xffffffffu, grow || out_grow)) {
                    if (grow) {
                        l *= ex2(ref - top);
                        ref = top;
                    }
                    const float now = out_grow ? out_top : out_ref;
                    const float alpha = out_grow ? ex2(out_ref - now) : 1.0f;
                    out_ref = now;
                    if (j > 0 && __any_sync(0xffffffffu, out_grow)) {
#pragma unroll 1
                        for (int k = 0; k < EP / 2; k += 32) {
                            uint32_t o[32];
                            tmem_load32(o_col + k, o);
                            tmem_wait_load32(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_store32(o_col + k, o);
                        }
                    }
                }
                // ref - out_ref is below 2^7: out_ref counts ref's own token with an exponent of at least kLeastExponent
                const float v_down = ex2(ref - out_ref + kPromptShift);
                Pair sum[2] = {0, 0};
#pragma unroll
                for (int k = 1; k >= 0; --k) {
                    uint32_t p[16];
                    // above 2^126 only where all weights are below 2^-111; a NaN scale stays
                    const float f = factor * sc[k], vf = min_or_nan(sc[4 + k] * v_down, 0x1p126f);
                    if (k == 0) {
                        tmem_load32(s_col, s);
                        tmem_wait_load32(s);
                    }
                    if (ragged) weigh<true>(s, f, vf, ref, live - k * 32, p, sum);
                    else weigh<false>(s, f, vf, ref, 32, p, sum);
                    tmem_store16(s_col + k * 32, p);
                }
                tmem_wait_store();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready);
                float sum_a, sum_b;
                unpair(add2(sum[0], sum[1]), sum_a, sum_b);
                l += sum_a + sum_b;
                live -= kTokTile;
            }
            c += item_steps;
            left -= item_steps + kItemCost;
            ++items;
            if (steps == 0) {  // no rows here: keep pace with the other row tile, whose warps report their queries too
                mbar_wait(bars + kQReady * 8, (items - 1) & 1, dead);
                __syncwarp();
                continue;
            }
            mbar_wait(s_full, phase & 1, dead);
            ++phase;
            __syncwarp();
            tc_fence_after();
            // The sums of both threads, through the memory of the row's queries, which are done with.
            uint8_t* const rows = smem + S::kQuery + g * S::kOperand;
            *reinterpret_cast<float2*>(rows + operand_offset(r, half)) = make_float2(ref, l);
            pair_sync(pair);
            {
                const float2 o = *reinterpret_cast<const float2*>(rows + operand_offset(r, half ^ 1));
                const float most = fmaxf(ref, o.x);
                l = l * (ref == most ? 1.0f : ex2(ref - most)) + o.y * (o.x == most ? 1.0f : ex2(o.x - most));
                ref = most;
            }
            pair_sync(pair);  // both have read them: outputs, or the next queries, take their places
            // only an item's end divides by its sum; `live` is the limit less the columns of these tiles and those before
            if (item_steps == pos.tiles) l = row_sum(l, live + (pos.tile + item_steps) * kTokTile + half * 64 > 0);
            if (*dead) l = __int_as_float(0x7fc00000);
            const float v_up = exp2f(out_ref - ref - kPromptShift);
            if (item_steps < pos.tiles) {
                // an item that other CTAs work on too: one that began before this stretch, or goes on behind it
                const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + (pos.tile > 0 ? 0 : 1);
                const size_t at = slot * kItemRows + g * kRowTile + r;
                float4* const out = reinterpret_cast<float4*>(w.out) + slot * (EP / 4) * kItemRows +
                                    half * (EP / 8) * kItemRows + g * kRowTile + r;
#pragma unroll 1
                for (int k = 0; k < EP / 2; k += 32) {
                    uint32_t o[32];
                    tmem_load32(o_col + k, o);
                    tmem_wait_load32(o);
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        out[(k + i) / 4 * kItemRows] =
                            make_float4(__uint_as_float(o[i]) * v_up, __uint_as_float(o[i + 1]) * v_up,
                                        __uint_as_float(o[i + 2]) * v_up, __uint_as_float(o[i + 3]) * v_up);
                }
                if (half == 0) w.stats[at] = make_float2(ref, l);
                continue;
            }
            const float inv_l = v_up / l;
            // the rows go through the memory of their queries, which are done with, so that stores are of whole rows
#pragma unroll 1
            for (int k0 = 0; k0 < EP / 2; k0 += 32) {
                uint32_t o[32];
                tmem_load32(o_col + k0, o);
                tmem_wait_load32(o);
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    uint32_t q[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float u = l == 0.0f ? 0.0f : __uint_as_float(o[i + 2 * e]) * inv_l;
                        const float v = l == 0.0f ? 0.0f : __uint_as_float(o[i + 2 * e + 1]) * inv_l;
                        if (a.query_bf16) {
                            const __nv_bfloat162 b = __floats2bfloat162_rn(u, v);
                            q[e] = *reinterpret_cast<const uint32_t*>(&b);
                        } else {
                            q[e] = pack_half2(u, v);
                        }
                    }
                    *reinterpret_cast<uint4*>(rows + operand_offset(r, (half * (EP / 2) + k0 + i) / 8)) =
                        make_uint4(q[0], q[1], q[2], q[3]);
                }
            }
            pair_sync(pair);
            // this pair's 32 rows: its two warps take 16 each, a row of EP / 8 lanes at a time
            {
                const int first = (warp & 3) * 32 + half * 16;
#pragma unroll 1
                for (int i = lane; i < 16 * (EP / 8); i += 32) {
                    const int rr = first + i / (EP / 8), c8 = i % (EP / 8);
                    const int orow_in = pos.rt * kItemRows + g * kRowTile + rr;
                    if (orow_in >= a.rows || c8 * 8 >= a.head_dim) continue;
                    const int t = orow_in / a.group, jj = orow_in - t * a.group;
                    const size_t at = ((head * a.group + jj) * a.tokens + t) * a.head_dim + c8 * 8;
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) =
                        *reinterpret_cast<const uint4*>(rows + operand_offset(rr, c8));
                }
            }
            pair_sync(pair);  // the next queries take the place of these rows
            int at_end = row;
            asm volatile("" : "+r"(at_end));  // worked out again: not held through the loop
            const int t = at_end / a.group, jj = at_end - t * a.group;
            const size_t orow = (head * a.group + jj) * a.tokens + t;
            if (row < a.rows && half == 0) {
                const float lse2 = l == 0.0f ? -INFINITY : ref + log2f(l);
                if (a.lse != nullptr) a.lse[orow] = lse2 * kLn2;
                if (w.lse2 != nullptr) w.lse2[head * a.rows + row] = lse2;
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kConvertWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTmemCols) : "memory");
    }
}

constexpr int kMergeRows = 64;

// Joins the parts of the items that more than one CTA of k_kv_prompt worked on: a block for each boundary between two
// stretches and 64 of an item's 256 rows, four threads a row. The item's first boundary does the work.
template <int EP>
__global__ void __launch_bounds__(256) k_kv_prompt_merge(KvAttnArgs a, PromptParts w, int row_tiles) {
    enter_kernel();
    const PromptList list = *w.list;
    if (list.each * (blockIdx.x + 1) >= list.total) return;
    const PromptItem pos(w, row_tiles, w.starts[blockIdx.x + 1]);
    // an item that begins here, or before the stretch that ends here, is not this block's
    if (pos.tile == 0 || pos.tile > list.each) return;
    const int c0 = blockIdx.x, parts = 2 + (pos.tiles - pos.tile - 1) / static_cast<int>(list.each);
    constexpr int kVec = EP / 16;  // float4 of the row a thread has
    const int quarter = threadIdx.x >> 6, r = blockIdx.y * kMergeRows + (threadIdx.x & 63), row = pos.rt * kItemRows + r;
    if (row >= a.rows) return;
    const size_t head = static_cast<size_t>(pos.n) * a.kv_heads + pos.h;
    // part k is in slot 2 (c0 + k) but for the first, which goes on behind its stretch: 2 c0 + 1
    const float2* const stats = w.stats + static_cast<size_t>(c0) * 2 * kItemRows + r;
    const float4* const out = reinterpret_cast<const float4*>(w.out) +
                              (static_cast<size_t>(c0) * 2 * (EP / 4) + quarter * kVec) * kItemRows + r;
    float m = -INFINITY;
    for (int k = 0; k < parts; ++k) m = fmaxf(m, stats[(k == 0 ? 1 : 2 * k) * kItemRows].x);
    float l = 0.0f;
    float4 acc[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) acc[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < parts; ++k) {
        const int64_t slot = k == 0 ? 1 : 2 * k;
        const float2 st = stats[slot * kItemRows];
        const float f = st.x == m ? 1.0f : ex2(st.x - m);
        l += st.y * f;
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const float4 o = out[(slot * (EP / 4) + v) * kItemRows];
            acc[v].x = fmaf(o.x, f, acc[v].x);
            acc[v].y = fmaf(o.y, f, acc[v].y);
            acc[v].z = fmaf(o.z, f, acc[v].z);
            acc[v].w = fmaf(o.w, f, acc[v].w);
        }
    }
    l = row_sum(l, kv_limit(a, row, kv_length(a.lengths, pos.n, a.capacity), kv_count(a.counts, pos.n, a.tokens)) > 0);
    const float g = l == 0.0f ? 0.0f : 1.0f / l;
    const int t = row / a.group, jj = row - t * a.group;
    const size_t orow = (head * a.group + jj) * a.tokens + t;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
        const int e = (quarter * kVec + v) * 4;
        if (e >= a.head_dim) continue;
        uint2 u;
        if (a.query_bf16) {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(acc[v].x * g, acc[v].y * g);
            const __nv_bfloat162 hi = __floats2bfloat162_rn(acc[v].z * g, acc[v].w * g);
            u = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        } else {
            u = make_uint2(pack_half2(acc[v].x * g, acc[v].y * g), pack_half2(acc[v].z * g, acc[v].w * g));
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + orow * a.head_dim + e) = u;
    }
    if (quarter == 0) {
        const float lse2 = l == 0.0f ? -INFINITY : m + log2f(l);
        if (a.lse != nullptr) a.lse[orow] = lse2 * kLn2;
        if (w.lse2 != nullptr) w.lse2[head * a.rows + row] = lse2;
    }
}

template <bool E4M3, int EP>
int launch(const KvAttnArgs& a, const KvPromptPlan& p, char* ws, float* lse2, cudaStream_t stream) {
    using S = PromptShape<EP>;
    const int row_tiles = (a.rows + kItemRows - 1) / kItemRows;
    int64_t* const prefix = reinterpret_cast<int64_t*>(ws + p.prefix);
    PromptList* const list = reinterpret_cast<PromptList*>(ws + p.list);
    PromptStart* const starts = reinterpret_cast<PromptStart*>(ws + p.starts);
    const PromptParts w{reinterpret_cast<float*>(ws + p.out), reinterpret_cast<float2*>(ws + p.stats), list, starts, prefix,
                        lse2};
    int st = launch_kernel("dt_kv_attention", k_kv_prompt_plan<false>, dim3(1), 1024, 0, stream, 1, a, list, starts, prefix,
                           prefix + static_cast<int64_t>(a.batch) * (row_tiles + 1), row_tiles, p.ctas);
    if (st != DT_OK) return st;
    st = launch_kernel("dt_kv_attention", k_kv_prompt<E4M3, EP>, dim3(p.ctas), kPromptThreads, S::kSmem, stream, 1, a, w, row_tiles);
    if (st != DT_OK || p.ctas < 2) return st;
    return launch_kernel("dt_kv_attention", k_kv_prompt_merge<EP>, dim3(p.ctas - 1, kItemRows / kMergeRows), 256, 0, stream, 1,
                         a, w, row_tiles);
}

// ---------------------------------------------------------------------------------------------------------------
// Weights of each token, summed over many query rows
// ---------------------------------------------------------------------------------------------------------------
// S^T = K Q^T, 128 keys against tiles of 128 query rows: a thread owns a key and adds up 2^(score - log2 sum of the row)
// over the rows, so there are no atomics and the order of the sum is fixed. An item is (sequence, head, 128 keys); the
// row tiles of all items stand in one list, as above, and items that are split leave 128 sums a part.
// Warps 0-3 and 4-7 take turns at the row tiles; they also turn an item's keys into the operand. Warp 8 issues the
// products into four buffers of 128 TMEM columns, warp 9 copies row blocks (k_kv_row_blocks, laid out as operands) with
// one bulk copy each. Bound by the exponentials: 1024 cycles a tile against 512 of the tensor core. 2 x 2001 tokens, 16
// and 4 heads: 43 us, of which 20 are the tiles; mma.sync without the tensor memory took 900.
template <int EP>
struct ColumnShape {
    static constexpr int kOperand = 128 * EP * 2;
    // what a row tile needs: the operand, then (factor, log2 sum) and the limit of each row
    static constexpr int kBlock = kOperand + 128 * 8 + 128 * 4;
    static constexpr int kStages = 3;
    static constexpr int kBlockRoom = (kBlock + 1023) / 1024 * 1024;
    static constexpr int kKeys = 0;
    static constexpr int kBlocks = kOperand;
    static constexpr int kBars = kBlocks + kStages * kBlockRoom;
    static constexpr int kSums = kBars + 256;
    static constexpr int kSmem = kSums + 128 * 4;
};
constexpr int kColumnThreads = 320;
enum ColumnBar { kBFull = 0, kBEmpty = 3, kTFull = 6, kTEmpty = 10, kKReady = 14, kColumnBars = 15 };

// The query rows of 128-row tiles as operand blocks in the workspace, with each row's score factor, log2 sum (+infinity
// for rows that give no weight: 2^-infinity is 0) and limit.
template <bool E4M3, int EP>
__global__ void __launch_bounds__(128) k_kv_row_blocks(KvAttnArgs a, const float* __restrict__ lse2, uint8_t* blocks) {
    enter_kernel();
    const int tiles = (a.rows + kRowTile - 1) / kRowTile;
    const size_t head = blockIdx.x / tiles;
    const int n = static_cast<int>(head / a.kv_heads), h = static_cast<int>(head % a.kv_heads);
    const int r = threadIdx.x, row = static_cast<int>(blockIdx.x % tiles) * kRowTile + r;
    uint8_t* const out = blocks + static_cast<size_t>(blockIdx.x) * ColumnShape<EP>::kBlock;
    const int len = kv_length(a.lengths, n, a.capacity), cnt = kv_count(a.counts, n, a.tokens);
    const int lim = kv_limit(a, row, len, cnt);
    const uint16_t* p = nullptr;
    if (lim > 0) {
        const int t = row / a.group, jj = row - t * a.group;
        p = static_cast<const uint16_t*>(a.query) + n * a.q_stride_n + static_cast<int64_t>(h * a.group + jj) * a.q_stride_h +
            t * a.q_stride_t;
    }
    uint32_t x[EP / 2];
    load_row<EP / 8>(a, p, 0, x);
    const float amax = row_max<EP / 2>(a, x);
    float mul, inv;
    row_power(amax, mul, inv);
#pragma unroll
    for (int c = 0; c < EP / 8; ++c) {
        uint32_t q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpack16(x[c * 4 + j], a.query_bf16);
            q[j] = pack_half2(f.x * mul, f.y * mul);
        }
        *reinterpret_cast<uint4*>(out + operand_offset(r, c)) = make_uint4(q[0], q[1], q[2], q[3]);
    }
    const float l = lim > 0 ? lse2[head * a.rows + row] : INFINITY;
    reinterpret_cast<float2*>(out + ColumnShape<EP>::kOperand)[r] = make_float2(inv * a.scale_log2, l);
    reinterpret_cast<int*>(out + ColumnShape<EP>::kOperand + 128 * 8)[r] = lim;
}

struct ColumnParts {
    PromptParts list;      // out: [slot][128] sums
    const uint8_t* blocks;
};

template <bool E4M3, int EP>
__global__ void __launch_bounds__(kColumnThreads, 1) k_kv_columns(KvAttnArgs a, ColumnParts w, int key_tiles) {
    enter_kernel();
    using S = ColumnShape<EP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_addr(smem);
    const uint32_t bars = base + S::kBars;
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + S::kBars + kColumnBars * 8);
    volatile uint32_t* const dead = tmem_slot + 1;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const PromptList list = *w.list.list;
    const int64_t x_begin = list.each * blockIdx.x;
    if (x_begin >= list.total) return;
    const PromptStart start = w.list.starts[blockIdx.x];
    const int count = static_cast<int>(min(list.each, list.total - x_begin)) - start.lead;
    if (count <= 0) return;
    const int row_tiles = (a.rows + kRowTile - 1) / kRowTile;

    if (tid == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(bars + (kBFull + i) * 8, 1);
            mbar_init(bars + (kBEmpty + i) * 8, 1 + 4);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(bars + (kTFull + i) * 8, 1);
            mbar_init(bars + (kTEmpty + i) * 8, 4);
        }
        mbar_init(bars + kKReady * 8, 8);
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_addr(const_cast<uint32_t*>(tmem_slot)))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    // Every role walks the same items; c counts the row tiles of this CTA.
    PromptItem pos(w.list, key_tiles, start);
    uint32_t c = 0;
    if (warp == 9) {
        // ---- row blocks ----
        for (int left = count;;) {
            const int steps = min(pos.tiles - pos.tile, left);
            const int first = row_tiles - pos.tiles + pos.tile;
            const size_t head = static_cast<size_t>(pos.n) * a.kv_heads + pos.h;
            const uint8_t* src = w.blocks + (head * row_tiles + first) * S::kBlock;
            for (int j = 0; j < steps; ++j, ++c, src += S::kBlock) {
                const uint32_t st = c % S::kStages, full = bars + (kBFull + st) * 8;
                mbar_wait(bars + (kBEmpty + st) * 8, (c / S::kStages & 1) ^ 1, dead);
                __syncwarp();
                if (__any_sync(0xffffffffu, *dead != 0)) {  // the stage may not be free
                    left = 0;
                    break;
                }
                if (elect_one()) {
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full), "n"(S::kBlock) : "memory");
                    asm volatile(
                        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                            base + S::kBlocks + st * S::kBlockRoom),
                        "l"(src), "n"(S::kBlock), "r"(full)
                        : "memory");
                }
                __syncwarp();
            }
            left -= steps + kItemCost;
            if (left <= 0) break;
            pos.next(w.list, key_tiles, a.kv_heads);
        }
        // the last copies have landed before the CTA ends
        for (uint32_t k = c > S::kStages ? c - S::kStages : 0; k < c; ++k)
            mbar_drain(bars + (kBFull + k % S::kStages) * 8, k / S::kStages & 1);
    } else if (warp == 8) {
        // ---- products ----
        const uint64_t k_desc = operand_desc(base + S::kKeys, 16, 1024);
        constexpr uint32_t kInstr = instr_desc(kRowTile, false);
        for (int left = count, item = 0;; ++item) {
            const int steps = min(pos.tiles - pos.tile, left);
            mbar_wait(bars + kKReady * 8, item & 1, dead);
            for (int j = 0; j < steps; ++j, ++c) {
                const uint32_t st = c % S::kStages, b = c & 3;
                mbar_wait(bars + (kBFull + st) * 8, c / S::kStages & 1, dead);
                mbar_wait(bars + (kTEmpty + b) * 8, (c >> 2 & 1) ^ 1, dead);
                __syncwarp();
                tc_fence_after();
                const uint64_t q_desc = operand_desc(base + S::kBlocks + st * S::kBlockRoom, 16, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < EP / 16; ++k) {
                        const uint32_t off = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
                        mma_ss(tmem + b * 128, k_desc + off, q_desc + off, kInstr, k > 0);
                    }
                    tc_commit(bars + (kTFull + b) * 8);
                    tc_commit(bars + (kBEmpty + st) * 8);
                }
                __syncwarp();
            }
            left -= steps + kItemCost;
            if (left <= 0) break;
            pos.next(w.list, key_tiles, a.kv_heads);
        }
        // the last products are done before the tensor memory is given up
        mbar_drain(bars + (kTFull + ((c - 1) & 3)) * 8, ((c - 1) >> 2) & 1);
    } else {
        // ---- sums ----
        const int turn = warp >> 2;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        float* const sums = reinterpret_cast<float*>(smem + S::kSums);
        for (int left = count;;) {
            const int steps = min(pos.tiles - pos.tile, left);
            const size_t head = static_cast<size_t>(pos.n) * a.kv_heads + pos.h;
            const int len = kv_length(a.lengths, pos.n, a.capacity), tok = pos.rt * kTokTile;
            const int key = tok + (tid & 127);
            // the keys: a thread takes 16 codes at a time
            for (int v = tid; v < 128 * (EP / 16); v += 256) {
                const int r = v / (EP / 16), e = v % (EP / 16);
                uint4 q = make_uint4(0, 0, 0, 0);
                if (tok + r < len && e * 16 < a.head_dim)
                    q = __ldg(reinterpret_cast<const uint4*>(a.key + (head * a.capacity + tok + r) * a.head_dim + e * 16));
                uint4 lo, hi;
                codes_to_half<E4M3, 0>(q.x, lo.x, lo.y);
                codes_to_half<E4M3, 0>(q.y, lo.z, lo.w);
                codes_to_half<E4M3, 0>(q.z, hi.x, hi.y);
                codes_to_half<E4M3, 0>(q.w, hi.z, hi.w);
                *reinterpret_cast<uint4*>(smem + S::kKeys + operand_offset(r, 2 * e)) = lo;
                *reinterpret_cast<uint4*>(smem + S::kKeys + operand_offset(r, 2 * e + 1)) = hi;
            }
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + kKReady * 8);
            // one scale for the 32 keys of a warp
            const int span = tok + (warp & 3) * 32;
            const float ks = span < len ? a.key_scale[head * a.nblocks + (span >> a.block_shift)] : 0.0f;
            const Pair ks2 = pair_of(ks, ks);
            Pair total = 0;
            for (int j = 0; j < steps; ++j, ++c) {
                if ((c & 1) != static_cast<uint32_t>(turn)) continue;
                Pair sum[2] = {0, 0};  // of this tile: thousands of small weights added to one number would lose bits
                const uint32_t st = c % S::kStages, b = c & 3;
                mbar_wait(bars + (kTFull + b) * 8, c >> 2 & 1, dead);
                mbar_wait(bars + (kBFull + st) * 8, c / S::kStages & 1, dead);  // the block's numbers, for this thread too
                __syncwarp();
                tc_fence_after();
                const uint8_t* const block = smem + S::kBlocks + st * S::kBlockRoom;
                const float4* const rows = reinterpret_cast<const float4*>(block + S::kOperand);
                const int2* const limits = reinterpret_cast<const int2*>(block + S::kOperand + 128 * 8);
                // rows that see less than all of these keys: the first of the tile, where there are any
                const bool ragged = reinterpret_cast<const int*>(limits)[0] < tok + kTokTile ||
                                    reinterpret_cast<const int*>(limits)[127] < tok + kTokTile;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t s[32];
                    tmem_load32(tmem + b * 128 + k * 32 + lanes, s);
                    tmem_wait_load32(s);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float4 f = rows[(k * 32 + i) / 2];  // factor and log2 sum of two rows
                        const Pair x = fma2(pair_of(__uint_as_float(s[i]), __uint_as_float(s[i + 1])),
                                            mul2(pair_of(f.x, f.z), ks2), pair_of(-f.y, -f.w));
                        float u, v;
                        unpair(x, u, v);
                        u = ex2(u);
                        v = ex2(v);
                        if (ragged) {
                            const int2 lim = limits[(k * 32 + i) / 2];
                            if (key >= lim.x) u = 0.0f;
                            if (key >= lim.y) v = 0.0f;
                        }
                        sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pair_of(u, v));
                    }
                }
                total = add2(total, add2(sum[0], sum[1]));
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bars + (kTEmpty + b) * 8);
                    mbar_arrive(bars + (kBEmpty + st) * 8);
                }
            }
            float u, v;
            unpair(total, u, v);
            u += v;
            // both groups' tiles are done, and with them every product of these keys
            if (turn == 1) sums[tid & 127] = u;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (turn == 0) {
                u += sums[tid];
                if (*dead) u = __int_as_float(0x7fc00000);
                if (steps < pos.tiles) {
                    const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + (pos.tile > 0 ? 0 : 1);
                    w.list.out[slot * 128 + tid] = u;
                } else if (key < len) {
                    float* const o = a.weights + head * a.capacity + key;
                    *o = a.accumulate ? *o + u : u;
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");  // the sums have been read
            left -= steps + kItemCost;
            if (left <= 0) break;
            pos.next(w.list, key_tiles, a.kv_heads);
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Adds up the parts of the key tiles that more than one CTA of k_kv_columns worked on.
__global__ void __launch_bounds__(128) k_kv_columns_merge(KvAttnArgs a, PromptParts w, int key_tiles) {
    enter_kernel();
    const PromptList list = *w.list;
    if (list.each * (blockIdx.x + 1) >= list.total) return;
    const PromptItem pos(w, key_tiles, w.starts[blockIdx.x + 1]);
    if (pos.tile == 0 || pos.tile > list.each) return;
    const int c0 = blockIdx.x, parts = 2 + (pos.tiles - pos.tile - 1) / static_cast<int>(list.each);
    const int key = pos.rt * kTokTile + threadIdx.x;
    if (key >= kv_length(a.lengths, pos.n, a.capacity)) return;
    float u = 0.0f;
    for (int k = 0; k < parts; ++k) u += w.out[(static_cast<size_t>(c0) * 2 + (k == 0 ? 1 : 2 * k)) * 128 + threadIdx.x];
    float* const o = a.weights + (static_cast<size_t>(pos.n) * a.kv_heads + pos.h) * a.capacity + key;
    *o = a.accumulate ? *o + u : u;
}

template <bool E4M3, int EP>
int launch_columns(const KvAttnArgs& a, const KvColumnPlan& p, char* ws, const float* lse2, cudaStream_t stream) {
    using S = ColumnShape<EP>;
    const int key_tiles = static_cast<int>((a.capacity + kTokTile - 1) / kTokTile);
    const int64_t blocks = static_cast<int64_t>(a.batch) * a.kv_heads * ((a.rows + kRowTile - 1) / kRowTile);
    if (blocks > INT32_MAX) return set_error(DT_ERR_INVALID, "dt_kv_attention: too many blocks");
    int64_t* const prefix = reinterpret_cast<int64_t*>(ws + p.prefix);
    PromptList* const list = reinterpret_cast<PromptList*>(ws + p.list);
    PromptStart* const starts = reinterpret_cast<PromptStart*>(ws + p.starts);
    uint8_t* const rows = reinterpret_cast<uint8_t*>(ws + p.blocks);
    const ColumnParts w{PromptParts{reinterpret_cast<float*>(ws + p.sums), nullptr, list, starts, prefix, nullptr}, rows};
    int st = launch_kernel("dt_kv_attention", k_kv_row_blocks<E4M3, EP>, dim3(static_cast<unsigned>(blocks)), 128, 0, stream, 1, a,
                           lse2, rows);
    if (st != DT_OK) return st;
    st = launch_kernel("dt_kv_attention", k_kv_prompt_plan<true>, dim3(1), 1024, 0, stream, 1, a, list, starts, prefix,
                       prefix + static_cast<int64_t>(a.batch) * (key_tiles + 1), key_tiles, p.ctas);
    if (st != DT_OK) return st;
    st = launch_kernel("dt_kv_attention", k_kv_columns<E4M3, EP>, dim3(p.ctas), kColumnThreads, S::kSmem, stream, 1, a, w, key_tiles);
    if (st != DT_OK || p.ctas < 2) return st;
    return launch_kernel("dt_kv_attention", k_kv_columns_merge, dim3(p.ctas - 1), 128, 0, stream, 1, a, w.list, key_tiles);
}

}  // namespace

namespace dtb {

KvPromptPlan kv_prompt_plan(int64_t batch, int64_t rows, int64_t head_dim, int sms) {
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t ep = head_dim <= 64 ? 64 : 128, row_tiles = (rows + kItemRows - 1) / kItemRows;
    KvPromptPlan p{};
    p.ctas = sms;
    p.out = 0;
    p.stats = up(static_cast<size_t>(sms) * 2 * kItemRows * ep * 4);
    p.list = p.stats + up(static_cast<size_t>(sms) * 2 * kItemRows * 8);
    p.starts = p.list + up(sizeof(PromptList));
    p.prefix = p.starts + up(static_cast<size_t>(sms) * sizeof(PromptStart));
    p.bytes = p.prefix + up((static_cast<size_t>(batch) * (row_tiles + 1) + batch + 1) * 8);
    return p;
}

int kv_prompt_attention(const KvAttnArgs& a, int code, const KvPromptPlan& p, void* workspace, float* lse2,
                        cudaStream_t stream) {
    char* const ws = static_cast<char*>(workspace);
    if (a.head_dim <= 64)
        return code == DT_KV_E4M3 ? launch<true, 64>(a, p, ws, lse2, stream) : launch<false, 64>(a, p, ws, lse2, stream);
    return code == DT_KV_E4M3 ? launch<true, 128>(a, p, ws, lse2, stream) : launch<false, 128>(a, p, ws, lse2, stream);
}

KvColumnPlan kv_column_plan(int64_t batch, int64_t kv_heads, int64_t rows, int64_t head_dim, int64_t capacity, int sms) {
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t block = head_dim <= 64 ? ColumnShape<64>::kBlock : ColumnShape<128>::kBlock;
    const size_t row_tiles = (rows + kRowTile - 1) / kRowTile, key_tiles = (capacity + kTokTile - 1) / kTokTile;
    KvColumnPlan p{};
    p.ctas = sms;
    p.blocks = 0;
    p.sums = up(static_cast<size_t>(batch) * kv_heads * row_tiles * block);
    p.list = p.sums + up(static_cast<size_t>(sms) * 2 * 128 * 4);
    p.starts = p.list + up(sizeof(PromptList));
    p.prefix = p.starts + up(static_cast<size_t>(sms) * sizeof(PromptStart));
    p.bytes = p.prefix + up((static_cast<size_t>(batch) * (key_tiles + 1) + batch + 1) * 8);
    return p;
}

int kv_column_sums(const KvAttnArgs& a, int code, const KvColumnPlan& p, void* workspace, const float* lse2,
                   cudaStream_t stream) {
    char* const ws = static_cast<char*>(workspace);
    if (a.head_dim <= 64)
        return code == DT_KV_E4M3 ? launch_columns<true, 64>(a, p, ws, lse2, stream)
                                  : launch_columns<false, 64>(a, p, ws, lse2, stream);
    return code == DT_KV_E4M3 ? launch_columns<true, 128>(a, p, ws, lse2, stream)
                              : launch_columns<false, 128>(a, p, ws, lse2, stream);
}

}  // namespace dtb
