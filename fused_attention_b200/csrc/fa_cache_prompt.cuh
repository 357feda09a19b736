// Attention over the cache for many query rows a key/value head: prompts, and chunks of them.
//
// The query heads that share a key/value head and the tokens of a sequence are rows, as in fa_cache_rows.cuh; a work item is 256 of
// them (two tiles of 128, the rows of one tcgen05 tile each) of one sequence and key/value head, against the keys that the
// last of them sees, or, where there are fewer items than SMs, against one of `parts` equal shares of those keys, joined by
// fa_cache_prompt_join.  CTAs are persistent, one an SM, and take items in turn, those with the most keys first.  512 threads:
//
//   warps 0-3, 4-7   softmax of query tile 0 / 1, a thread a row: scores out of tensor memory, exponentials, P (fp16) into tensor
//                    memory; at an item's end the division and Y
//   warps 8-11       loading: codes of 128 keys and values a step into registers, a step ahead, from there as fp16 into the ring of
//                    operand tiles in shared memory (the conversion is exact: no scale is applied to it); queries; scales
//   warp 12, 14      issue Q K^T, P V (tcgen05.mma, fp32 sums in tensor memory)
//   warp 13          works out the items, and which of them have value scales far apart
//
// Scales.  A step's keys have eight groups of 16 with a scale each for K and V (pages are 16 tokens or more).  As in
// fa_cache_rows.cuh the exponent of a weight is score * (row's factor * key scale) + log2(value scale) - M, one multiply-add
// a pair of scores with factors that change from group to group, and the row sum divides the value scale out again (items whose value
// scales lie far apart, kSpanOfScales, go through a loop of their own that takes an exponential more a score: the two cases below with
// every other page zeros and the rest values up to 7 * 10^6, 564 and 198 us).
// A page whose scale is NaN (or below zero) becomes keys that are NaN and values that are zero, so that only rows that see it are NaN.
//
// Bound by the tensor pipe and the exponentials as fa_fwd_pipelined is (per step and tile 1024 tensor clocks of products at
// H = 128 and 1024 clocks of exponentials); what is added here is shared-memory traffic, 64 KB a step written by the loading
// warps beside the 192 KB that the products read.  Measured: a prompt of 4096 tokens on 8000 keys, 32 heads of 128, 383 to 423 us,
// 58 to 64 % of the products' peak (the tensor pipe busy 47 % of a launch by itself, 427 us); 16 prompts of 777 tokens, 16 heads of 64,
// 146 to 151 us.  A step of both tiles takes about 4800 clocks, in which the issuing and loading warps wait for the softmax: registers are
// what it lacks, a row's 128 scores leave few.  (fa_fwd_pair, whose keys have no scales and come as fp16, takes 2750 to 2800 for a step of
// as many scores.)
#pragma once

#include <type_traits>

#include "fa_cache.cuh"
#include "fa_cache_rows.cuh"

namespace fa {

constexpr int kPromptTile = 128;
constexpr int kPromptThreads = 512;
constexpr int kPromptGroups = kPromptTile / 16;   // of keys with a scale of their own

struct PromptArgs {
    CacheView c;
    CacheSeqs s;
    const uint8_t* q;
    uint8_t* y;              // [B, T, heads * H] contiguous
    int64_t q_b, q_t;        // strides in bytes
    uint32_t group, by_group, causal, bf16;
    uint32_t pairs;          // items of a sequence and key/value head, without their parts
    uint32_t whole, parts, items;   // the first `whole` items are worked on whole, the others cut into `parts`; items: with their parts
    float scale_log2;        // log2(e) / sqrt(H)
    float* part_o;           // [items - whole, 256, H]
    float2* part_ml;         // [items - whole, 256]
};

template <int H>
struct PromptCfg {
    static constexpr int kBoxCols = H < 64 ? H : 64;               // of an operand box: a row is one swizzle span
    static constexpr int kSwz = kBoxCols * 2;
    static constexpr int kBoxBytes = kPromptTile * kSwz;
    static constexpr int kTileBytes = kPromptTile * H * 2;
    static constexpr int kQBuffers = H == 128 ? 1 : 2;
    static constexpr int kSlots = H == 128 ? 4 : 8;                // of the ring: K and V tiles in turn
    static constexpr bool kSharedS = H == 128;                     // one score tile for both query tiles: no room for two
    static constexpr uint32_t kColS0 = 0, kColS1 = kSharedS ? 0 : 128;
    static constexpr uint32_t kColP0 = kSharedS ? 128 : 320, kColP1 = kSharedS ? 192 : 448;
    static constexpr uint32_t kColO0 = 256, kColO1 = 384;
    static constexpr int kSmemBytes = (2 * kQBuffers + kSlots) * kTileBytes + 1024;
    // Registers of a thread by role: 128 a thread at launch, so twice the softmax warps' and the others' are 512 at most.  A row of
    // scores is 128 of them; loading holds 32 of codes at H = 128, 16 or fewer below.  Softmax, loading and issuing at H = 64 (16 prompts
    // of 777 tokens): 200, 64, 48 150 us, 208, 64, 32 144, 208, 56, 40 153, 216, 48, 32 181; at H = 128 (4096 tokens on 8000 keys): 192, 80,
    // 48 394, 192, 88, 40 390, 200, 72, 40 420, 184, 96, 48 462.
    static constexpr int kSoftmaxRegs = H == 128 ? 192 : 208, kLoadRegs = H == 128 ? 88 : 64, kIssueRegs = H == 128 ? 40 : 32;
    static_assert(2 * kSoftmaxRegs + kLoadRegs + kIssueRegs <= 512, "registers of the four warpgroups");
    // barriers
    static constexpr int QFULL = 0, QEMPTY = QFULL + kQBuffers, FULL = QEMPTY + kQBuffers, EMPTY = FULL + kSlots, S0 = EMPTY + kSlots, SFREE0 = S0 + 2,
                         P0 = SFREE0 + 2, PV0 = P0 + 2, FINAL = PV0 + 2, FINAL2 = FINAL + 1, COEF = FINAL2 + 1, SCALE = COEF + 8, ITEM = SCALE + kSlots, IFREE = ITEM + 4,
                         kBarriers = IFREE + 4;
};

// Scales of a step's groups as the softmax takes them.
struct __align__(16) PromptScales {
    float ks[kPromptGroups], vlog[kPromptGroups], vinv[kPromptGroups];
};
// One, two groups' values.  Volatile: they are loaded where they are used, and not held in registers, of which a row's scores take most.
__device__ __forceinline__ float one_group(uint32_t addr) {
    float x;
    asm volatile("ld.volatile.shared.f32 %0, [%1];" : "=f"(x) : "r"(addr));
    return x;
}
__device__ __forceinline__ float2 two_groups(uint32_t addr) {
    float2 x;
    asm volatile("ld.volatile.shared.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(addr));
    return x;
}

__device__ __forceinline__ uint32_t prompt_swizzled(uint32_t row, uint32_t piece, uint32_t span) {
    return row * span + ((piece ^ ((row * span >> 7) & (span / 16u - 1u))) << 4);
}

// 16 bytes of global memory (zeros where `in` is false: nothing is read then), or 8 and the 8 at `from` + 64.  Volatile: these stand
// where their registers have just been let go of, long before their use.
__device__ __forceinline__ void ld_zero_16(const uint8_t* from, bool in, uint4& w) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                 "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "=&r"(w.x), "=&r"(w.y), "=&r"(w.z), "=&r"(w.w) : "l"(from), "r"(static_cast<uint32_t>(in)));
}
__device__ __forceinline__ void ld_16(const uint8_t* from, uint4& w) {
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(from));
}
__device__ __forceinline__ void ld_8_8(const uint8_t* from, uint4& w) {
    asm volatile("ld.global.v2.u32 {%0, %1}, [%4];\n\tld.global.v2.u32 {%2, %3}, [%4 + 64];" : "=&r"(w.x), "=&r"(w.y), "=&r"(w.z), "=&r"(w.w) : "l"(from));
}

// What an item is: one warp works it out ahead of the others (lengths come from memory, rows and heads from divisions) and passes it
// on in shared memory.
using PlainItem = std::integral_constant<bool, false>;
using WideItem = std::integral_constant<bool, true>;   // value scales far apart
#ifdef FA_DEBUG
// Whether 16 tokens of a page begin `at` units of 16 bytes behind their head's first code.
__device__ __forceinline__ bool codes_inside(const CacheView& c, bool is_v, uint32_t at) {
    const uint64_t page = is_v ? c.v_page : c.k_page, token = is_v ? c.v_token : c.k_token, from = static_cast<uint64_t>(at) * 16u;
    for (uint32_t in_page = 0; in_page < c.page; in_page += 16)
        if (from >= in_page * token && (page == 0 ? from == in_page * token : (from - in_page * token) % page == 0 && (from - in_page * token) / page < c.n_pages)) return true;
    return false;
}
#endif
struct PromptItem {
    uint32_t b, head;
    uint32_t t0, first;             // the first row is row `first` of `group` of token t0
    uint32_t n_rows, held, count;
    uint32_t farthest;              // keys [0, farthest) are seen by some row
    uint32_t step0, steps;          // this part's
    uint32_t tile_steps[2];         // ... that query tile 0, 1 takes part in: the first of them
    uint32_t slot;                  // of the part's sums; kNoToken: not a part
    uint32_t there;                 // 0 behind the last item
};
constexpr uint32_t kPromptItems = 4;   // that are known ahead

// Keys [0, ...) that some of the rows [row0, row0 + rows) sees.
__device__ __forceinline__ uint32_t prompt_farthest(const PromptArgs& p, const PromptItem& it, uint32_t row0, uint32_t rows) {
    const uint32_t t_first = row0 / p.group, t_end = rows == 0 ? 0u : min(it.count, (row0 + rows - 1u) / p.group + 1u);   // tokens [t_first, t_end)
    if (t_first >= t_end) return 0;
    return p.causal ? (it.held + t_end > it.count ? min(it.held, it.held + t_end - it.count) : 0u) : it.held;
}
__device__ __forceinline__ PromptItem prompt_item(const PromptArgs& p, uint32_t index) {
    PromptItem it;
    const uint32_t heads = p.s.B * p.c.heads;
    uint32_t part = 0, parts = 1;
    it.slot = kNoToken;
    if (index >= p.whole) {
        it.slot = index - p.whole;
        parts = p.parts, part = it.slot % parts, index = p.whole + it.slot / parts;
    }
    const uint32_t bh = index % heads, pair = p.pairs - 1u - index / heads, row0 = pair * (2 * kPromptTile);
    it.b = bh / p.c.heads;
    it.head = bh % p.c.heads;
    it.t0 = row0 / p.group;
    it.first = row0 % p.group;
    it.n_rows = min(2u * kPromptTile, p.s.T * p.group - row0);
    it.held = cache_length(p.c, p.s, it.b);
    it.count = cache_count(p.s, it.b);
    const uint32_t half = min(it.n_rows, static_cast<uint32_t>(kPromptTile));
    const uint32_t far[2] = {prompt_farthest(p, it, row0, half), prompt_farthest(p, it, row0 + half, it.n_rows - half)};
    it.farthest = max(far[0], far[1]);
    const uint32_t all = (it.farthest + kPromptTile - 1u) / kPromptTile;
    it.step0 = all * part / parts;
    it.steps = all * (part + 1u) / parts - it.step0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t mine = (far[i] + kPromptTile - 1u) / kPromptTile;
        it.tile_steps[i] = mine <= it.step0 ? 0u : min(it.steps, mine - it.step0);
    }
    it.there = 1;
    return it;
}
// Whether the value scales of a head's pages with the keys [key0, end) lie further apart than kSpanOfScales.  All lanes of a warp.
__device__ __forceinline__ bool prompt_wide(const PromptArgs& p, uint32_t b, uint32_t head, uint32_t key0, uint32_t end, uint32_t lane) {
    const int32_t* const table = p.s.table + b * p.s.table_stride;
    const uint32_t blocks = ((end - 1u) >> p.c.page_shift) + 1u;
    int least = 255, most = 0;   // biased exponents
#pragma unroll 2
    for (uint32_t block = (key0 >> p.c.page_shift) + lane; block < blocks; block += 32) {
        if (!FA_CACHE_OK(p.c.status, kDbgEntry, b < p.s.B && block < p.s.width)) break;
        const uint32_t page = static_cast<uint32_t>(table[block]);
        if (page >= p.c.n_pages) continue;
        const int size = max(__float_as_int(p.c.v_scale[static_cast<uint64_t>(page) * p.c.heads + head]) >> 23, 27);   // (2^-100 at least)
        least = min(least, size), most = max(most, size);
    }
    return __reduce_max_sync(0xFFFFFFFFu, most) - __reduce_min_sync(0xFFFFFFFFu, least) > kSpanOfScales;
}
// Token and query head (of the key/value head's) of row r of an item.  `by_group`: 2^32 / group rounded up, with which the product's
// upper half is the quotient (group < 2^16, and what is divided is less than group + 256).
__device__ __forceinline__ void prompt_row(const PromptArgs& p, uint32_t t0, uint32_t first, uint32_t r, uint32_t& t, uint32_t& i) {
    const uint32_t n = first + r, q = p.group == 1 ? n : __umulhi(n, p.by_group);
    t = t0 + q;
    i = n - q * p.group;
}

template <int H>
__device__ __forceinline__ void prompt_issue_qk(uint32_t tS, uint32_t sQ, uint32_t sK) {
    using C = PromptCfg<H>;
    constexpr uint32_t idesc = make_idesc_f16(kPromptTile, 0);
    const uint64_t dq = make_smem_desc<C::kSwz>(sQ, 16), dk = make_smem_desc<C::kSwz>(sK, 16);
#pragma unroll
    for (int ks = 0; ks < H / 16; ++ks) {
        const uint32_t off = ((ks * 16) / C::kBoxCols) * C::kBoxBytes + ((ks * 16) % C::kBoxCols) * 2;
        mma_ss(tS, dq + (off >> 4), dk + (off >> 4), idesc, ks > 0 ? 1u : 0u);
    }
}
template <int H>
__device__ __forceinline__ void prompt_issue_pv(uint32_t tO, uint32_t tP, uint32_t sV, uint32_t accumulate) {
    using C = PromptCfg<H>;
    constexpr uint32_t idesc = make_idesc_f16(H, 1);
    const uint64_t dv = make_smem_desc<C::kSwz>(sV, C::kBoxBytes);
#pragma unroll
    for (int ks = 0; ks < kPromptTile / 16; ++ks) mma_ts(tO, tP + ks * 8, dv + ((ks * 16 * C::kSwz) >> 4), idesc, (accumulate | ks) ? 1u : 0u);
}

// Weights of the groups kG0 and kG0 + 1 of a row, packed as fp16 pairs (8 words a group); adds the groups' sums to `l`, with the value
// scale divided out.  The exponent is one multiply-add, score * cu + (vlog - ref): `ref` is a whole number, so that with scales
// that are powers of two the bracket is exact.  `shrink`: see prompt_reference.  kWide: see kSpanOfScales.
template <int kG0, int kSame, bool kWide>
__device__ __forceinline__ void prompt_weights(const float (&s)[kPromptTile], uint32_t sc, float coef, float shrink, float ref, uint32_t (&pk)[16], float& l) {
    constexpr int kAt = kSame == 4 ? kG0 & ~3 : kG0;
    float2 ks, vlog, vinv;
    if constexpr (kSame == 1) {
        ks = two_groups(sc + 4 * kAt), vlog = two_groups(sc + 4 * (kPromptGroups + kAt)), vinv = two_groups(sc + 4 * (2 * kPromptGroups + kAt));
    } else {
        ks.x = one_group(sc + 4 * kAt), vlog.x = one_group(sc + 4 * (kPromptGroups + kAt)), vinv.x = one_group(sc + 4 * (2 * kPromptGroups + kAt));
    }
    uint64_t sum_a = 0, sum_b = 0, c2 = 0, a2 = 0, bare2 = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int u = kG0 + half;
        if (half == 0 || kSame == 1) {
            // (at least 1e-37: a masked score, -inf, must stay that)
            const float cu = fmaxf(coef * (half ? ks.y : ks.x), 1e-37f), add = fmaf(half ? vlog.y : vlog.x, shrink, -ref);
            c2 = pack_f32x2(cu, cu), a2 = pack_f32x2(add, add);
            if (kWide) {   // (a page that is not there adds nothing)
                const float bare = (half ? vinv.y : vinv.x) == 0.0f ? -INFINITY : kSumLift - ref;
                bare2 = pack_f32x2(bare, bare);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float x0, x1;
            unpack_f32x2(fma_f32x2(pack_f32x2(s[u * 16 + 2 * e], s[u * 16 + 2 * e + 1]), c2, a2), x0, x1);
            const float w0 = ex2_approx(x0), w1 = ex2_approx(x1);
            pk[half * 8 + e] = pack_half2(w0, w1);
            uint64_t both = pack_f32x2(w0, w1);
            if (kWide) {
                unpack_f32x2(fma_f32x2(pack_f32x2(s[u * 16 + 2 * e], s[u * 16 + 2 * e + 1]), c2, bare2), x0, x1);
                both = pack_f32x2(ex2_approx(x0), ex2_approx(x1));
            }
            if (e & 1) sum_b = add_f32x2(sum_b, both);
            else sum_a = add_f32x2(sum_a, both);
        }
        if (half == 1 || kSame == 1) {
            float lo, hi;
            unpack_f32x2(add_f32x2(sum_a, sum_b), lo, hi);
            l = fmaf(lo + hi, kWide ? kSumUnlift : half && kSame == 1 ? vinv.y : vinv.x, l);
            sum_a = sum_b = 0;
        }
    }
}
// Largest of 16 scores.
__device__ __forceinline__ float largest_of_16(const float* x) {
    float a = max3(x[0], x[1], x[2]), b = max3(x[3], x[4], x[5]);
#pragma unroll
    for (int e = 6; e < 14; e += 4) {
        a = max3(a, x[e], x[e + 1]);
        b = max3(b, x[e + 2], x[e + 3]);
    }
    return max3(a, b, fmaxf(x[14], x[15]));
}
// Largest exponent of a row.
template <int kSame>
__device__ __forceinline__ float prompt_top(const float (&s)[kPromptTile], uint32_t sc, float coef, float shrink) {
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kPromptGroups; u += kSame) {
        float most = largest_of_16(s + u * 16);
#pragma unroll
        for (int v = 1; v < kSame; ++v) most = fmaxf(most, largest_of_16(s + (u + v) * 16));
        top = fmaxf(top, fmaf(most, fmaxf(coef * one_group(sc + 4 * u), 1e-37f), one_group(sc + 4 * (kPromptGroups + u)) * shrink));
    }
    return top;
}
// A new reference for a row whose largest exponent is `top`, and the factor for O so far; `l` is multiplied by it.  Beside one of 2^22 and more an
// exponent would not be known to a fraction, and a weight could exceed fp16: all the row's exponents are then shrunk by a power of
// two that brings it below.  The largest stays the largest, and exponents of that size differ by whole numbers or not at all, so
// that hardly anything but the largest counts before and after (scores that tie beside value scales that differ are not weighed exactly there).
template <bool kWide>
__device__ __forceinline__ float prompt_reference(float top, float& m, float& coef, float& shrink, float& l) {
    const float grown = 1.0f / shrink, whole = top * grown;
    const uint32_t size = (__float_as_uint(whole) >> 23) & 0xFFu;   // biased exponent
    const float now = size > 127u + 22u ? __uint_as_float((127u + 127u + 22u - size) << 23) : 1.0f;
    const float m_new = ceilf(whole * now), by = m * grown - m_new * (1.0f / now), alpha = ex2_approx(by);
    m = m_new;
    l = kWide ? times_power(l, by) : l * alpha;
    coef *= grown * now;
    shrink = now;
    return alpha;
}

// kSame: how many groups in a row have one scale (a page's: 4 at 64 tokens and more, 2 at 32, 1 at 16).  The softmax reads and
// combines the scales once for so many: with pages of 64 tokens 391 us against 408 (a prompt of 4096 tokens on 8000 keys, 32 heads of
// 128), 150 against 157 (16 prompts of 777, heads of 64).
template <int H, int kSame>
__global__ void __launch_bounds__(kPromptThreads, 1) fa_cache_prompt(const PromptArgs p) {
    using C = PromptCfg<H>;
    constexpr uint32_t NS = C::kSlots, kGroups = kPromptGroups;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[C::kBarriers];
    __shared__ PromptScales scales[NS];           // of step g in entry g % NS (free when the V tile of that step is)
    // Rows' factors, by item.  Eight, because loading may be ahead of a softmax by no more than the ring has steps (four at most):
    // a step's V tile is let go of when both tiles that take part in the step have given their P.
    __shared__ float s_coef[8][2 * kPromptTile];
    __shared__ PromptItem items[kPromptItems];
    __shared__ uint32_t s_wide[8];                // whether an item's value scales lie far apart (kSpanOfScales); by item, as s_coef
    __shared__ uint32_t tmem_slot, abort_flag;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ring = base + 2 * C::kQBuffers * C::kTileBytes;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    auto q_addr = [&](uint32_t k, uint32_t i) { return base + ((k % C::kQBuffers) * 2 + i) * C::kTileBytes; };
    auto slot_addr = [&](uint32_t n) { return ring + (n % NS) * C::kTileBytes; };
    const WaitCtl ctl{p.c.status, &abort_flag, kWaitCapCycles, nullptr, 0};

    if (tid == 0) {
        for (int i = 0; i < C::kBarriers; ++i) {
            const bool by_loaders = (i >= C::QFULL && i < C::QEMPTY) || (i >= C::FULL && i < C::EMPTY);
            const bool by_softmax = i >= C::SFREE0 && i < C::PV0;
            // (an item is let go of by 8 softmax warps, 4 loading and 2 issuing; of its rows' factors warp 13 is one more, with s_wide)
            mbar_init(bar(i), i >= C::IFREE ? 14u : i >= C::COEF && i < C::SCALE ? 5u : by_loaders || by_softmax ? 4u : 1u);
        }
        abort_flag = 0;
        fence_mbar_init();
    }
#ifdef FA_DEBUG
    if (tid == 0) g_dbg.tmem_base = 0, g_dbg.tmem_cols = 512, g_dbg.ctl = ctl;
    for (uint32_t i = tid; i < sizeof(scales) / 4; i += kPromptThreads) reinterpret_cast<uint32_t*>(scales)[i] = 0xFFFFFFFFu;
    for (uint32_t i = tid; i < sizeof(s_coef) / 4; i += kPromptThreads) reinterpret_cast<uint32_t*>(s_coef)[i] = 0xFFFFFFFFu;
    FA_CACHE_POISON(base, (2 * C::kQBuffers + C::kSlots) * C::kTileBytes);
    fence_proxy_async_smem();
    auto tile_ok = [&](uint32_t at, uint32_t from, uint32_t tiles) { return at >= from && at + 16u <= from + tiles * C::kTileBytes; };
#endif
    if (warp == 12) {
        tmem_alloc(smem_u32(&tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_wait();
    grid_dep_launch();
    const uint32_t tmem = tmem_slot;
#ifdef FA_DEBUG
    if (tid == 0) g_dbg.tmem_base = tmem;
    __syncthreads();
#endif
    auto item_wait = [&](uint32_t n) { return mbar_wait(bar(C::ITEM + n % kPromptItems), (n / kPromptItems) & 1u, ctl, kCacheTimeout | C::ITEM); };
    auto item_done = [&](uint32_t n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::IFREE + n % kPromptItems));
    };

    if (warp < 8) {
        // ---------------------------------------------------------------- softmax of tile i
        setmaxnreg_inc<C::kSoftmaxRegs>();
        const uint32_t i = warp >> 2, r = tid & 127u, lane_off = ((warp & 3u) * 32u) << 16;
        const uint32_t tS = tmem + lane_off + (i ? C::kColS1 : C::kColS0), tP = tmem + lane_off + (i ? C::kColP1 : C::kColP0),
                       tO = tmem + lane_off + (i ? C::kColO1 : C::kColO0);
        uint32_t g = 0, k = 0, before = 0;   // this tile's steps, items with steps, steps of the items in front of this one
        for (uint32_t nth = 0;; ++nth) {
            if (!item_wait(nth)) break;
            const volatile PromptItem& it = items[nth % kPromptItems];   // (read where it is needed, not held in registers)
            if (it.there == 0) break;
            const uint32_t row = i * kPromptTile + r, steps = it.tile_steps[i];
            uint32_t key0 = it.step0 * kPromptTile, step = before, limit, t, h;
            prompt_row(p, it.t0, it.first, row, t, h);
            {   // keys that the row sees
                const uint32_t held = it.held, count = it.count;
                limit = !p.causal ? held : held + t >= count ? min(held, held + t - count + 1u) : 0u;
                if (row >= it.n_rows || t >= count) limit = 0;
            }
            // a row that sees nothing counts as seeing everything, so that nobody waits for it, and is written as zeros
            const uint32_t masked_from = limit == 0 ? kNoToken : limit;
            float m = -INFINITY, l = 0.0f, coef = 0.0f, shrink = 1.0f;
            if (steps > 0) {
                mbar_wait(bar(C::COEF + (k & 7u)), (k >> 3) & 1u, ctl, kCacheTimeout | C::COEF);
                coef = s_coef[k & 7u][row];
            }
            auto pass = [&](auto is_wide) {   // over the item's steps
                constexpr bool kWide = decltype(is_wide)::value;
#pragma unroll 1
                for (uint32_t j = 0; j < steps; ++j, ++g, ++step, key0 += kPromptTile) {
                    mbar_wait(bar(C::S0 + i), g & 1u, ctl, kCacheTimeout | (C::S0 + i));
                    tc_fence_after();
                    __syncwarp();
                    float s[kPromptTile];
#pragma unroll
                    for (int c = 0; c < kPromptTile; c += 32) tmem_ld32(tS + c, s + c);
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(C::SFREE0 + (C::kSharedS ? 0 : i)));
                    const uint32_t sc = smem_u32(scales) + (step % NS) * static_cast<uint32_t>(sizeof(PromptScales));
                    mbar_wait(bar(C::SCALE + step % NS), (step / NS) & 1u, ctl, kCacheTimeout | C::SCALE);
                    if (__any_sync(0xFFFFFFFFu, key0 + kPromptTile > masked_from)) {
                        const int valid = static_cast<int>(masked_from) - static_cast<int>(key0);
#pragma unroll
                        for (int w = 0; w < 4; ++w) {   // (a bit a score: fewer instructions than a comparison each, 168 us against 173 with 16 prompts of 777)
                            const int left = valid - w * 32;
                            const uint32_t seen = left >= 32 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << left) - 1u;
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(seen >> e & 1u)) s[w * 32 + e] = -INFINITY;
                        }
                    }
                    // The reference moves when an exponent exceeds it by more than 8 (weights stay below 2^9); a row that has seen nothing
                    // yet takes the first that it sees.
                    const float top = prompt_top<kSame>(s, sc, coef, shrink);
                    float alpha = 1.0f;
                    if (__any_sync(0xFFFFFFFFu, top > m + kRowsSlack)) {
                        if (top > m + kRowsSlack) alpha = prompt_reference<kWide>(top, m, coef, shrink, l);
                    }
                    const float ref = m == -INFINITY ? 0.0f : m;
                    // the first quarter's weights are kept in registers: the last step's P V may still be reading P
                    uint32_t pk[16];
                    prompt_weights<0, kSame, kWide>(s, sc, coef, shrink, ref, pk, l);
                    if (g > 0) {
                        mbar_wait(bar(C::PV0 + i), (g - 1u) & 1u, ctl, kCacheTimeout | (C::PV0 + i));
                        tc_fence_after();
                    }
                    __syncwarp();
                    tmem_st16(tP, pk);
                    prompt_weights<2, kSame, kWide>(s, sc, coef, shrink, ref, pk, l);
                    tmem_st16(tP + 16, pk);
                    prompt_weights<4, kSame, kWide>(s, sc, coef, shrink, ref, pk, l);
                    tmem_st16(tP + 32, pk);
                    prompt_weights<6, kSame, kWide>(s, sc, coef, shrink, ref, pk, l);
                    tmem_st16(tP + 48, pk);
                    if (j > 0 && __any_sync(0xFFFFFFFFu, alpha != 1.0f)) {   // (an item's first P V overwrites O)
                        // here, where the scores' registers are free; the last step's P V has retired, and the next waits for P
                        constexpr int kCols = 16;
#pragma unroll 1
                        for (int c = 0; c < H; c += kCols) {
                            float o[kCols];
                            uint32_t w[kCols];
                            tmem_ld16(tO + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < kCols; ++e) w[e] = __float_as_uint(o[e] * alpha);
                            tmem_st16(tO + c, w);
                        }
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(C::P0 + i));
                }
            };
            if (steps > 0) {
                if (__builtin_expect(s_wide[k & 7u] != 0, 0)) pass(WideItem());
                else pass(PlainItem());
            }
            // ---- the item's end: this row of O.  (The next item's first P V waits for P from these warps.)
            const bool any = steps > 0, there = row < it.n_rows;
            if (it.steps > 0) ++k, before += it.steps;
            if (any) {
                mbar_wait(bar(C::PV0 + i), (g - 1u) & 1u, ctl, kCacheTimeout | (C::PV0 + i));
                tc_fence_after();
                __syncwarp();
            }
            const uint32_t slot = it.slot;
            if (slot == kNoToken) {
                const float f = masked_from == kNoToken || l == 0.0f ? 0.0f : 1.0f / l;
                prompt_row(p, it.t0, it.first, row, t, h);
                uint8_t* const to = p.y + ((static_cast<uint64_t>(it.b) * p.s.T + t) * (p.c.heads * p.group) + it.head * p.group + h) * (2 * H);
                const bool inside = !there || FA_CACHE_OK(p.c.status, kDbgRow, it.b < p.s.B && t < p.s.T && h < p.group && it.head < p.c.heads);
                constexpr int kCols = H < 32 ? 16 : 32;
#pragma unroll 1
                for (int c = 0; c < H; c += kCols) {
                    float o[kCols];
                    if (any) {
                        tmem_ld<kCols>(tO + c, o);
                        tmem_wait_ld();
                    }
                    if (there && inside) {
#pragma unroll
                        for (int e = 0; e < kCols; e += 8) {
                            uint4 w = make_uint4(0, 0, 0, 0);
                            if (masked_from != kNoToken)
                                w = make_uint4(pack_16(o[e] * f, o[e + 1] * f, p.bf16), pack_16(o[e + 2] * f, o[e + 3] * f, p.bf16),
                                               pack_16(o[e + 4] * f, o[e + 5] * f, p.bf16), pack_16(o[e + 6] * f, o[e + 7] * f, p.bf16));
                            *reinterpret_cast<uint4*>(to + 2 * (c + e)) = w;
                        }
                    }
                }
            } else {
                const uint64_t at = static_cast<uint64_t>(slot) * (2 * kPromptTile) + row;
                constexpr int kCols = H < 32 ? 16 : 32;
                const bool inside = FA_CACHE_OK(p.c.status, kDbgScratch, slot < p.items - p.whole);
                if (there && inside) p.part_ml[at] = make_float2(masked_from == kNoToken || !any ? -INFINITY : m / shrink, masked_from == kNoToken || !any ? 0.0f : l);
                if (any)
#pragma unroll 1
                    for (int c = 0; c < H; c += kCols) {
                        float o[kCols];
                        tmem_ld<kCols>(tO + c, o);
                        tmem_wait_ld();
                        if (there && inside) {
#pragma unroll
                            for (int e = 0; e < kCols; e += 4) *reinterpret_cast<float4*>(p.part_o + at * H + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                        }
                    }
            }
            tc_fence_before();
            item_done(nth);
        }
    } else if (warp < 12) {
        // ---------------------------------------------------------------- loading
        setmaxnreg_dec<C::kLoadRegs>();
        constexpr uint32_t kLanes = H / 16;                // that share a row of codes, 16 each
        constexpr uint32_t kRowsPass = 128 / kLanes;
        constexpr uint32_t kPasses = kPromptTile / kRowsPass;
        constexpr uint32_t kFirst = H == 128 ? 8 : 16;     // distance of the lanes' first codes
        const uint32_t lt = tid - 256u, j16 = lt % kLanes, r_in = lt / kLanes;
        uint32_t n = 0, k = 0, g = 0;   // ring items, items, steps so far
        for (uint32_t nth = 0;; ++nth) {
            if (!item_wait(nth)) break;
            const PromptItem& it = items[nth % kPromptItems];
            if (it.there == 0) break;
            if (it.steps == 0) {
                item_done(nth);
                continue;
            }
            const int32_t* const table = p.s.table + it.b * p.s.table_stride;
            // ---- a step's pages: lane l (of every warp) has group l's.  The table entry is asked for a step ahead, the scales half
            // a step: nothing may depend at once on what has just been asked for.
            // A group's place is a multiple of 16 bytes from its head's first page; what is not there is read from that page and thrown
            // away (`spoilt`), so that loads depend on nothing but their address.
            int32_t entry = -1;
            bool wanted = false, none = false;
            float ks = 1.0f, vs = 1.0f;
            uint32_t k_at = 0, v_at = 0;
            auto ask = [&](uint32_t step) {
                const uint32_t at = (it.step0 + step) * kPromptTile + (lane & 7u) * 16u;
                wanted = step < it.steps && at < it.farthest && FA_CACHE_OK(p.c.status, kDbgEntry, it.b < p.s.B && (at >> p.c.page_shift) < p.s.width);
                entry = wanted ? table[at >> p.c.page_shift] : -1;
            };
            auto look_up = [&] {
                ks = 1.0f, vs = 1.0f;
                none = static_cast<uint32_t>(entry) >= p.c.n_pages;
                k_at = v_at = 0;
                if (none) {
                    if (wanted && lane < 8 && warp == 8) cache_report(p.c.status, kCacheBadPage);
                } else {
                    const uint64_t s_at = static_cast<uint64_t>(entry) * p.c.heads + it.head;
                    ks = p.c.k_scale[s_at], vs = p.c.v_scale[s_at];
                    const uint32_t in_page = ((lane & 7u) * 16u) & (p.c.page - 1);
                    k_at = static_cast<uint32_t>((static_cast<uint64_t>(entry) * p.c.k_page + in_page * p.c.k_token) >> 4);
                    v_at = static_cast<uint32_t>((static_cast<uint64_t>(entry) * p.c.v_page + in_page * p.c.v_token) >> 4);
                }
            };
            uint4 codes[kPasses];
            const uint8_t* const k_base = p.c.k + it.head * p.c.k_head + (r_in & 15u) * p.c.k_token + kFirst * j16;
            const uint8_t* const v_base = p.c.v + it.head * p.c.v_head + (r_in & 15u) * p.c.v_token + kFirst * j16;
            // pass c of a step's keys (values): this thread's 16 codes
            auto load = [&](uint32_t c, bool is_v) {
                const uint32_t group_at = __shfl_sync(0xFFFFFFFFu, is_v ? v_at : k_at, (c * kRowsPass + r_in) >> 4);
                const uint8_t* const from = (is_v ? v_base : k_base) + static_cast<uint64_t>(group_at) * 16u;
                if (!FA_CACHE_OK(p.c.status, kDbgCodes, it.head < p.c.heads && codes_inside(p.c, is_v != 0, group_at))) return;
                if constexpr (H == 128) ld_8_8(from, codes[c]);   // eight codes of either operand box
                else ld_16(from, codes[c]);
            };
            ask(0);
            // ---- queries, several rows of a thread in flight
            if (k >= C::kQBuffers) mbar_wait(bar(C::QEMPTY + k % C::kQBuffers), (k / C::kQBuffers - 1u) & 1u, ctl, kCacheTimeout | C::QEMPTY);
            constexpr uint32_t kQLanes = H / 8, kQRows = 128 / kQLanes, kQPasses = 2 * kPromptTile / kQRows, kFlight = kQPasses < 4 ? kQPasses : 4;
            const uint32_t piece = lt % kQLanes;
#pragma unroll 1
            for (uint32_t pass = 0; pass < kQPasses; pass += kFlight) {
                uint4 in_flight[kFlight];
#pragma unroll
                for (uint32_t f = 0; f < kFlight; ++f) {
                    const uint32_t r = (pass + f) * kQRows + lt / kQLanes;
                    uint32_t t, h;
                    prompt_row(p, it.t0, it.first, r, t, h);
                    const bool in = r < it.n_rows && t < it.count && FA_CACHE_OK(p.c.status, kDbgRow, it.b < p.s.B && t < p.s.T && h < p.group && it.head < p.c.heads);
                    ld_zero_16(p.q + (in ? it.b * p.q_b + t * p.q_t + static_cast<int64_t>(it.head * p.group + h) * (2 * H) + 16 * piece : 0), in, in_flight[f]);
                }
#pragma unroll
                for (uint32_t f = 0; f < kFlight; ++f) {
                    const uint32_t r = (pass + f) * kQRows + lt / kQLanes;
                    uint4 w = in_flight[f];
                    float coef = p.scale_log2;
                    if (p.bf16) {   // to the range of fp16, by a power of two a row
                        uint32_t x[4] = {w.x, w.y, w.z, w.w};
                        float most = 0.0f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 y = unpack_16(x[e], true);
                            most = fmaxf(most, fmaxf(fabsf(y.x), fabsf(y.y)));
                        }
#pragma unroll
                        for (uint32_t d = kQLanes / 2; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
                        const uint32_t e8 = max(__float_as_uint(most) >> 23, 40u);   // biased: 2^(e8 - 127) <= most, unless that is tiny
                        float up = 1.0f;
                        if (e8 < 255) coef *= __uint_as_float((e8 - 7) << 23), up = __uint_as_float((261 - e8) << 23);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 y = unpack_16(x[e], true);
                            x[e] = pack_half2(y.x * up, y.y * up);
                        }
                        w = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                    constexpr uint32_t kPieces = C::kSwz / 16;   // of a box's row
                    const uint32_t q_to = q_addr(k, r >> 7) + (piece / kPieces) * C::kBoxBytes + prompt_swizzled(r & 127u, piece % kPieces, C::kSwz);
                    if (FA_CACHE_OK(p.c.status, kDbgTile, tile_ok(q_to, q_addr(k, r >> 7), 1))) st_shared_v4(q_to, w.x, w.y, w.z, w.w);
                    if (piece == 0) s_coef[k & 7u][r] = coef;
                }
            }
            look_up();
#pragma unroll
            for (uint32_t c = 0; c < kPasses; ++c) load(c, false);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar(C::QFULL + k % C::kQBuffers));
                mbar_arrive(bar(C::COEF + (k & 7u)));
            }
            ++k;

            // ---- keys and values, K and V of a step in turn
#pragma unroll 1
            for (uint32_t step = 0; step < it.steps; ++step, ++g) {
                // groups without a page (lower byte), and with a scale that is NaN or below zero; whether the keys end within the step
                const uint32_t gone = __ballot_sync(0xFFFFFFFFu, none) & 0xFFu, poisoned = __ballot_sync(0xFFFFFFFFu, !(ks >= 0.0f && vs >= 0.0f)) & 0xFFu;
                const uint32_t left = it.farthest - (it.step0 + step) * kPromptTile;
                const bool spoilt = (gone | poisoned) != 0 || left < kPromptTile;
                ask(step + 1);
#pragma unroll
                for (uint32_t is_v = 0; is_v < 2; ++is_v, ++n) {
                    if (n >= NS) mbar_wait(bar(C::EMPTY + n % NS), (n / NS - 1u) & 1u, ctl, kCacheTimeout | (C::EMPTY + n % NS));
                    if (is_v == 0 && lane < kGroups && warp == 8) {   // (the V tile of the step that had this entry has been let go of)
                        PromptScales& sc = scales[g % NS];
                        const bool bad = !(ks >= 0.0f && vs >= 0.0f);
                        const float held_up = bad || !(vs > 0x1p-100f) ? (bad ? 1.0f : 0x1p-100f) : vs, vlog = __log2f(held_up);
                        sc.ks[lane] = bad ? 1.0f : ks;
                        sc.vlog[lane] = none ? -INFINITY : vlog;
                        sc.vinv[lane] = none ? 0.0f : exp2f(-vlog);
                    }
                    if (is_v == 1) look_up();   // of the next step
                    const uint32_t to = slot_addr(n);
#pragma unroll
                    for (uint32_t c = 0; c < kPasses; ++c) {
                        const uint32_t r = c * kRowsPass + r_in;
                        uint32_t x[8];
                        e4m3x4_to_half2(codes[c].x, x[0], x[1]);
                        e4m3x4_to_half2(codes[c].y, x[2], x[3]);
                        e4m3x4_to_half2(codes[c].z, x[4], x[5]);
                        e4m3x4_to_half2(codes[c].w, x[6], x[7]);
                        if (spoilt) {
                            const bool out = r >= left || (gone >> (r >> 4) & 1u), bad = poisoned >> (r >> 4) & 1u;
                            const uint32_t instead = !out && bad && !is_v ? 0x7E007E00u : 0u;
                            if (out || bad)
#pragma unroll
                                for (int e = 0; e < 8; ++e) x[e] = instead;
                        }
                        // two pieces of 8 values: eight lanes, one row (two at H = 64), all banks
                        constexpr uint32_t kPieces = C::kSwz / 16;
                        if constexpr (H == 128) {
                            const uint32_t at = to + prompt_swizzled(r, j16, C::kSwz);
                            if (FA_CACHE_OK(p.c.status, kDbgTile, tile_ok(at, to, 1) && tile_ok(at + C::kBoxBytes, to, 1) && tile_ok(to, ring, NS))) {
                                st_shared_v4(at, x[0], x[1], x[2], x[3]);
                                st_shared_v4(at + C::kBoxBytes, x[4], x[5], x[6], x[7]);
                            }
                        } else {
                            static_assert(H == 128 || H == C::kBoxCols, "one box");
                            const uint32_t lower = to + prompt_swizzled(r, (2 * j16) % kPieces, C::kSwz), upper = to + prompt_swizzled(r, (2 * j16 + 1) % kPieces, C::kSwz);
                            if (FA_CACHE_OK(p.c.status, kDbgTile, tile_ok(lower, to, 1) && tile_ok(upper, to, 1) && tile_ok(to, ring, NS))) {
                                st_shared_v4(lower, x[0], x[1], x[2], x[3]);
                                st_shared_v4(upper, x[4], x[5], x[6], x[7]);
                            }
                        }
                        // what comes next takes the registers' place
                        load(c, is_v == 0);   // (behind the last step: the first page's, not used)
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(bar(C::FULL + n % NS));
                        if (is_v == 0 && warp == 8) mbar_arrive(bar(C::SCALE + g % NS));
                    }
                }
            }
            item_done(nth);
        }
    } else {
        // ---------------------------------------------------------------- issue: warp 12 Q K^T, warp 14 P V
        setmaxnreg_dec<C::kIssueRegs>();
        if (warp == 12 || warp == 14) {
            const bool leader = elect_one();
            bool ok = true;   // once a wait has given up nothing more is issued
            auto wait = [&](int b, uint32_t parity) { ok &= mbar_wait(bar(b), parity, ctl, kCacheTimeout | static_cast<uint32_t>(b)); };
            uint32_t g = 0, k = 0, done[2] = {0, 0};   // steps, items, steps of either tile
            for (uint32_t nth = 0;; ++nth) {
                if (!item_wait(nth)) break;
                const PromptItem& it = items[nth % kPromptItems];
                if (it.there == 0) break;
                const uint32_t steps = it.steps, tile_steps[2] = {it.tile_steps[0], it.tile_steps[1]};
                item_done(nth);   // (everything about it is in registers)
                if (steps == 0) continue;
#pragma unroll 1
                for (uint32_t j = 0; j < steps; ++j, ++g) {
                    if (warp == 12) {
                        if (j == 0) wait(C::QFULL + k % C::kQBuffers, (k / C::kQBuffers) & 1u);
                        wait(C::FULL + (2 * g) % NS, (2 * g / NS) & 1u);
#pragma unroll
                        for (uint32_t i = 0; i < 2; ++i) {
                            if (j >= tile_steps[i]) continue;
                            // a score tile's next use needs the reading of the one before (with one tile for both: whosever that was)
                            const uint32_t uses = C::kSharedS ? done[0] + done[1] : done[i];
                            if (uses > 0) wait(C::SFREE0 + (C::kSharedS ? 0 : i), (uses - 1u) & 1u);
                            ++done[i];
                            tc_fence_after();
                            if (leader && ok) {
                                prompt_issue_qk<H>(tmem + (i ? C::kColS1 : C::kColS0), q_addr(k, i), slot_addr(2 * g));
                                tc_commit(bar(C::S0 + i));
                            }
                        }
                        if (leader && ok) {
                            tc_commit(bar(C::EMPTY + (2 * g) % NS));
                            if (j + 1 == steps) tc_commit(bar(C::QEMPTY + k % C::kQBuffers));
                        }
                    } else {
                        wait(C::FULL + (2 * g + 1) % NS, ((2 * g + 1) / NS) & 1u);
#pragma unroll
                        for (uint32_t i = 0; i < 2; ++i) {
                            if (j >= tile_steps[i]) continue;
                            wait(C::P0 + i, done[i] & 1u);
                            ++done[i];
                            tc_fence_after();
                            if (leader && ok) {
                                prompt_issue_pv<H>(tmem + (i ? C::kColO1 : C::kColO0), tmem + (i ? C::kColP1 : C::kColP0), slot_addr(2 * g + 1), j > 0 ? 1u : 0u);
                                tc_commit(bar(C::PV0 + i));
                            }
                        }
                        if (leader && ok) tc_commit(bar(C::EMPTY + (2 * g + 1) % NS));
                    }
                    __syncwarp();
                }
                ++k;
            }
            // every product issued has to retire before tensor and shared memory are let go of
            const int last = warp == 12 ? C::FINAL : C::FINAL2;
            if (leader) tc_commit(bar(last));
            __syncwarp();
            mbar_wait_certain(bar(last), 0, ctl, kCacheTimeout | static_cast<uint32_t>(last));
        } else if (warp == 13) {
            // ------------------------------------------------------------ items, in rounds of a CTA each, there and back: whoever had the
            // longest of a round has the shortest of the next
            uint32_t nth = 0, k = 0;
            for (uint32_t round = 0;; ++round) {
                const uint32_t index = round * gridDim.x + ((round & 1u) ? gridDim.x - 1u - blockIdx.x : blockIdx.x);
                const bool end = round * gridDim.x >= p.items;
                if (!end && index >= p.items) continue;
                PromptItem it = {};
                if (!end) it = prompt_item(p, index);
                if (!end && lane == 0 && it.step0 == 0 && !cache_length_ok(p.c, p.s, it.b)) cache_report(p.c.status, kCacheBadPosition);
                const bool there = nth < kPromptItems || mbar_wait(bar(C::IFREE + nth % kPromptItems), (nth / kPromptItems - 1u) & 1u, ctl, kCacheTimeout | C::IFREE);
                if (!__all_sync(0xFFFFFFFFu, there)) break;
                if (lane == 0) {
                    items[nth % kPromptItems] = it;
                    mbar_arrive(bar(C::ITEM + nth % kPromptItems));
                }
                __syncwarp();
                ++nth;
                if (end) break;
                if (it.steps == 0) continue;
                const bool wide = prompt_wide(p, it.b, it.head, it.step0 * kPromptTile, min(it.farthest, (it.step0 + it.steps) * kPromptTile), lane);
                if (lane == 0) {
                    s_wide[k & 7u] = wide;
                    mbar_arrive(bar(C::COEF + (k & 7u)));
                }
                __syncwarp();
                ++k;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0) report_expired(ctl);
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Puts an item's parts together: a warp a row.
template <int H>
__global__ void __launch_bounds__(128) fa_cache_prompt_join(const PromptArgs p) {
    grid_dep_wait();
    grid_dep_launch();
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const uint32_t row = static_cast<uint32_t>(at % (2 * kPromptTile)), item = static_cast<uint32_t>(at / (2 * kPromptTile));   // of those that are cut
    if (item >= (p.items - p.whole) / p.parts) return;
    const uint32_t heads = p.s.B * p.c.heads, bh = (p.whole + item) % heads, pair = p.pairs - 1u - (p.whole + item) / heads;
    const uint32_t r = pair * (2 * kPromptTile) + row;
    if (r >= p.s.T * p.group) return;
    auto slot = [&](uint32_t part) { return (static_cast<uint64_t>(item) * p.parts + part) * (2 * kPromptTile) + row; };
    float top = -INFINITY;
    for (uint32_t i = lane; i < p.parts; i += 32) top = fmaxf(top, p.part_ml[slot(i)].x);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    float sum = 0.0f, x[H >= 64 ? H / 32 : 2];
    constexpr uint32_t kWide = H >= 64 ? H / 32 : 2;   // dimensions of a lane
#pragma unroll
    for (uint32_t e = 0; e < kWide; ++e) x[e] = 0.0f;
    for (uint32_t i = 0; i < p.parts; ++i) {
        const float2 ml = p.part_ml[slot(i)];
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;   // a part without keys: its rows were not written
        const float f = ml.x == -INFINITY ? 0.0f : ex2_approx(ml.x - top);
        sum += times_power(ml.y, ml.x - top);
        if (lane * kWide < H)
#pragma unroll
            for (uint32_t e = 0; e < kWide; e += 2) {
                const float2 o = *reinterpret_cast<const float2*>(p.part_o + slot(i) * H + lane * kWide + e);
                x[e] += o.x * f, x[e + 1] += o.y * f;
            }
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t t = r / p.group, h = bh % p.c.heads * p.group + r % p.group;
    uint8_t* const to = p.y + ((static_cast<uint64_t>(bh / p.c.heads) * p.s.T + t) * (p.c.heads * p.group) + h) * (2 * H);
    if (lane * kWide < H)
#pragma unroll
        for (uint32_t e = 0; e < kWide; e += 2) *reinterpret_cast<uint32_t*>(to + 2 * (lane * kWide + e)) = pack_16(x[e] * f, x[e + 1] * f, p.bf16 != 0);
}

}  // namespace fa
