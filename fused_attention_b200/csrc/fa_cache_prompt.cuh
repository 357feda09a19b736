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
//
// Scales.  A step's keys have eight groups of 16 with a scale each for K and V (pages are 16 tokens or more).  As in
// fa_cache_rows.cuh the exponent of a weight is score * (row's factor * key scale) + log2(value scale) - M, one multiply-add
// a pair of scores with factors that change from group to group, and the row sum divides the value scale out again.
// A page whose scale is NaN becomes keys that are NaN and values that are zero, so that only rows that see it are NaN.
//
// Bound by the tensor pipe and the exponentials as fa_fwd_pipelined is (per step and tile 1024 tensor clocks of products at
// H = 128 and 1024 clocks of exponentials); what is added here is shared-memory traffic, 64 KB a step written by the loading
// warps beside the 192 KB that the products read.
#pragma once

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
    uint32_t group, causal, bf16;
    uint32_t pairs;          // items of a sequence and key/value head, without their parts
    uint32_t parts, items;   // items: with their parts
    float scale_log2;        // log2(e) / sqrt(H)
    float* part_o;           // [items, 256, H]
    float2* part_ml;         // [items, 256]
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
    // barriers
    static constexpr int QFULL = 0, QEMPTY = QFULL + kQBuffers, FULL = QEMPTY + kQBuffers, EMPTY = FULL + kSlots, S0 = EMPTY + kSlots, SFREE0 = S0 + 2,
                         P0 = SFREE0 + 2, PV0 = P0 + 2, FINAL = PV0 + 2, FINAL2 = FINAL + 1, COEF = FINAL2 + 1, SCALE = COEF + 4, kBarriers = SCALE + kSlots;
};

// Scales of a step's groups as the softmax takes them.
struct __align__(16) PromptScales {
    float ks[kPromptGroups], vlog[kPromptGroups], vinv[kPromptGroups];
};

__device__ __forceinline__ uint32_t prompt_swizzled(uint32_t row, uint32_t piece, uint32_t span) {
    return row * span + ((piece ^ ((row * span >> 7) & (span / 16u - 1u))) << 4);
}

// What an item is, the same for every role.
struct PromptItem {
    uint32_t b, head, row0, part;   // row0: first row, of T * group
    uint32_t held, count, n_rows;
    uint32_t farthest;              // keys [0, farthest) are seen by some row
    uint32_t step0, steps;          // this part's
};
template <int H>
__device__ __forceinline__ uint32_t prompt_index(const PromptArgs& p, uint32_t round) {
    const uint32_t c = (round & 1u) ? gridDim.x - 1u - blockIdx.x : blockIdx.x;   // there and back: whoever had the longest of a round has the shortest of the next
    return round * gridDim.x + c;
}
__device__ __forceinline__ PromptItem prompt_item(const PromptArgs& p, uint32_t index) {
    PromptItem it;
    const uint32_t heads = p.s.B * p.c.heads;
    it.part = index % p.parts;
    index /= p.parts;
    const uint32_t bh = index % heads, pair = p.pairs - 1u - index / heads;
    it.b = bh / p.c.heads;
    it.head = bh % p.c.heads;
    it.row0 = pair * (2 * kPromptTile);
    it.n_rows = min(2u * kPromptTile, p.s.T * p.group - it.row0);
    it.held = cache_length(p.c, p.s, it.b);
    it.count = cache_count(p.s, it.b);
    const uint32_t t_first = it.row0 / p.group, t_end = min(it.count, (it.row0 + it.n_rows - 1u) / p.group + 1u);   // tokens [t_first, t_end)
    it.farthest = 0;
    if (t_first < t_end) it.farthest = p.causal ? (it.held + t_end > it.count ? min(it.held, it.held + t_end - it.count) : 0u) : it.held;
    const uint32_t all = (it.farthest + kPromptTile - 1u) / kPromptTile;
    it.step0 = all * it.part / p.parts;
    it.steps = all * (it.part + 1u) / p.parts - it.step0;
    return it;
}
// Keys that row r of the item sees.
__device__ __forceinline__ uint32_t prompt_limit(const PromptArgs& p, const PromptItem& it, uint32_t r) {
    const uint32_t t = (it.row0 + r) / p.group;
    if (r >= it.n_rows || t >= it.count) return 0;
    if (!p.causal) return it.held;
    return it.held + t >= it.count ? min(it.held, it.held + t - it.count + 1u) : 0u;
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

// Weights of the groups [kG0, kG1) of a row, packed as fp16 pairs (8 words a group); adds the groups' sums to `raw`, and to `l`
// with the value scale divided out.  The exponent is one multiply-add, score * cu + (vlog - ref): `ref` is a whole number, so that
// with scales that are powers of two the bracket is exact.  kAnySize: of a reference that is too large for that (2^22 and more,
// where a score's product is no longer known to a fraction) it is taken off the rounded exponent.
constexpr float kPromptLargeRef = 4194304.0f;
template <int kG0, int kG1, bool kAnySize = false>
__device__ __forceinline__ void prompt_weights(const float (&s)[kPromptTile], const PromptScales& sc, float coef, float ref, uint32_t* pk, float& raw, float& l) {
#pragma unroll
    for (int u = kG0; u < kG1; ++u) {
        // (at least 1e-37: a masked score, -inf, must stay that)
        const bool large = kAnySize && fabsf(ref) > kPromptLargeRef;
        const float cu = fmaxf(coef * sc.ks[u], 1e-37f), add = large ? sc.vlog[u] : sc.vlog[u] - ref, behind = large ? -ref : 0.0f;
        const uint64_t c2 = pack_f32x2(cu, cu), a2 = pack_f32x2(add, add);
        uint64_t sum_a = 0, sum_b = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float x0, x1;
            unpack_f32x2(fma_f32x2(pack_f32x2(s[u * 16 + 2 * e], s[u * 16 + 2 * e + 1]), c2, a2), x0, x1);
            if (kAnySize) x0 += behind, x1 += behind;
            const float w0 = ex2_approx(x0), w1 = ex2_approx(x1);
            if (e & 1) sum_b = add_f32x2(sum_b, pack_f32x2(w0, w1));
            else sum_a = add_f32x2(sum_a, pack_f32x2(w0, w1));
            pk[(u - kG0) * 8 + e] = pack_half2(w0, w1);
        }
        float lo, hi;
        unpack_f32x2(add_f32x2(sum_a, sum_b), lo, hi);
        raw += lo + hi;
        l = fmaf(lo + hi, sc.vinv[u], l);
    }
}
// Largest exponent of a row, rounded up to a whole number.
__device__ __forceinline__ float prompt_top(const float (&s)[kPromptTile], const PromptScales& sc, float coef) {
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kPromptGroups; ++u) {
        float a = max3(s[u * 16], s[u * 16 + 1], s[u * 16 + 2]), b = max3(s[u * 16 + 3], s[u * 16 + 4], s[u * 16 + 5]);
#pragma unroll
        for (int e = 6; e < 14; e += 4) {
            a = max3(a, s[u * 16 + e], s[u * 16 + e + 1]);
            b = max3(b, s[u * 16 + e + 2], s[u * 16 + e + 3]);
        }
        a = max3(a, s[u * 16 + 14], s[u * 16 + 15]);
        top = fmaxf(top, fmaf(fmaxf(a, b), fmaxf(coef * sc.ks[u], 1e-37f), sc.vlog[u]));
    }
    return ceilf(top);
}

template <int H>
__global__ void __launch_bounds__(kPromptThreads, 1) fa_cache_prompt(const PromptArgs p) {
    using C = PromptCfg<H>;
    constexpr uint32_t NS = C::kSlots, kGroups = kPromptGroups;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[C::kBarriers];
    __shared__ PromptScales scales[NS];           // of step g in entry g % NS (free when the V tile of that step is)
    // Rows' factors, by item.  Four: item k + 4's are written once the last Q K^T of item k + 2 (or a later one) has retired, which
    // needs the scores of item k + 1 read; whoever read those has long taken its factor of item k.
    __shared__ float s_coef[4][2 * kPromptTile];
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
            const bool by_loaders = (i >= C::QFULL && i < C::QEMPTY) || (i >= C::FULL && i < C::EMPTY) || (i >= C::COEF && i < C::SCALE);
            const bool by_softmax = i >= C::SFREE0 && i < C::PV0;
            mbar_init(bar(i), by_loaders || by_softmax ? 4u : 1u);
        }
        abort_flag = 0;
        fence_mbar_init();
    }
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

    if (warp < 8) {
        // ---------------------------------------------------------------- softmax of tile i
        setmaxnreg_inc<184>();
        const uint32_t i = warp >> 2, r = tid & 127u, lane_off = ((warp & 3u) * 32u) << 16;
        const uint32_t tS = tmem + lane_off + (i ? C::kColS1 : C::kColS0), tP = tmem + lane_off + (i ? C::kColP1 : C::kColP0),
                       tO = tmem + lane_off + (i ? C::kColO1 : C::kColO0);
        uint32_t g = 0, k = 0;
        for (uint32_t round = 0;; ++round) {
            const uint32_t index = prompt_index<H>(p, round);
            if (round * gridDim.x >= p.items) break;
            if (index >= p.items) continue;
            const PromptItem it = prompt_item(p, index);
            const uint32_t row = i * kPromptTile + r, limit = prompt_limit(p, it, row);
            // rows that see nothing count as seeing everything: nobody waits for them, and they are written as zeros
            const uint32_t masked_from = limit == 0 ? kNoToken : limit;
            float m = -INFINITY, l = 0.0f, coef = 0.0f;
            if (it.steps > 0) {
                mbar_wait(bar(C::COEF + (k & 3u)), (k >> 2) & 1u, ctl, kCacheTimeout | C::COEF);
                coef = s_coef[k & 3u][row];
            }
#pragma unroll 1
            for (uint32_t j = 0; j < it.steps; ++j, ++g) {
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
                const PromptScales& sc = scales[g % NS];
                mbar_wait(bar(C::SCALE + g % NS), (g / NS) & 1u, ctl, kCacheTimeout | C::SCALE);
                const uint32_t key0 = (it.step0 + j) * kPromptTile;
                if (__any_sync(0xFFFFFFFFu, key0 + kPromptTile > masked_from)) {
                    const int valid = static_cast<int>(masked_from) - static_cast<int>(key0);
#pragma unroll
                    for (int e = 0; e < kPromptTile; ++e)
                        if (e >= valid) s[e] = -INFINITY;
                }
                if (j == 0) m = prompt_top(s, sc, coef);
                // the first quarter's weights are kept in registers: the last step's P V may still be reading P
                uint32_t held[16];
                float raw = 0.0f, sum = 0.0f;
                const float ref = m == -INFINITY ? 0.0f : m;
                prompt_weights<0, 2>(s, sc, coef, ref, held, raw, sum);
                if (g > 0) {
                    mbar_wait(bar(C::PV0 + i), (g - 1u) & 1u, ctl, kCacheTimeout | (C::PV0 + i));
                    tc_fence_after();
                }
                __syncwarp();
                tmem_st16(tP, held);
#pragma unroll
                for (int c = 1; c < 4; ++c) {
                    uint32_t pk[16];
                    if (c == 1) prompt_weights<2, 4>(s, sc, coef, ref, pk, raw, sum);
                    if (c == 2) prompt_weights<4, 6>(s, sc, coef, ref, pk, raw, sum);
                    if (c == 3) prompt_weights<6, 8>(s, sc, coef, ref, pk, raw, sum);
                    tmem_st16(tP + c * 16, pk);
                }
                // M has to move when a weight exceeds 2^8, which none does while the row's sum stays below; a row that has seen
                // nothing so far takes the maximum of what it sees first
                bool moved = false;
                float top = m;
                const bool large = fabsf(m) > kPromptLargeRef && m != -INFINITY;
                if (__any_sync(0xFFFFFFFFu, !(raw <= 255.0f) || (m == -INFINITY && j > 0) || large)) {
                    top = prompt_top(s, sc, coef);
                    moved = top > m + kRowsSlack;
                }
                if (__any_sync(0xFFFFFFFFu, moved || large)) {
                    const float m_new = moved ? top : m, alpha = moved ? ex2_approx(m - m_new) : 1.0f;
                    m = m_new;
                    const float ref2 = m == -INFINITY ? 0.0f : m;
                    raw = sum = 0.0f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t pk[16];
                        if (c == 0) prompt_weights<0, 2, true>(s, sc, coef, ref2, pk, raw, sum);
                        if (c == 1) prompt_weights<2, 4, true>(s, sc, coef, ref2, pk, raw, sum);
                        if (c == 2) prompt_weights<4, 6, true>(s, sc, coef, ref2, pk, raw, sum);
                        if (c == 3) prompt_weights<6, 8, true>(s, sc, coef, ref2, pk, raw, sum);
                        tmem_st16(tP + c * 16, pk);
                    }
                    l = l * alpha + sum;
                    if (j > 0) {   // (an item's first P V overwrites O)
                        constexpr int kCols = H < 32 ? 16 : 32;
#pragma unroll
                        for (int c = 0; c < H; c += kCols) {
                            float o[kCols];
                            tmem_ld<kCols>(tO + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < kCols; ++e) o[e] *= alpha;
                            if constexpr (kCols == 32) {
                                tmem_st32(tO + c, o);
                            } else {
                                uint32_t w[16];
#pragma unroll
                                for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e]);
                                tmem_st16(tO + c, w);
                            }
                        }
                    }
                } else {
                    l += sum;
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(C::P0 + i));
            }
            // ---- the item's end: this row of O.  (The next item's first P V waits for P from these warps.)
            if (it.steps > 0) {
                ++k;
                mbar_wait(bar(C::PV0 + i), (g - 1u) & 1u, ctl, kCacheTimeout | (C::PV0 + i));
                tc_fence_after();
                __syncwarp();
            }
            const bool there = row < it.n_rows;
            if (p.parts == 1) {
                const float f = limit == 0 || l == 0.0f ? 0.0f : 1.0f / l;
                const uint32_t t = (it.row0 + row) / p.group, h = it.head * p.group + (it.row0 + row) % p.group;
                uint8_t* const to = p.y + ((static_cast<uint64_t>(it.b) * p.s.T + t) * (p.c.heads * p.group) + h) * (2 * H);
                constexpr int kCols = H < 32 ? 16 : 32;
#pragma unroll 1
                for (int c = 0; c < H; c += kCols) {
                    float o[kCols];
                    if (it.steps > 0) {
                        tmem_ld<kCols>(tO + c, o);
                        tmem_wait_ld();
                    }
                    if (there) {
#pragma unroll
                        for (int e = 0; e < kCols; e += 8) {
                            uint4 w = make_uint4(0, 0, 0, 0);
                            if (limit != 0)
                                w = make_uint4(pack_16(o[e] * f, o[e + 1] * f, p.bf16), pack_16(o[e + 2] * f, o[e + 3] * f, p.bf16),
                                               pack_16(o[e + 4] * f, o[e + 5] * f, p.bf16), pack_16(o[e + 6] * f, o[e + 7] * f, p.bf16));
                            *reinterpret_cast<uint4*>(to + 2 * (c + e)) = w;
                        }
                    }
                }
            } else {
                const uint64_t at = static_cast<uint64_t>(index) * (2 * kPromptTile) + row;
                constexpr int kCols = H < 32 ? 16 : 32;
                if (there) p.part_ml[at] = make_float2(limit == 0 || it.steps == 0 ? -INFINITY : m, limit == 0 || it.steps == 0 ? 0.0f : l);
                if (it.steps > 0)
#pragma unroll 1
                    for (int c = 0; c < H; c += kCols) {
                        float o[kCols];
                        tmem_ld<kCols>(tO + c, o);
                        tmem_wait_ld();
                        if (there) {
#pragma unroll
                            for (int e = 0; e < kCols; e += 4) *reinterpret_cast<float4*>(p.part_o + at * H + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                        }
                    }
            }
            tc_fence_before();
        }
    } else if (warp < 12) {
        // ---------------------------------------------------------------- loading
        setmaxnreg_dec<80>();
        constexpr uint32_t kLanes = H / 16;                // that share a row of codes, 16 each
        constexpr uint32_t kRowsPass = 128 / kLanes;
        constexpr uint32_t kPasses = kPromptTile / kRowsPass;
        const uint32_t lt = tid - 256u, j16 = lt % kLanes, r_in = lt / kLanes;
        uint32_t n = 0, k = 0, g = 0;   // ring items, items, steps so far
        for (uint32_t round = 0;; ++round) {
            const uint32_t index = prompt_index<H>(p, round);
            if (round * gridDim.x >= p.items) break;
            if (index >= p.items) continue;
            const PromptItem it = prompt_item(p, index);
            if (it.steps == 0) {
                if (lt == 0 && !cache_length_ok(p.c, p.s, it.b)) cache_report(p.c.status, kCacheBadPosition);
                continue;
            }
            if (lt == 0 && it.part == 0 && !cache_length_ok(p.c, p.s, it.b)) cache_report(p.c.status, kCacheBadPosition);
            const int32_t* const table = p.s.table + it.b * p.s.table_stride;
            // ---- a step's pages: lane l (of every warp) has group l's.  The table entry is asked for a step ahead, the scales half
            // a step: nothing may depend at once on what has just been asked for.
            int32_t page = -1, entry = -1;
            bool wanted = false;
            float ks = 1.0f, vs = 1.0f;
            auto ask = [&](uint32_t step) {
                const uint32_t at = (it.step0 + step) * kPromptTile + (lane & 7u) * 16u;
                wanted = step < it.steps && at < it.farthest;
                entry = wanted ? table[at >> p.c.page_shift] : -1;
            };
            auto look_up = [&] {
                page = entry, ks = 1.0f, vs = 1.0f;
                if (static_cast<uint32_t>(page) >= p.c.n_pages) {
                    if (wanted && lane < 8 && warp == 8) cache_report(p.c.status, kCacheBadPage);
                    page = -1;
                } else {
                    const uint64_t s_at = static_cast<uint64_t>(page) * p.c.heads + it.head;
                    ks = p.c.k_scale[s_at], vs = p.c.v_scale[s_at];
                }
            };
            uint4 codes[kPasses];
            // pass c of a step's keys (values): this thread's 16 codes; zeros where no row sees the token
            auto load = [&](uint32_t c, uint32_t step, bool is_v) {
                const uint32_t r = c * kRowsPass + r_in, at = (it.step0 + step) * kPromptTile + r;
                const int32_t pg = __shfl_sync(0xFFFFFFFFu, page, r >> 4);
                uint4 w = make_uint4(0, 0, 0, 0);
                if (pg >= 0 && at < it.farthest) {
                    const int64_t in_page = at & (p.c.page - 1);
                    w = *reinterpret_cast<const uint4*>(is_v ? p.c.v + pg * p.c.v_page + it.head * p.c.v_head + in_page * p.c.v_token + 16 * j16
                                                             : p.c.k + pg * p.c.k_page + it.head * p.c.k_head + in_page * p.c.k_token + 16 * j16);
                }
                codes[c] = w;
            };
            ask(0);
            look_up();
#pragma unroll
            for (uint32_t c = 0; c < kPasses; ++c) load(c, 0, false);

            // ---- queries
            if (k >= C::kQBuffers) mbar_wait(bar(C::QEMPTY + k % C::kQBuffers), (k / C::kQBuffers - 1u) & 1u, ctl, kCacheTimeout | C::QEMPTY);
            constexpr uint32_t kQLanes = H / 8, kQRows = 128 / kQLanes;
            const uint32_t piece = lt % kQLanes;
#pragma unroll 4
            for (uint32_t r = lt / kQLanes; r < 2 * kPromptTile; r += kQRows) {
                const uint32_t t = (it.row0 + r) / p.group, h = it.head * p.group + (it.row0 + r) % p.group;
                uint4 w = make_uint4(0, 0, 0, 0);
                if (r < it.n_rows && t < it.count) w = *reinterpret_cast<const uint4*>(p.q + it.b * p.q_b + t * p.q_t + static_cast<int64_t>(h) * (2 * H) + 16 * piece);
                float coef = p.scale_log2;
                if (p.bf16) {   // to the range of fp16, by a power of two a row
                    uint32_t x[4] = {w.x, w.y, w.z, w.w};
                    float most = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = unpack_16(x[e], true);
                        most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
#pragma unroll
                    for (uint32_t d = kQLanes / 2; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
                    const uint32_t e8 = max(__float_as_uint(most) >> 23, 40u);   // biased: 2^(e8 - 127) <= most, unless that is tiny
                    float f = 1.0f;
                    if (e8 < 255) coef *= __uint_as_float((e8 - 7) << 23), f = __uint_as_float((261 - e8) << 23);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 y = unpack_16(x[e], true);
                        x[e] = pack_half2(y.x * f, y.y * f);
                    }
                    w = make_uint4(x[0], x[1], x[2], x[3]);
                }
                constexpr uint32_t kPieces = C::kSwz / 16;   // of a box's row
                st_shared_v4(q_addr(k, r >> 7) + (piece / kPieces) * C::kBoxBytes + prompt_swizzled(r & 127u, piece % kPieces, C::kSwz), w.x, w.y, w.z, w.w);
                if (piece == 0) s_coef[k & 3u][r] = coef;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar(C::QFULL + k % C::kQBuffers));
                mbar_arrive(bar(C::COEF + (k & 3u)));
            }
            ++k;

            // ---- keys and values, K and V of a step in turn
#pragma unroll 1
            for (uint32_t step = 0; step < it.steps; ++step, ++g) {
                const uint32_t poisoned = __ballot_sync(0xFFFFFFFFu, ks != ks || vs != vs) & 0xFFu;   // groups
                const bool none = page < 0;
                ask(step + 1);
#pragma unroll 1
                for (uint32_t is_v = 0; is_v < 2; ++is_v, ++n) {
                    if (n >= NS) mbar_wait(bar(C::EMPTY + n % NS), (n / NS - 1u) & 1u, ctl, kCacheTimeout | (C::EMPTY + n % NS));
                    if (is_v == 0 && lane < kGroups && warp == 8) {   // (the V tile of the step that had this entry has been let go of)
                        PromptScales& sc = scales[g % NS];
                        const bool bad = ks != ks || vs != vs;
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
                        if (poisoned >> (r >> 4) & 1u) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) x[e] = is_v ? 0u : 0x7E007E00u;
                        }
                        // two pieces of 8 values; the lanes of the second box write theirs in the other order (their banks are those of the first)
                        constexpr uint32_t kPieces = C::kSwz / 16;
                        const uint32_t first = 2 * j16, swap = H == 128 ? j16 >> 2 : 0u;
                        const uint32_t box = to + (first / kPieces) * C::kBoxBytes;
                        const uint32_t a0 = box + prompt_swizzled(r, (first + swap) % kPieces, C::kSwz), a1 = box + prompt_swizzled(r, (first + 1 - swap) % kPieces, C::kSwz);
                        if (swap) {
                            st_shared_v4(a0, x[4], x[5], x[6], x[7]);
                            st_shared_v4(a1, x[0], x[1], x[2], x[3]);
                        } else {
                            st_shared_v4(a0, x[0], x[1], x[2], x[3]);
                            st_shared_v4(a1, x[4], x[5], x[6], x[7]);
                        }
                        // what comes next takes the registers' place
                        if (is_v == 0) load(c, step, true);
                        else if (step + 1 < it.steps) load(c, step + 1, false);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(bar(C::FULL + n % NS));
                        if (is_v == 0 && warp == 8) mbar_arrive(bar(C::SCALE + g % NS));
                    }
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- issue: warp 12 Q K^T, warp 14 P V
        setmaxnreg_dec<64>();
        if (warp == 12 || warp == 14) {
            const bool leader = elect_one();
            bool ok = true;   // once a wait has given up nothing more is issued
            auto wait = [&](int b, uint32_t parity) { ok &= mbar_wait(bar(b), parity, ctl, kCacheTimeout | static_cast<uint32_t>(b)); };
            uint32_t g = 0, k = 0;
            for (uint32_t round = 0;; ++round) {
                const uint32_t index = prompt_index<H>(p, round);
                if (round * gridDim.x >= p.items) break;
                if (index >= p.items) continue;
                const uint32_t steps = prompt_item(p, index).steps;
                if (steps == 0) continue;
#pragma unroll 1
                for (uint32_t j = 0; j < steps; ++j, ++g) {
                    if (warp == 12) {
                        if (j == 0) wait(C::QFULL + k % C::kQBuffers, (k / C::kQBuffers) & 1u);
                        wait(C::FULL + (2 * g) % NS, (2 * g / NS) & 1u);
#pragma unroll
                        for (uint32_t i = 0; i < 2; ++i) {
                            // one score tile: its use 2 g + i needs the reading of the one before; two: the reading of step g - 1's
                            if (C::kSharedS ? g + i > 0 : g > 0) wait(C::SFREE0 + (C::kSharedS ? 0 : i), C::kSharedS ? 1u - i : (g - 1u) & 1u);
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
                            wait(C::P0 + i, g & 1u);
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
    const uint32_t row = static_cast<uint32_t>(at % (2 * kPromptTile)), whole = static_cast<uint32_t>(at / (2 * kPromptTile));
    const uint32_t heads = p.s.B * p.c.heads, bh = whole % heads, pair = p.pairs - 1u - whole / heads;
    if (whole >= p.items / p.parts) return;
    const uint32_t r = pair * (2 * kPromptTile) + row;
    if (r >= p.s.T * p.group) return;
    auto slot = [&](uint32_t part) { return (static_cast<uint64_t>(whole) * p.parts + part) * (2 * kPromptTile) + row; };
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
        sum += ml.y * f;
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
