// Attention with keys and values multiplied out of latent vectors, the expanded form: for prompts.
//
//   s = scale * (q_nope . k_h + q_rope . r),  y = softmax(s) v_h        k_h, v_h: of the head; r: the token's rotary key, for all heads
//
// A CTA has 256 query rows (two tiles of 128) of one sequence and head, and goes over the keys that the last of them sees in steps of 128,
// as fa_cache_prompt.cuh does: scores in tensor memory, a softmax thread a row, P (16 bits) into tensor memory, Y in tensor memory.  The
// score's contraction has NOPE + rope dimensions, the last chunk of 64 of which is the rotary part, fetched from the tensor that all heads
// share.  Operands come by TMA in chunks of 128 rows by 64 dimensions into two rings, of keys and of values.  384 threads:
//
//   warps 0-3, 4-7   softmax of query tile 0 / 1, a thread a row
//   warp 8           fetches queries and keys
//   warp 9, 10       issue Q K^T, P V
//   warp 11          fetches values, and goes over those of steps that some row sees in part only: keys behind the last that any row sees become
//                    zeros, and so do keys that hold an infinity or a NaN, whose weights become NaN for the rows that see them.  0 * NaN
//                    reaches nobody
//
// Bound by the tensor pipe and the exponentials as fa_fwd_pipelined is: at NOPE = 128 a step of both tiles has 2560 tensor clocks of products and
// 2048 of exponentials, and takes 3450.  (In one ring, values of a step came to stand in the way of keys two steps later: 4030.  With a barrier a
// chunk and not a step it stayed at 4080: every wait that stands behind MMAs and commits costs the issuing warp 280 clocks.)  4096 tokens on 6000
// keys, 20 heads of 128 + 64: 222 to 249 us from box to box, 0.83 to 0.93 PFLOP/s, 50 to 56 % of the products' measured peak; 8 prompts of up to
// 777, 12 heads of 64 + 32, 39 to 43 us.  An item's beginning, end and up to three partly seen steps are what the second has most of, and CTAs that
// find nothing to do because `counts` is lower.  Persistent CTAs, items dealt out there and back, were slower, 236 and 54: items' lengths differ,
// and the hardware deals out better.
// At NOPE = 128 both tiles' scores take turns on one 128-column buffer (tensor memory: 128 + 2 * 64 of P + 2 * 128 of Y), which the other
// tile's P V covers; at 64 each has its own.  Items with the most keys go first.
#pragma once

#include <cuda.h>

#include "fa_latent_rows.cuh"

namespace fa {

constexpr int kExpandThreads = 384;
constexpr uint32_t kExpandTile = 128;
constexpr uint32_t kExpandChunk = kExpandTile * 128;   // bytes of 128 rows by 64 dimensions

// First code and number of reports of what these kernels found wrong, as a cache's status block.
__device__ uint32_t g_latent_status[4];

struct ExpandArgs {
    const int32_t* lengths;   // [B] or null: S each
    const int32_t* counts;    // [B] or null: T each
    uint8_t* y;               // [B, T, heads, NOPE] contiguous
    uint32_t B, T, S, heads, pairs, rope, causal;
    float scale_log2;
};

template <int NOPE>
struct ExpandCfg {
    static constexpr int kNope = NOPE / 64, kKey = kNope + 1;             // chunks of keys' own part, of keys
    // Steps in the rings: what shared memory has room for, keys first (they come to be used in one go).  A barrier a step and not a chunk: a
    // wait that stands behind MMAs and commits costs the issuing warps 280 clocks.
    static constexpr int kKSlots = kNope == 2 ? 2 : 3, kVSlots = kNope == 2 ? 1 : 4;
    static constexpr bool kSharedS = NOPE == 128;
    static constexpr uint32_t kColS0 = 0, kColS1 = kSharedS ? 0 : 128, kColP0 = kSharedS ? 128 : 256, kColP1 = kColP0 + 64, kColO0 = kColP1 + 64,
                              kColO1 = kColO0 + NOPE;
    static_assert(kColO1 + NOPE <= 512, "tensor memory");
    static constexpr uint32_t kOffK = 2 * kKey * kExpandChunk, kOffV = kOffK + kKSlots * kKey * kExpandChunk, kTiles = kOffV + kVSlots * kNope * kExpandChunk;
    static constexpr int kSmemBytes = kTiles + 1024;
    static constexpr int QFULL = 0, KFULL = 1, KEMPTY = KFULL + kKSlots, VFULL = KEMPTY + kKSlots, VEMPTY = VFULL + kVSlots, S = VEMPTY + kVSlots, SFREE = S + 2, P = SFREE + 2, PV = P + 2, BAD = PV + 2, FINAL = BAD + 4,
                         kBarriers = FINAL + 2;
    // 168 registers a thread at launch, so twice the softmax warps' and the others' are 504 at most
    static constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
    static_assert(2 * kSoftmaxRegs + kOtherRegs <= 504, "registers of the three warpgroups");
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, uint32_t bar, int32_t x, int32_t y, int32_t z, int32_t w) {
#ifdef FA_DEBUG
    if (!dbg_ok(dst >= g_dbg.smem_lo && dst + kExpandChunk <= g_dbg.smem_hi, kDbgSmemRange) || !dbg_ok((dst & 1023u) == 0 && (x & 7) == 0, kDbgSmemAlign)) return;
#endif
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}
__device__ __forceinline__ float largest_of_32(const float* x) {
    float a = max3(x[0], x[1], x[2]), b = max3(x[3], x[4], x[5]);
#pragma unroll
    for (int e = 6; e < 30; e += 4) {
        a = max3(a, x[e], x[e + 1]);
        b = max3(b, x[e + 2], x[e + 3]);
    }
    return max3(a, b, fmaxf(x[30], x[31]));
}

template <int NOPE, bool kBf16>
__global__ void __launch_bounds__(kExpandThreads, 1)
    fa_latent_prompt(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_qr, const __grid_constant__ CUtensorMap map_kv,
                     const __grid_constant__ CUtensorMap map_r, const ExpandArgs p) {
    using C = ExpandCfg<NOPE>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[C::kBarriers];
    __shared__ uint32_t s_bad[4][4];   // of the n-th partly seen step in entry n % 4: keys that hold no finite numbers
    __shared__ uint32_t tmem_slot, abort_flag;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    auto k_addr = [&](uint32_t j, uint32_t c) { return base + C::kOffK + ((j % C::kKSlots) * C::kKey + c) * kExpandChunk; };
    auto v_addr = [&](uint32_t j, uint32_t c) { return base + C::kOffV + ((j % C::kVSlots) * C::kNope + c) * kExpandChunk; };
    const WaitCtl ctl{g_latent_status, &abort_flag, kWaitCapCycles, nullptr, 0};
    constexpr bool bf16 = kBf16;

    if (tid == 0) {
        for (int i = 0; i < C::kBarriers; ++i) mbar_init(bar(i), i >= C::SFREE && i < C::PV ? 4u : 1u);
        abort_flag = 0;
        fence_mbar_init();
        prefetch_tensormap(&map_q), prefetch_tensormap(&map_qr), prefetch_tensormap(&map_kv), prefetch_tensormap(&map_r);
    }
#ifdef FA_DEBUG
    if (tid == 0) g_dbg.smem_lo = base, g_dbg.smem_hi = base + C::kTiles, g_dbg.tmem_base = 0, g_dbg.tmem_cols = 512, g_dbg.ctl = ctl;
    FA_CACHE_POISON(base, C::kTiles);
    fence_proxy_async_smem();
#endif
    if (warp == 9) {
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

    // ---- the item
    const uint32_t heads = p.B * p.heads, bh = blockIdx.x % heads, b = bh / p.heads, head = bh % p.heads;
    const uint32_t row0 = (p.pairs - 1u - blockIdx.x / heads) * (2 * kExpandTile);
    const int32_t length = p.lengths ? p.lengths[b] : static_cast<int32_t>(p.S), counted = p.counts ? p.counts[b] : static_cast<int32_t>(p.T);
    const uint32_t held = length < 0 ? 0u : min(static_cast<uint32_t>(length), p.S), count = counted < 0 ? 0u : min(static_cast<uint32_t>(counted), p.T);
    if (tid == 0 && row0 == 0 && head == 0 && (length != static_cast<int32_t>(held) || counted != static_cast<int32_t>(count))) cache_report(g_latent_status, kCacheBadPosition);
    // keys [0, ...) that row t sees
    auto limit_of = [&](uint32_t t) { return t >= count ? 0u : !p.causal ? held : held + t >= count ? min(held, held + t - count + 1u) : 0u; };
    // ... that some row of tile i sees; steps that it takes part in
    uint32_t far[2], steps[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t from = row0 + i * kExpandTile;
        far[i] = from < count ? limit_of(min(count, from + kExpandTile) - 1u) : 0u;
        steps[i] = (far[i] + kExpandTile - 1u) / kExpandTile;
    }
    const uint32_t farthest = max(far[0], far[1]), all = max(steps[0], steps[1]);
    // Steps from `partly` on are seen in part by some row.  (Rows that see nothing do not matter; the first that sees something sees least.)
    uint32_t least = farthest;
    if (p.causal && row0 < count) {
        const uint32_t first = held + row0 >= count ? row0 : count - held;   // first row at or behind position 0
        if (first < count) least = min(farthest, limit_of(first));
    }
    const uint32_t partly = least / kExpandTile;

    if (warp < 8) {
        // ---------------------------------------------------------------- softmax of tile i
        setmaxnreg_inc<C::kSoftmaxRegs>();
        const uint32_t i = warp >> 2, lane_off = ((warp & 3u) * 32u) << 16, t = row0 + tid;
        const uint32_t tS = tmem + lane_off + (i ? C::kColS1 : C::kColS0), tP = tmem + lane_off + (i ? C::kColP1 : C::kColP0), tO = tmem + lane_off + (i ? C::kColO1 : C::kColO0);
        const uint32_t limit = limit_of(t), masked_from = limit == 0 ? kSeesAll : limit;   // (a row that sees nothing waits for nobody; it is written as zeros)
        float m = -INFINITY, l = 0.0f;
        const uint32_t mine = steps[i];
#pragma unroll 1
        for (uint32_t j = 0; j < mine; ++j) {
            mbar_wait(bar(C::S + i), j & 1u, ctl, kCacheTimeout | (C::S + i));
            tc_fence_after();
            __syncwarp();
            float s[kExpandTile];
#pragma unroll
            for (uint32_t c = 0; c < kExpandTile; c += 32) tmem_ld32(tS + c, s + c);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::SFREE + (C::kSharedS ? 0 : i)));
            if (j >= partly) {
                const uint32_t n = j - partly;
                mbar_wait(bar(C::BAD + (n & 3u)), (n >> 2) & 1u, ctl, kCacheTimeout | C::BAD);
                const int valid = static_cast<int>(min(min(masked_from, farthest), 0x7FFFFFFFu)) - static_cast<int>(j * kExpandTile);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int left = valid - w * 32;
                    const uint32_t seen = left >= 32 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << left) - 1u;
                    const uint32_t bad = *reinterpret_cast<volatile uint32_t*>(&s_bad[n & 3u][w]);
                    if (bad != 0) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (bad >> e & 1u) s[w * 32 + e] = __int_as_float(0x7FC00000);
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(seen >> e & 1u)) s[w * 32 + e] = -INFINITY;
                }
            }
            const float top = fmaxf(fmaxf(largest_of_32(s), largest_of_32(s + 32)), fmaxf(largest_of_32(s + 64), largest_of_32(s + 96))) * p.scale_log2;
            float alpha = 1.0f;
            if (top > m + kLatentSlack) {
                alpha = ex2_approx(m - top);
                m = top;
                l *= alpha;
            }
            const float ref = m == -INFINITY ? 0.0f : m;
            const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2), ref2 = pack_f32x2(-ref, -ref);
            uint64_t sum_a = 0, sum_b = 0;
            // a quarter of the row at a time; the last step's P V may still be reading P while the first is worked out
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float x0, x1;
                    unpack_f32x2(fma_f32x2(pack_f32x2(s[q * 32 + 2 * e], s[q * 32 + 2 * e + 1]), scale2, ref2), x0, x1);
                    const float w0 = ex2_approx(x0), w1 = ex2_approx(x1);
                    pk[e] = pack_16(w0, w1, bf16);   // as in fa_latent_rows: an MMA takes one type of both operands
                    const float2 y = unpack_16(pk[e], bf16);   // summed as rounded
                    if (e & 1) sum_b = add_f32x2(sum_b, pack_f32x2(y.x, y.y));
                    else sum_a = add_f32x2(sum_a, pack_f32x2(y.x, y.y));
                }
                if (q == 0) {
                    if (j > 0) {
                        mbar_wait(bar(C::PV + i), (j - 1u) & 1u, ctl, kCacheTimeout | (C::PV + i));
                        tc_fence_after();
                    }
                    __syncwarp();
                }
                tmem_st16(tP + 16 * q, pk);
            }
            float lo, hi;
            unpack_f32x2(add_f32x2(sum_a, sum_b), lo, hi);
            l += lo + hi;
            if (j > 0 && __any_sync(0xFFFFFFFFu, alpha != 1.0f)) {
#pragma unroll 1
                for (uint32_t c = 0; c < NOPE; c += 16) {
                    float o[16];
                    uint32_t x[16];
                    tmem_ld16(tO + c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(o[e] * alpha);
                    tmem_st16(tO + c, x);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::P + i));
        }
        // ---- Y
        if (mine > 0) {
            mbar_wait(bar(C::PV + i), (mine - 1u) & 1u, ctl, kCacheTimeout | (C::PV + i));
            tc_fence_after();
            __syncwarp();
        }
        const bool there = t < p.T, zero = limit == 0 || l == 0.0f;
        const float f = zero ? 0.0f : 1.0f / l;
        uint8_t* const to = p.y + ((static_cast<uint64_t>(b) * p.T + t) * p.heads + head) * (2 * NOPE);
#pragma unroll 1
        for (uint32_t c = 0; c < NOPE; c += 32) {
            float o[32];
            if (mine > 0) {
                tmem_ld32(tO + c, o);
                tmem_wait_ld();
            }
            if (there) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (!zero)
                        w = make_uint4(pack_16(o[e] * f, o[e + 1] * f, bf16), pack_16(o[e + 2] * f, o[e + 3] * f, bf16), pack_16(o[e + 4] * f, o[e + 5] * f, bf16),
                                       pack_16(o[e + 6] * f, o[e + 7] * f, bf16));
                    *reinterpret_cast<uint4*>(to + 2 * (c + e)) = w;
                }
            }
        }
        tc_fence_before();
    } else {
        setmaxnreg_dec<C::kOtherRegs>();
        if (warp == 8) {
            // ------------------------------------------------------------ queries, keys: a head's own part, the rotary part
            const bool leader = elect_one();
            bool ok = true;
            uint32_t n = 0;   // steps asked for
            if (all > 0 && leader) {
                mbar_expect_tx(bar(C::QFULL), 2 * C::kKey * kExpandChunk);
                for (uint32_t i = 0; i < 2; ++i)
                    for (uint32_t c = 0; c < C::kKey; ++c)
                        tma_load_4d(base + (i * C::kKey + c) * kExpandChunk, c < C::kNope ? &map_q : &map_qr, bar(C::QFULL), c < C::kNope ? 64 * c : 0, head, row0 + i * kExpandTile, b);
            }
            for (; n < all; ++n) {
                if (n >= C::kKSlots) ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar(C::KEMPTY + n % C::kKSlots), (n / C::kKSlots - 1u) & 1u, ctl, kCacheTimeout | C::KEMPTY));
                if (!ok) break;
                if (leader) {
                    const uint32_t full = bar(C::KFULL + n % C::kKSlots);
                    mbar_expect_tx(full, C::kKey * kExpandChunk);
                    for (uint32_t c = 0; c < C::kNope; ++c) tma_load_4d(k_addr(n, c), &map_kv, full, 64 * c, head, n * kExpandTile, b);
                    tma_load_4d(k_addr(n, C::kNope), &map_r, full, 0, 0, n * kExpandTile, b);
                }
                __syncwarp();
            }
            // What was asked for lands before the CTA ends: the MMAs have waited for it, unless a wait gave up.
            if (*ctl.abort_flag != 0u) {
                if (all > 0) mbar_wait_certain(bar(C::QFULL), 0, ctl, kCacheTimeout | C::QFULL);
                for (uint32_t x = n > C::kKSlots ? n - C::kKSlots : 0; x < n; ++x) mbar_wait_certain(bar(C::KFULL + x % C::kKSlots), (x / C::kKSlots) & 1u, ctl, kCacheTimeout | C::KFULL);
            }
        } else if (warp == 11) {
            // ------------------------------------------------------------ values
            const bool leader = elect_one();
            bool ok = true;
            uint32_t n = 0;   // steps asked for
            for (; n < all; ++n) {
                const uint32_t j = n;
                if (n >= C::kVSlots) ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar(C::VEMPTY + n % C::kVSlots), (n / C::kVSlots - 1u) & 1u, ctl, kCacheTimeout | C::VEMPTY));
                if (!ok) break;
                if (leader) {
                    const uint32_t full = bar(C::VFULL + n % C::kVSlots);
                    mbar_expect_tx(full, C::kNope * kExpandChunk);
                    for (uint32_t c = 0; c < C::kNope; ++c) tma_load_4d(v_addr(n, c), &map_kv, full, NOPE + 64 * c, head, n * kExpandTile, b);
                }
                __syncwarp();
                if (j < partly) continue;
                // a step that some row sees in part
                const uint32_t nth = j - partly, key0 = j * kExpandTile;
                uint32_t bad[4] = {0, 0, 0, 0};   // this lane's keys: lane + 32 k
                mbar_wait(bar(C::VFULL + j % C::kVSlots), (j / C::kVSlots) & 1u, ctl, kCacheTimeout | C::VFULL);
                for (uint32_t c = 0; c < C::kNope; ++c)
                    for (uint32_t k = 0; k < 4; ++k) {
                        const uint32_t key = lane + 32 * k;
                        if (key0 + key < least || key0 + key >= farthest) continue;
                        uint32_t x[8][4];   // the key's row of the chunk, in any order
#pragma unroll
                        for (uint32_t q = 0; q < 8; ++q) ld_shared_v4(v_addr(j, c) + key * 128 + ((q ^ (key & 7u)) << 4), x[q]);
#pragma unroll
                        for (uint32_t q = 0; q < 8; ++q) bad[k] |= not_finite(x[q], bf16);
                    }
                for (uint32_t k = 0; k < 4; ++k) {
                    const uint32_t key = lane + 32 * k;
                    if (bad[k] || key0 + key >= farthest)
                        for (uint32_t c = 0; c < C::kNope; ++c)
                            for (uint32_t q = 0; q < 8; ++q) st_shared_v4(v_addr(j, c) + key * 128 + (q << 4), 0, 0, 0, 0);
                    const uint32_t which = __ballot_sync(0xFFFFFFFFu, bad[k] != 0);
                    if (lane == 0) *reinterpret_cast<volatile uint32_t*>(&s_bad[nth & 3u][k]) = which;
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(C::BAD + (nth & 3u)));
            }
            if (*ctl.abort_flag != 0u)
                for (uint32_t x = n > C::kVSlots ? n - C::kVSlots : 0; x < n; ++x) mbar_wait_certain(bar(C::VFULL + x % C::kVSlots), (x / C::kVSlots) & 1u, ctl, kCacheTimeout | C::VFULL);
        } else {
            // ------------------------------------------------------------ warp 9: Q K^T, warp 10: P V
            const bool leader = elect_one();
            bool ok = true;   // once a wait has given up nothing more is issued
            auto wait = [&](int x, uint32_t parity) { ok &= mbar_wait(bar(x), parity, ctl, kCacheTimeout | static_cast<uint32_t>(x)); };
            const uint32_t idesc_s = idesc_16bit(kExpandTile, kExpandTile, false, false, bf16), idesc_y = idesc_16bit(kExpandTile, 64, false, true, bf16);
            const uint32_t rope_steps = p.rope / 16;
            uint32_t uses = 0;
            if (warp == 9 && all > 0) wait(C::QFULL, 0);
            for (uint32_t j = 0; j < all; ++j) {
                if (warp == 9) wait(C::KFULL + j % C::kKSlots, (j / C::kKSlots) & 1u);
                else wait(C::VFULL + j % C::kVSlots, (j / C::kVSlots) & 1u);
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    if (j >= steps[i]) continue;
                    if (warp == 9) {
                        // the scores' buffer has been read by whoever had it last
                        const uint32_t before = C::kSharedS ? uses : j;
                        if (before > 0) wait(C::SFREE + (C::kSharedS ? 0 : i), (before - 1u) & 1u);
                        ++uses;
                        tc_fence_after();
                        if (leader && ok) {
                            const uint32_t tS = tmem + (i ? C::kColS1 : C::kColS0);
#pragma unroll
                            for (uint32_t c = 0; c < C::kKey; ++c) {
                                const uint64_t dq = make_smem_desc<128>(base + (i * C::kKey + c) * kExpandChunk, 16), dk = make_smem_desc<128>(k_addr(j, c), 16);
                                const uint32_t ks_end = c < C::kNope ? 4u : rope_steps;
                                for (uint32_t ks = 0; ks < ks_end; ++ks) mma_ss(tS, dq + 2 * ks, dk + 2 * ks, idesc_s, c + ks > 0 ? 1u : 0u);
                            }
                            tc_commit(bar(C::S + i));
                        }
                    } else {
                        wait(C::P + i, j & 1u);
                        tc_fence_after();
                        if (leader && ok) {
#pragma unroll
                            for (uint32_t c = 0; c < C::kNope; ++c) {
                                const uint64_t dv = make_smem_desc<128>(v_addr(j, c), 16);
#pragma unroll
                                for (uint32_t ks = 0; ks < kExpandTile / 16; ++ks)
                                    mma_ts(tmem + (i ? C::kColO1 : C::kColO0) + 64 * c, tmem + (i ? C::kColP1 : C::kColP0) + 8 * ks, dv + ks * (2048 >> 4), idesc_y, j + ks > 0 ? 1u : 0u);
                            }
                            tc_commit(bar(C::PV + i));
                        }
                    }
                }
                if (leader && ok) tc_commit(bar(warp == 9 ? C::KEMPTY + j % C::kKSlots : C::VEMPTY + j % C::kVSlots));
                __syncwarp();
            }
            const int last = C::FINAL + (warp == 9 ? 0 : 1);
            if (leader) tc_commit(bar(last));
            __syncwarp();
            mbar_wait_certain(bar(last), 0, ctl, kCacheTimeout | static_cast<uint32_t>(last));
        }
        tc_fence_before();
    }
    __syncthreads();
    if (tid == 0) report_expired(ctl);
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace fa
