// Selecting the pages of a sequence that a query attends to.
//
// Score of a page for a query head: sum over the dimensions of max(q8 lo8, q8 hi8), the largest product that any key within the
// page's bounds can have, where q8 = rint(q * (1 / max |q| * 127)) and lo8, hi8 = rint(code / 4) are whole numbers of 8 bits.  All
// sums are whole numbers below 2^24 and exact in fp32 in any order, so that which pages are taken does not depend on how the
// work is cut, and ties are ties.  The score is multiplied by max |q| * (1 / 127), the maximum over the query heads that share the
// key/value head is taken and multiplied by the page's key scale.  A product with hi8 is the larger one where q8 >= 0, with lo8
// where q8 <= 0, so the sum is two matrix products, of the positive part of q8 with hi8 and of the negative part with lo8:
// mma.sync m16n8k16 on fp16, which holds these numbers exactly.
//
// fa_cache_scores reads 2 H + 4 bytes a page and head: with 32 sequences of 30000 to 131072 tokens 95 MB of DRAM in 37 us, 2.6 TB/s, in a
// launch by itself (the whole call, whose launches overlap, 37 us too).  Neither reading nor the products are near their limits:
// unpacking and rounding the bounds takes about two instructions a value, some 5 us.  What is left is the way from memory: three CTAs an
// SM, as many as its registers allow, have one turn of bounds a warp on it (a longer queue has not been tried).  The pages of all sequences are dealt
// out to the CTAs in equal shares; a warp takes 16 pages at a time, whose bounds it asks for a turn ahead, and multiplies them by
// all of the sequence's queries, which are rounded once a CTA; queries of several tokens share tiles of 16 rows.
// fa_cache_take then finds the `keep` highest of a query's scores.
#pragma once

#include "fa_cache.cuh"

namespace fa {

struct SelectArgs {
    CacheView c;
    CacheSeqs s;
    const uint8_t* q;
    int64_t q_b, q_t;        // strides in bytes
    uint32_t* keys;          // [B, T, kv heads, width]: sortable scores
    int32_t* pages;          // [B, T, kv heads, keep]
    uint32_t group, keep, first, last, bf16;
    uint32_t per_tile;       // tokens whose heads share a tile of 16 rows (1 where they are more than 16)
    uint32_t tiles;          // tiles that a CTA holds
    uint32_t turns;          // groups of 16 * tiles heads of a token (1 but for more than 64 of them)
    uint32_t token_chunks;   // of a CTA's tokens each
};

constexpr int kScoreWarps = 4;
constexpr int kScorePages = 16;    // of a warp at a time: two n-tiles
constexpr int kScoreCtas = 3;      // on an SM (four take registers that its pages are held in: 52 us against 45 with 32 long sequences)
constexpr int kScoreTiles = 4;     // of 16 query rows that a CTA holds at most

constexpr int kTakeThreads = 256;
constexpr int kTakeBinBits = 9;      // (32 queries on 20001 tokens, the whole call: 8 bits 17.3 us, 9 17.4, 10 18.3, 11 22.2; on 60000 in pages of 16: 76.1, 74.9, 76.0, 77.3)
constexpr uint32_t kTakeBins = 1u << kTakeBinBits;
constexpr uint32_t kTakeAlways = 0xFFFFFFFFu;   // key of a page that is taken whatever its score

// Whole numbers of the same order as the floats (a NaN above all), below kTakeAlways.
__device__ __forceinline__ uint32_t sortable(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);   // (-0 is 0)
    return min(u ^ (u & 0x80000000u ? 0xFFFFFFFFu : 0x80000000u), kTakeAlways - 1u);
}

// What the queries see: token t of `count` stands at position held - count + t; -1 where there is none.
__device__ __forceinline__ int64_t query_position(const CacheView& c, const CacheSeqs& s, uint32_t b, uint32_t t) {
    const int64_t held = cache_length(c, s, b), count = cache_count(s, b);
    const int64_t at = held - count + t;
    return t < count && at >= 0 ? at : -1;
}

// 16, 8 or 4 bytes of bounds.  Volatile: asked for where it stands, a turn ahead of its use.
template <int kBytes>
__device__ __forceinline__ void ld_bounds(const uint8_t* from, uint4& w) {
    w = make_uint4(0, 0, 0, 0);
    if constexpr (kBytes == 16) asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(from));
    else if constexpr (kBytes == 8) asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "l"(from));
    else asm volatile("ld.global.u32 %0, [%1];" : "=r"(w.x) : "l"(from));
}

// Scores of the pages [64 u0, 64 u1) of sequence b, for a head and the tokens of a chunk.  All threads of the CTA.
template <int H>
__device__ __forceinline__ void score_pages(const SelectArgs& p, uint32_t b, uint32_t head, uint32_t token_chunk, uint32_t u0, uint32_t u1, uint4* s_frag,
                                            float (*s_qs)[16], float (*s_val)[16][kScorePages + 1]) {
    constexpr int kHalves = H == 128 ? 2 : 1, kBytes = H >= 64 ? 16 : H / 4, kWords = kBytes / 4, kSteps = kHalves * kWords;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3u;
    const bool bf16 = p.bf16 != 0, many = p.group > 16;   // many: a token a CTA
    const uint32_t held = cache_length(p.c, p.s, b), count = cache_count(p.s, b);
    if (threadIdx.x == 0 && u0 == 0 && head == 0 && token_chunk == 0 && !cache_length_ok(p.c, p.s, b)) cache_report(p.c.status, kCacheBadPosition);
    const uint32_t t0 = many ? token_chunk : token_chunk * p.tiles * p.per_tile;
    if (held == 0 || t0 >= count) return;
    const uint32_t n_pages = min((held + p.c.page - 1) >> p.c.page_shift, u1 * (kScoreWarps * kScorePages));   // (pages in front of this are the call's)
    const uint32_t t_end = min(count, t0 + (many ? 1u : p.tiles * p.per_tile));

    for (uint32_t turn = 0; turn < p.turns; ++turn) {
        __syncthreads();   // what was there has been read
        // ---- q8 into fragments, a warp a tile
        for (uint32_t tile = warp; tile < p.tiles; tile += kScoreWarps) {
            float most[2], raw[2][kHalves][kBytes];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t r = u * 8 + g;
                const uint32_t t = many ? t0 : t0 + tile * p.per_tile + r / p.group, i = many ? (turn * p.tiles + tile) * 16 + r : r % p.group;
                const bool in = t < t_end && (many ? i < p.group : r < p.per_tile * p.group) && FA_CACHE_OK(p.c.status, kDbgRow, b < p.s.B && t < p.s.T && i < p.group);
                const uint8_t* const row = p.q + (in ? b * p.q_b + t * p.q_t + static_cast<int64_t>(head * p.group + i) * (2 * H) + 2 * t4 * kBytes : 0);
                most[u] = 0.0f;
#pragma unroll
                for (int half = 0; half < kHalves; ++half)
#pragma unroll
                    for (int j = 0; j < kWords; ++j) {
                        uint2 w = make_uint2(0, 0);
                        if (in) w = *reinterpret_cast<const uint2*>(row + half * 128 + 8 * j);
                        const float2 x = unpack_16(w.x, bf16), y = unpack_16(w.y, bf16);
                        raw[u][half][4 * j] = x.x, raw[u][half][4 * j + 1] = x.y, raw[u][half][4 * j + 2] = y.x, raw[u][half][4 * j + 3] = y.y;
                        most[u] = fmaxf(most[u], fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
                    }
                most[u] = fmaxf(most[u], __shfl_xor_sync(0xFFFFFFFFu, most[u], 1));
                most[u] = fmaxf(most[u], __shfl_xor_sync(0xFFFFFFFFu, most[u], 2));
                // (rows that are not there must not be the largest)
                if (t4 == 0) s_qs[tile][r] = in ? __fmul_rn(most[u], 1.0f / 127.0f) : -1.0f;
            }
            const float up[2] = {most[0] > 0.0f ? __fmul_rn(__frcp_rn(most[0]), 127.0f) : 0.0f, most[1] > 0.0f ? __fmul_rn(__frcp_rn(most[1]), 127.0f) : 0.0f};
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
#pragma unroll
                for (int j = 0; j < kWords; ++j) {
                    uint32_t plus[4], minus[4];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const float x = rintf(__fmul_rn(raw[u][half][4 * j + 2 * i], up[u])), y = rintf(__fmul_rn(raw[u][half][4 * j + 2 * i + 1], up[u]));
                            plus[2 * i + u] = pack_half2(fmaxf(x, 0.0f), fmaxf(y, 0.0f));
                            minus[2 * i + u] = pack_half2(fminf(x, 0.0f), fminf(y, 0.0f));
                        }
                    uint4* const to = s_frag + ((tile * kSteps + half * kWords + j) * 2) * 32 + lane;
                    to[0] = make_uint4(plus[0], plus[1], plus[2], plus[3]);
                    to[32] = make_uint4(minus[0], minus[1], minus[2], minus[3]);
                }
        }
        __syncthreads();

        // ---- 16 pages at a time: the table entries are asked for two turns ahead, the bounds one, when the registers of this turn's
        // are free again
        constexpr uint32_t stride = kScoreWarps * kScorePages;
        int32_t entry[2];
        float scale[2];
        bool there[2];
        uint4 raw[2][kHalves][2];
        auto ask_pages = [&](uint32_t p0) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const uint32_t mine = p0 + 8 * n + g;
                entry[n] = mine < n_pages && FA_CACHE_OK(p.c.status, kDbgEntry, b < p.s.B && mine < p.s.width) ? p.s.table[b * p.s.table_stride + mine] : -1;
            }
        };
        auto ask_bounds = [&](uint32_t p0) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                int32_t page = entry[n];
                if (static_cast<uint32_t>(page) >= p.c.n_pages) {
                    if (p0 + 8 * n + g < n_pages && t4 == 0 && turn == 0) cache_report(p.c.status, kCacheBadPage);
                    page = -1;
                }
                // (a page that is not there: read the first, and never take it for its score)
                const uint64_t at = static_cast<uint64_t>(page < 0 ? 0 : page) * p.c.heads + head;
                there[n] = page >= 0;
                const bool inside = FA_CACHE_OK(p.c.status, kDbgCodes, at < static_cast<uint64_t>(p.c.n_pages) * p.c.heads);
                scale[n] = p.c.k_scale[inside ? at : 0];   // (nothing may wait for it here)
                const uint8_t* const from = p.c.bounds + (inside ? at : 0) * (2 * H) + t4 * kBytes;
#pragma unroll
                for (int half = 0; half < kHalves; ++half)
#pragma unroll
                    for (int e = 0; e < 2; ++e) ld_bounds<kBytes>(from + e * H + half * 64, raw[n][half][e]);
            }
        };
        uint32_t p0 = (u0 * kScoreWarps + warp) * kScorePages;
        if (p0 < n_pages) {
            ask_pages(p0);
            ask_bounds(p0);
            ask_pages(p0 + stride);
        }
        for (; p0 < n_pages; p0 += stride) {
            // ---- bounds of pages p0 + g and p0 + 8 + g: whole numbers in fp16
            uint32_t hi[2][kHalves][kWords][2], lo[2][kHalves][kWords][2];
            const __half2 quarter = __float2half2_rn(0.25f), round = __float2half2_rn(1536.0f);   // (the unit of fp16 there is 1)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int half = 0; half < kHalves; ++half)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t w[4] = {raw[n][half][e].x, raw[n][half][e].y, raw[n][half][e].z, raw[n][half][e].w};
#pragma unroll
                        for (int j = 0; j < kWords; ++j) {
                            uint32_t x[2];
                            e4m3x4_to_half2(w[j], x[0], x[1]);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const __half2 y = __hsub2(__hfma2(*reinterpret_cast<const __half2*>(&x[i]), quarter, round), round);
                                (e ? hi : lo)[n][half][j][i] = *reinterpret_cast<const uint32_t*>(&y);
                            }
                        }
                    }
            // scales of the pages that this lane writes: page p0 + lane % 16
            const float scale_lo = __shfl_sync(0xFFFFFFFFu, there[0] ? scale_or_nan(scale[0]) : -1.0f, (lane & 7u) * 4),
                        scale_hi = __shfl_sync(0xFFFFFFFFu, there[1] ? scale_or_nan(scale[1]) : -1.0f, (lane & 7u) * 4);
            const float my_scale = lane & 8u ? scale_hi : scale_lo;
            if (p0 + stride < n_pages) {
                ask_bounds(p0 + stride);
                ask_pages(p0 + 2 * stride);
            }
            const uint32_t my_page = p0 + (lane & 15u);
            float best = -INFINITY;   // (many)
            for (uint32_t tile = 0; tile < p.tiles; ++tile) {
                float d[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                for (int half = 0; half < kHalves; ++half)
#pragma unroll
                    for (int j = 0; j < kWords; ++j) {
                        const uint4* const from = s_frag + ((tile * kSteps + half * kWords + j) * 2) * 32 + lane;
                        const uint4 x = from[0], y = from[32];
                        const uint32_t plus[4] = {x.x, x.y, x.z, x.w}, minus[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            mma_m16n8k16(d[n], plus, hi[n][half][j][0], hi[n][half][j][1]);
                            mma_m16n8k16(d[n], minus, lo[n][half][j][0], lo[n][half][j][1]);
                        }
                    }
                // ---- the largest of a token's heads, through the warp's own corner of shared memory
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float qs = s_qs[tile][u * 8 + g];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) s_val[warp][u * 8 + g][n * 8 + 2 * t4 + e] = qs < 0.0f ? -INFINITY : __fmul_rn(d[n][2 * u + e], qs);
                }
                __syncwarp();
                for (uint32_t i = lane >> 4; i < (many ? 1u : p.per_tile); i += 2) {
                    const uint32_t t = many ? t0 : t0 + tile * p.per_tile + i, rows = many ? 16u : p.group;
                    if (t >= t_end) break;
                    float x = best;
                    for (uint32_t r = 0; r < rows; ++r) x = fmaxf(x, s_val[warp][(many ? 0u : i * p.group) + r][lane & 15u]);
                    if (many) {
                        best = x;
                        if (tile + 1 < p.tiles) break;
                    }
                    if (my_page < n_pages && FA_CACHE_OK(p.c.status, kDbgScratch, my_page < p.s.width && t < p.s.T && head < p.c.heads)) {
                        const int64_t position = query_position(p.c, p.s, b, t);
                        const int64_t own = position >> p.c.page_shift;
                        uint32_t key = sortable(my_scale == -1.0f ? -INFINITY : __fmul_rn(x, my_scale));
                        if (my_page < p.first || static_cast<int64_t>(my_page) > own - static_cast<int64_t>(p.last)) key = kTakeAlways;
                        if (position < 0 || static_cast<int64_t>(my_page) > own) key = 0;   // behind the query
                        uint32_t* const at = p.keys + ((static_cast<uint64_t>(b) * p.s.T + t) * p.c.heads + head) * p.s.width + my_page;
                        *at = turn > 0 ? max(key, *at) : key;
                    }
                }
                __syncwarp();
            }
        }
    }
}

template <int H>
__global__ void __launch_bounds__(kScoreWarps * 32, kScoreCtas) fa_cache_scores(const SelectArgs p) {
    extern __shared__ __align__(16) uint4 s_frag[];   // [tiles][kSteps][positive, negative part][lane]
    FA_CACHE_POISON(smem_u32(s_frag), p.tiles * (H / 16) * 2 * 32 * 16);
    __shared__ float s_qs[kScoreTiles][16];
    __shared__ float s_val[kScoreWarps][16][kScorePages + 1];
    grid_dep_wait();
    grid_dep_launch();
    __shared__ uint32_t s_share[kShareWords + kScoreWarps];
    const uint32_t per_seq = p.c.heads * p.token_chunks;
    constexpr uint32_t kUnit = kScoreWarps * kScorePages;   // pages
    auto units = [&](uint32_t i) { return max(1u, (cache_length(p.c, p.s, i) + kUnit * p.c.page - 1) / (kUnit * p.c.page)); };
    uint32_t unit, unit_end, b, before;
    if (!share_of<kScoreWarps>(units, false, p.s.B, per_seq, 1, s_share, unit, unit_end, b, before)) return;
    while (unit < unit_end) {
        const uint32_t n_units = units(b), problem = (unit - before) / n_units, u0 = unit - before - problem * n_units, u1 = min(n_units, u0 + (unit_end - unit));
        unit += u1 - u0;
        const uint32_t b_now = b, b_next = unit == before + n_units * per_seq ? b + 1 : b;
        if (b_next != b) before = unit;
        b = b_next;
        score_pages<H>(p, b_now, problem % p.c.heads, problem / p.c.heads, u0, u1, s_frag, s_qs, s_val);
    }
}

// Sum over the lanes of this one and those in front of it.
__device__ __forceinline__ uint32_t sum_upto(uint32_t x, uint32_t lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, d);
        if (lane >= static_cast<uint32_t>(d)) x += y;
    }
    return x;
}

// The `keep` highest keys of a query, the lowest pages of equal ones, in the order of the pages.  Their threshold is found by counting:
// the keys' range, lowest to highest, is cut into kTakeBins equal bins, the keys of each are counted, and the bin that the threshold
// lies in is the next range, unless all of its keys are wanted or it has one value.  The range is 32 bits, so four counts are enough
// for any keys; spread as scores are, one or two are needed.  Bound by the way through its barriers: 3 us of the 8.1 that one query on
// 313 pages takes.  A search over the threshold's bits, up to 16 counts, took 4 (the whole call with 32 queries on 20001 tokens: 17.4
// us and 21.8, on 131072: 47.7 and 51.8).
// kHeld: keys of a thread in registers (0: any number, from memory each time).
template <int kHeld>
__global__ void __launch_bounds__(kTakeThreads) fa_cache_take(const SelectArgs p) {
    constexpr uint32_t kWarps = kTakeThreads / 32, kBinsEach = kTakeBins / kTakeThreads;
    __shared__ uint32_t s_bins[kTakeBins];
    __shared__ uint32_t s_low[kWarps], s_high[kWarps], s_sum[kWarps];
    __shared__ uint32_t s_scan[kWarps][2], s_found[3];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
#pragma unroll
    for (uint32_t i = 0; i < kBinsEach; ++i) s_bins[i * kTakeThreads + tid] = 0;
    grid_dep_wait();
    grid_dep_launch();
    const uint64_t index = blockIdx.x;   // (b, t, head)
    const uint64_t bt = index / p.c.heads;
    const uint32_t t = static_cast<uint32_t>(bt % p.s.T), b = static_cast<uint32_t>(bt / p.s.T);
    const int64_t position = query_position(p.c, p.s, b, t);
    const uint32_t n = position < 0 ? 0u : static_cast<uint32_t>((position >> p.c.page_shift) + 1);   // pages that the query sees
    const uint32_t* const keys = p.keys + index * p.s.width;
    int32_t* const out = p.pages + index * p.keep;
    if (n <= p.keep) {
        for (uint32_t i = tid; i < p.keep; i += kTakeThreads) out[i] = i < n ? static_cast<int32_t>(i) : -1;
        return;
    }
    const uint32_t per = (n + kTakeThreads - 1) / kTakeThreads;   // keys of a thread, one behind the other
    const uint32_t begin = min(n, tid * per), end = FA_CACHE_OK(p.c.status, kDbgScratch, n <= p.s.width && (kHeld == 0 || per <= kHeld)) ? min(n, begin + per) : begin;
    uint32_t mine[kHeld > 0 ? kHeld : 1];
    if (kHeld > 0) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) mine[i] = begin + i < end ? keys[begin + i] : 0u;
    }
    auto put = [&](uint32_t place, uint32_t i) {
        if (FA_CACHE_OK(p.c.status, kDbgRow, place < p.keep && i < p.s.width)) out[place] = static_cast<int32_t>(i);
    };
    auto each = [&](auto&& f) {
        if (kHeld > 0) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (begin + i < end) f(begin + i, mine[i]);
        } else {
            for (uint32_t i = begin; i < end; ++i) f(i, keys[i]);
        }
    };
    // The range, without the pages that are always taken, or of those alone where there are more of them than are wanted.
    uint32_t low = kTakeAlways, high = 0, always = 0;
    each([&](uint32_t, uint32_t key) {
        if (key == kTakeAlways) ++always;
        else low = min(low, key), high = max(high, key);
    });
    low = __reduce_min_sync(0xFFFFFFFFu, low), high = __reduce_max_sync(0xFFFFFFFFu, high), always = __reduce_add_sync(0xFFFFFFFFu, always);
    if (lane == 0) s_low[warp] = low, s_high[warp] = high, s_sum[warp] = always;
    __syncthreads();
    always = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) low = min(low, s_low[w]), high = max(high, s_high[w]), always += s_sum[w];
    uint32_t want = p.keep - always;   // of the keys in [low, low + range], which are more than that
    if (always >= p.keep) want = p.keep, low = high = kTakeAlways;
    uint32_t range = high - low;
    uint32_t least, ties;   // taken: the keys above `least`, and the first `ties` that are equal to it
    for (;;) {
        const uint32_t shift = max(32 - __clz(range), kTakeBinBits) - kTakeBinBits;   // range >> shift < kTakeBins
        each([&](uint32_t, uint32_t key) {
            if (key >= low && key - low <= range) atomicAdd(&s_bins[(key - low) >> shift], 1u);
        });
        __syncthreads();
        // keys from the highest bin on: thread 0 has the highest bins
        uint32_t count[kBinsEach], sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < kBinsEach; ++i) {
            uint32_t& bin = s_bins[kTakeBins - 1 - (tid * kBinsEach + i)];
            sum += count[i] = bin;
            bin = 0;
        }
        const uint32_t upto = sum_upto(sum, lane);
        if (lane == 31) s_sum[warp] = upto;
        __syncthreads();
        uint32_t front = upto - sum;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) front += w < warp ? s_sum[w] : 0u;
        if (front < want && want <= front + sum) {   // one thread's
#pragma unroll
            for (uint32_t i = 0; i < kBinsEach; ++i) {
                if (front < want && want <= front + count[i])
                    s_found[0] = kTakeBins - 1 - (tid * kBinsEach + i), s_found[1] = want - front, s_found[2] = count[i];
                front += count[i];
            }
        }
        __syncthreads();
        low += s_found[0] << shift, want = s_found[1];
        if (want == s_found[2]) {   // the whole bin (it is not the one with the lowest key, n > keep, so that `low` is not 0)
            least = low - 1, ties = 0;
            break;
        }
        if (shift == 0) {
            least = low, ties = want;
            break;
        }
        range = min((1u << shift) - 1u, high - low);   // (the highest bin may reach beyond `high`, to the pages that are always taken)
    }
    // how many that are above, equal the threads in front have
    uint32_t mine_above = 0, mine_equal = 0;
    each([&](uint32_t, uint32_t key) { mine_above += key > least ? 1u : 0u, mine_equal += key == least ? 1u : 0u; });
    const uint32_t upto_above = sum_upto(mine_above, lane), upto_equal = sum_upto(mine_equal, lane);
    if (lane == 31) s_scan[warp][0] = upto_above, s_scan[warp][1] = upto_equal;
    __syncthreads();
    uint32_t front_above = upto_above - mine_above, front_equal = upto_equal - mine_equal;
    for (uint32_t w = 0; w < warp; ++w) front_above += s_scan[w][0], front_equal += s_scan[w][1];
    each([&](uint32_t i, uint32_t key) {
        if (key > least) {
            put(front_above + min(front_equal, ties), i);
            ++front_above;
        } else if (key == least) {
            if (front_equal < ties) put(front_above + front_equal, i);
            ++front_equal;
        }
    });
}

}  // namespace fa
