// Attention over the cache for few query rows a key/value head: single tokens, drafted tokens, tokens with a list of pages.
//
// The query heads that share a key/value head, and the sequence's T tokens, are rows of one problem: row t * group + i.  A
// problem is 16 * MT of these rows of one sequence and key/value head (with a list of pages: the rows of one token).  What
// bounds it is memory, 2 H bytes a token and head (64 sequences of up to 8192 tokens, 8 heads of 128: 96 us, 523 MB, 5.4 TB/s; 2 of
// 131000, 4 heads: 56 us with the join, 268 MB), so the work is cut by keys: all problems' units of 128 tokens stand in one row, with
// kRowsSetup units in front of each problem's, CTA c of G takes units [c W / G, (c + 1) W / G) of the W there are, whatever problems
// they belong to, and a problem that several CTAs share is put together by fa_cache_join or fa_cache_join_few.  Lengths are only
// known on the device, so every CTA adds them up itself.  With 25 rows (16 sequences of up to 4001 tokens: 38 us, 2.0 TB/s) the
// products and exponentials count beside the reading.
//
// Inside a CTA each warp takes 32 tokens of a unit, through a ring of its own in shared memory that cp.async fills: nobody
// waits for another warp before the end of the problem.  Both products are mma.sync m16n8k16 in fp16 (with these rows a tcgen05 tile of
// 128 would be mostly empty; one with the keys as its rows and these as its columns has not been tried): a thread reads the codes of
// its own fragment straight from the ring, the order of the dimensions in Q K^T and of the tokens in P V being chosen so that they are 16
// contiguous bytes, and turns them into fp16, which is exact.
//
// Scales: the key scale is multiplied into the fp32 scores.  The value scale goes into the exponent: w = 2^(s + log2 scale - M)
// with M the running maximum of just that exponent, so that P needs no second rounding and cannot leave fp16, whatever the
// scales; the row sum takes it out again, l = sum over pages of (sum of w) / scale, in fp32 (where scales lie
// far apart, kSpanOfScales, by an exponential more a score).  M moves only when an exponent passes it by more than 8 (w <= 2^8), so the sums
// are seldom rescaled.
#pragma once

#include "fa_cache.cuh"

namespace fa {

constexpr int kRowsWarps = 4;
constexpr int kRowsStage = 32;                       // tokens of a warp's stage
constexpr int kRowsUnit = kRowsWarps * kRowsStage;   // tokens of a unit
// What a problem costs a CTA beside its tokens (queries, the way to the first key, joining the warps), in units: counted when the
// work is dealt out, so that a CTA with many short sequences gets fewer tokens.  (0, 1, 2, 3 units: 117, 106, 96, 99 us with 64
// sequences of 100 to 8192 tokens; 36.0, 34.7, 33.8, 33.6 with 16 and lists of 64 pages.)
constexpr uint32_t kRowsSetup = 2;
constexpr float kRowsSlack = 8.0f;                   // how far an exponent may pass M before M moves
constexpr uint32_t kNoToken = 0x7FFFFFFFu;           // position of tokens that are not there

struct RowsArgs {
    CacheView c;
    CacheSeqs s;
    const uint8_t* q;
    uint8_t* y;              // [B, T, heads * H] contiguous
    const int32_t* pages;    // [B, T, kv heads, keep] or null
    int64_t q_b, q_t;        // strides in bytes
    uint32_t group, keep, causal, bf16;
    uint32_t row_tiles;      // problems of a sequence and key/value head
    uint32_t rows;           // rows of a problem (at most 16 MT; the last may have fewer)
    uint32_t min_units;      // units that a CTA takes at least; 0: a CTA takes a problem
    float scale_log2;        // log2(e) / sqrt(H)
    float* part_o;           // [2 G slots, 16 MT rows, H]
    float2* part_ml;         // [2 G slots, 16 MT rows]
    int2* shares;            // [problems]: first and last CTA
#ifdef FA_DEBUG
    uint64_t slots, problems;   // that the scratch has room for
#endif
};

template <int H, int MT>
struct RowsCfg {
    static constexpr int kRows = 16 * MT;
    static constexpr int kCodes = kRowsStage * H;                  // bytes of a stage's keys (or values)
    static constexpr int kMeta = 32;                               // a stage's scales and positions
    static constexpr int kStageBytes = 2 * kCodes + kMeta;
    static constexpr int kStages = 2;
    static constexpr int kRing = kRowsWarps * kStages * kStageBytes;
    static constexpr int kMerge = kRowsWarps * kRows * H * 4;
    static constexpr int kTiles = kRing > kMerge ? kRing : kMerge;
    static constexpr int kQ = kRows * H * 2;
    static constexpr int kSmem = kTiles + kQ + kRows * 8 + kRowsWarps * kRows * 8 + 128;
    static constexpr int kCtas = MT == 1 ? 3 : 2;                  // per SM
};

__device__ __forceinline__ uint32_t rows_units(const RowsArgs& p, uint32_t b) {
    const uint32_t tokens = p.pages != nullptr ? p.keep << p.c.page_shift : cache_length(p.c, p.s, b);
    return max(1u, (tokens + kRowsUnit - 1) / kRowsUnit);
}

// 16 bytes of the ring: chunk `c` of row `r`, rows of H bytes, chunks moved about so that the reads below meet few conflicts.
template <int H>
__device__ __forceinline__ uint32_t key_chunk(uint32_t r, uint32_t c) {
    return r * H + ((H == 128 ? c ^ ((r & 1u) << 2) : c) << 4);
}
template <int H>
__device__ __forceinline__ uint32_t value_chunk(uint32_t r, uint32_t c) {
    return r * H + ((H == 128 ? c ^ (r & 6u) : H == 64 ? c ^ ((r >> 1) & 3u) : c) << 4);
}
// 16 (8) bytes of global memory, zeros where `in` is false.  Volatile: asked for where it stands.
template <int kBytes>
__device__ __forceinline__ void ld_or_zero(const uint8_t* from, bool in, uint32_t (&w)[kBytes / 4]) {
    if constexpr (kBytes == 16)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                     "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                     : "=&r"(w[0]), "=&r"(w[1]), "=&r"(w[2]), "=&r"(w[3]) : "l"(from), "r"(static_cast<uint32_t>(in)));
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\t@p ld.global.v2.u32 {%0, %1}, [%2];\n\t}"
                     : "=&r"(w[0]), "=&r"(w[1]) : "l"(from), "r"(static_cast<uint32_t>(in)));
}
__device__ __forceinline__ void cp_async_16_all(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int kBytes>
__device__ __forceinline__ void ld_codes(uint32_t addr, uint32_t (&w)[kBytes / 4 > 0 ? kBytes / 4 : 1]) {
    if constexpr (kBytes == 16) {
        ld_shared_v4(addr, w);
    } else if constexpr (kBytes == 8) {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    } else if constexpr (kBytes == 4) {
        w[0] = ld_shared_u32(addr);
    } else {
        uint16_t h;
        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(h) : "r"(addr));
        w[0] = h;
    }
}

// kRest: what the weights lose when they are rounded to fp16 is multiplied too.  For results in fp16, whose own rounding is no larger: with
// it the error is that of the results' rounding alone, without it 1.4 times that; in bf16 it would not show (1.01 times).  All fp16 calls
// have it, so that how exact a sequence's results are does not depend on what else is in the call.
//   kRestApart   by a product of its own (64 sequences of 100 to 8192 tokens, 4 rows: 111 us, 97 without)
//   kRestAbove   by the same product: a problem has eight rows at most then, and the m-tile's upper eight are what the weights of the lower
//                ones have lost (those calls 96 us; one of 301 tokens 8.2 us, 9.0 with kRestApart)
enum : int { kRestNone = 0, kRestApart, kRestAbove };
template <int H, int MT, int kRest>
__global__ void __launch_bounds__(kRowsWarps * 32, RowsCfg<H, MT>::kCtas) fa_cache_rows(const RowsArgs p) {
    using Cfg = RowsCfg<H, MT>;
    constexpr int kThreads = kRowsWarps * 32;
    constexpr int kHalves = H == 128 ? 2 : 1;            // 64-byte halves of a key row
    constexpr int kKeyBytes = H >= 64 ? 16 : H / 4;      // that a thread reads of a half
    constexpr int kValueBytes = H / 8;                   // that a thread reads of a value row
    constexpr int kTilesN = H / 8;                       // n-tiles of P V
    constexpr bool kAbove = kRest == kRestAbove;
    static_assert(!kAbove || MT == 1, "eight rows");
    constexpr int kU = kAbove ? 1 : 2, kE = 2 * kU;      // a thread's rows of an m-tile, its scores of an n-tile
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, t4 = lane & 3u;
    const uint32_t ring = smem_u32(smem) + warp * (Cfg::kStages * Cfg::kStageBytes);
    uint8_t* const q_frag = smem + Cfg::kTiles;
    float* const s_coef = reinterpret_cast<float*>(q_frag + Cfg::kQ);
    uint32_t* const s_limit = reinterpret_cast<uint32_t*>(s_coef + Cfg::kRows);
    float2* const s_ml = reinterpret_cast<float2*>(s_limit + Cfg::kRows);
    uint32_t* const s_share = reinterpret_cast<uint32_t*>(s_ml + kRowsWarps * Cfg::kRows);
    volatile uint32_t* const s_now = s_share + kShareWords + kRowsWarps;
    FA_CACHE_POISON(smem_u32(smem), Cfg::kSmem);
    grid_dep_wait();
    grid_dep_launch();
    const bool bf16 = p.bf16 != 0;
    const uint32_t per_seq = p.c.heads * p.row_tiles;   // problems of a sequence

    // ---- this CTA's units
    uint32_t unit, unit_end, before = 0, b = 0;   // `before`: units of the sequences in front of b
    if (p.min_units == 0) {
        b = blockIdx.x / per_seq;
        const uint32_t n = rows_units(p, b);
        unit = (blockIdx.x - b * per_seq) * n;
        unit_end = unit + n;
    } else {
        const bool alike = p.pages != nullptr;   // every sequence has as many
        if (!share_of<kRowsWarps>([&](uint32_t i) { return rows_units(p, i) + kRowsSetup; }, alike, p.s.B, per_seq, p.min_units, s_share, unit, unit_end, b, before)) return;
    }

    const uint32_t setup = p.min_units == 0 ? 0u : kRowsSetup;   // units in front of a problem's own
    for (bool first_segment = true; unit < unit_end;) {
        const uint32_t n_units = rows_units(p, b), all_units = n_units + setup;
        const uint32_t within = unit - before;
        const uint32_t problem = within / all_units, w0 = within - problem * all_units, w1 = min(all_units, w0 + (unit_end - unit));
        const uint32_t u0 = max(w0, setup) - setup, u1 = max(w1, setup) - setup;
        unit += w1 - w0;
        if (u1 == 0) continue;   // (the next CTA begins with the problem's first unit)
        const uint32_t head = problem / p.row_tiles, tile = problem % p.row_tiles;
        const uint32_t row0 = tile * p.rows;   // rows of the sequence and head: T * group
        const uint32_t n_rows = min(p.rows, p.s.T * p.group - row0);
        const uint32_t held = cache_length(p.c, p.s, b), count = cache_count(p.s, b);
        if (tid == 0 && u0 == 0 && !cache_length_ok(p.c, p.s, b)) cache_report(p.c.status, kCacheBadPosition);
        // keys that a row of token t sees; of all rows [nearest, farthest)
        auto limit_of = [&](uint32_t t) {
            if (t >= count) return 0u;
            if (!p.causal) return held;
            return held + t >= count ? min(held, held + t - count + 1u) : 0u;
        };
        const uint32_t t_first = row0 / p.group, t_last = (row0 + n_rows - 1) / p.group;
        const uint32_t nearest = min(limit_of(t_first), limit_of(t_last));
        const uint32_t farthest = t_first >= count ? 0u : limit_of(min(t_last, count - 1u));

        // ---- the ring.  Lane l knows the pages of group l (16 tokens) of the warp's next 16 stages.
        const uint32_t n_stages = u1 - u0;
        // (what is needed once in 16 stages is kept in shared memory, not in registers)
        if (tid == 0) {
            s_now[0] = b, s_now[1] = (b * p.s.T + t_first) * p.c.heads + head, s_now[2] = u0;
            // whether the problem is this CTA's alone, its last unit, the place of its sums; where the work goes on
            const bool over = unit == before + all_units * per_seq;
            s_now[3] = u0 == 0 && u1 == n_units, s_now[4] = before + (problem + 1) * all_units - 1, s_now[5] = 2 * blockIdx.x + (first_segment ? 0u : 1u);
            s_now[6] = unit, s_now[7] = unit_end, s_now[8] = over ? unit : before, s_now[9] = over ? b + 1 : b, s_now[10] = problem;
        }
        __syncthreads();
        constexpr uint32_t kChunks = H / 16;                 // of a row; 32 lanes copy 32 / kChunks rows at a time
        constexpr uint32_t kRowsAtOnce = 32 / kChunks;
        const uint32_t copy_row = lane / kChunks, copy_chunk = lane % kChunks;
        const bool copies = copy_row < 16;                   // (H = 16: half the lanes)
        const uint8_t* const k_base = p.c.k + static_cast<int64_t>(head) * p.c.k_head + static_cast<int64_t>(copy_row) * p.c.k_token + copy_chunk * 16;
        const uint8_t* const v_base = p.c.v + static_cast<int64_t>(head) * p.c.v_head + static_cast<int64_t>(copy_row) * p.c.v_token + copy_chunk * 16;
        int32_t my_page = -1;
        uint32_t my_at = kNoToken;   // position of the group's first token
        auto look_up = [&](uint32_t stage) {
            const int32_t* const table = p.s.table + s_now[0] * p.s.table_stride;
            const int32_t* const list = p.pages != nullptr ? p.pages + static_cast<uint64_t>(s_now[1]) * p.keep : nullptr;
            const uint32_t token = (s_now[2] + stage + (lane >> 1)) * kRowsUnit + warp * kRowsStage + (lane & 1u) * 16;
            my_page = -1, my_at = kNoToken;
            if (stage + (lane >> 1) >= n_stages) return;
            uint32_t block = token >> p.c.page_shift;
            if (list != nullptr) {
                const bool listed = FA_CACHE_OK(p.c.status, kDbgEntry, s_now[1] < static_cast<uint64_t>(p.s.B) * p.s.T * p.c.heads);
                const int32_t chosen = listed && block < p.keep ? list[block] : -1;
                if (chosen < 0) return;   // (not filled)
                block = static_cast<uint32_t>(chosen);
            }
            const bool inside = block < p.s.width;
            const uint64_t at = (static_cast<uint64_t>(block) << p.c.page_shift) + (token & (p.c.page - 1));
            if (inside && FA_CACHE_OK(p.c.status, kDbgEntry, s_now[0] < p.s.B)) my_page = table[block];   // (an entry that no token reaches may be anything)
            bool bad = list != nullptr && !inside;
            if (!bad && at < farthest) {
                bad = static_cast<uint32_t>(my_page) >= p.c.n_pages;
                my_at = static_cast<uint32_t>(at);
            } else {
                my_page = -1;
            }
            if (bad) {
                my_page = -1, my_at = kNoToken;
                cache_report(p.c.status, kCacheBadPage);
            }
        };
        auto issue = [&](uint32_t stage) {
            if (stage < n_stages) {
                if ((stage & 15u) == 0) look_up(stage);
                const uint32_t to = ring + (stage % Cfg::kStages) * Cfg::kStageBytes, from_lane = 2 * (stage & 15u);
#pragma unroll
                for (int half = 0; half < 2; ++half) {   // (a group of 16 tokens never spans two pages)
                    const int32_t page = __shfl_sync(0xFFFFFFFFu, my_page, from_lane + half);
                    const uint32_t at = __shfl_sync(0xFFFFFFFFu, my_at, from_lane + half), in_page = at & (p.c.page - 1);
                    const uint32_t meta = to + 2 * Cfg::kCodes + 4 * half;
                    if (lane == 0) st_shared_u32(meta + 16, at);
                    const uint64_t ph = page < 0 ? 0u : static_cast<uint32_t>(page);
                    const uint8_t* k0 = k_base + ph * static_cast<uint32_t>(p.c.k_page) + in_page * static_cast<uint32_t>(p.c.k_token);
                    const uint8_t* v0 = v_base + ph * static_cast<uint32_t>(p.c.v_page) + in_page * static_cast<uint32_t>(p.c.v_token);
                    const bool holds = page < 0 || FA_CACHE_OK(p.c.status, kDbgCodes, static_cast<uint32_t>(page) < p.c.n_pages && head < p.c.heads && in_page + 16 <= p.c.page);
                    if (!copies || !holds || !FA_CACHE_OK(p.c.status, kDbgTile, to + Cfg::kStageBytes <= smem_u32(smem) + Cfg::kRing)) {
                    } else if (page >= 0 && at + 16 <= farthest) {
#pragma unroll
                        for (uint32_t r = 0; r < 16; r += kRowsAtOnce) {
                            cp_async_16_all(to + key_chunk<H>(half * 16 + r + copy_row, copy_chunk), k0);
                            cp_async_16_all(to + Cfg::kCodes + value_chunk<H>(half * 16 + r + copy_row, copy_chunk), v0);
                            k0 += kRowsAtOnce * static_cast<uint32_t>(p.c.k_token), v0 += kRowsAtOnce * static_cast<uint32_t>(p.c.v_token);
                        }
                    } else {   // what no row may see is not read (its codes may be anything), but filled with zeros
#pragma unroll
                        for (uint32_t r = 0; r < 16; r += kRowsAtOnce) {
                            const bool in = page >= 0 && at + r + copy_row < farthest;
                            cp_async_16_zero(to + key_chunk<H>(half * 16 + r + copy_row, copy_chunk), in ? k0 : p.c.k, in);
                            cp_async_16_zero(to + Cfg::kCodes + value_chunk<H>(half * 16 + r + copy_row, copy_chunk), in ? v0 : p.c.v, in);
                            k0 += kRowsAtOnce * static_cast<uint32_t>(p.c.k_token), v0 += kRowsAtOnce * static_cast<uint32_t>(p.c.v_token);
                        }
                    }
                    if (lane < 2) {
                        const float* const scale = (lane ? p.c.v_scale : p.c.k_scale) + ph * p.c.heads + head;
                        if (page >= 0) cp_async_4(meta + 8 * lane, reinterpret_cast<uint64_t>(scale));
                        else st_shared_u32(meta + 8 * lane, 0x3F800000u);
                    }
                }
            }
            cp_async_commit();
        };
        // ---- queries, a warp 8 rows, asked for ahead of the first keys
        constexpr int kPart = H >= 32 ? 16 : 8;                          // bytes of a fragment's part: 8 (4) dimensions
        constexpr int kParts = H >= 64 ? 2 : 1;
        const uint32_t q_row = warp * 8 + g, q_token = (row0 + q_row) / p.group;
        uint32_t w[kHalves * kParts][kPart / 4];
        if (warp < 2 * MT) {
            const uint32_t i = (row0 + q_row) - q_token * p.group;
            const bool in = q_row < n_rows && q_token < count && FA_CACHE_OK(p.c.status, kDbgRow, b < p.s.B && q_token < p.s.T && i < p.group && head < p.c.heads);
            const uint8_t* const q_at = p.q + (in ? b * p.q_b + q_token * p.q_t + static_cast<int64_t>(head * p.group + i) * (2 * H) + 2 * t4 * kKeyBytes : 0);
#pragma unroll
            for (int x = 0; x < kHalves * kParts; ++x) ld_or_zero<kPart>(q_at + 2 * ((x / kParts) * 64 + (x % kParts) * 8), in, w[x]);
        }
        issue(0);
        // ---- into fragments: rows whose fp16 form could overflow (bf16) are scaled by a power of two
        if (warp < 2 * MT) {
            float coef = p.scale_log2;
            if (bf16) {
                float most = 0.0f;
#pragma unroll
                for (int x = 0; x < kHalves * kParts; ++x)
#pragma unroll
                    for (int e = 0; e < kPart / 4; ++e) {
                        const float2 y = unpack_16(w[x][e], true);
                        most = fmaxf(most, fmaxf(fabsf(y.x), fabsf(y.y)));
                    }
                most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
                const uint32_t e8 = max(__float_as_uint(most) >> 23, 40u);   // biased: 2^(e8 - 127) <= most, unless that is tiny
                // to [2^7, 2^8): what does not lie in fp16's range then is 2^-22 of the row's largest or less
                float up = 1.0f;
                if (e8 < 255) coef *= __uint_as_float((e8 - 7) << 23), up = __uint_as_float((261 - e8) << 23);
#pragma unroll
                for (int x = 0; x < kHalves * kParts; ++x)
#pragma unroll
                    for (int e = 0; e < kPart / 4; ++e) {
                        const float2 y = unpack_16(w[x][e], true);
                        w[x][e] = pack_half2(y.x * up, y.y * up);
                    }
            }
#pragma unroll
            for (int x = 0; x < kHalves * kParts; ++x) {   // (rows of a warp: m-tile warp / 2, its upper or lower eight)
                const uint32_t item = (((warp >> 1) * kHalves + x / kParts) * 2 + (warp & 1u)) * kParts + x % kParts;
                uint8_t* const to = q_frag + (item * 32 + lane) * kPart;
                if constexpr (kPart == 16) *reinterpret_cast<uint4*>(to) = make_uint4(w[x][0], w[x][1], w[x][2], w[x][3]);
                else *reinterpret_cast<uint2*>(to) = make_uint2(w[x][0], w[x][1]);
            }
            if (t4 == 0) s_coef[q_row] = coef, s_limit[q_row] = q_row < n_rows ? limit_of(q_token) : kNoToken;   // (rows that are not there hold nobody up)
        }
        __syncthreads();
        float coef[MT][2], m[MT][2], l[MT][2], o[MT][kTilesN][4];
        uint32_t limit[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                coef[mt][u] = s_coef[mt * 16 + u * 8 + g];
                limit[mt][u] = s_limit[mt * 16 + u * 8 + g];
                m[mt][u] = -INFINITY, l[mt][u] = 0.0f;
            }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < kTilesN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][j][e] = 0.0f;

        float vtop = -INFINITY;   // log2 of the largest value scale that the warp has met
        for (uint32_t stage = 0; stage < n_stages; ++stage) {
            issue(stage + 1);
            cp_async_wait_group<1>();
            __syncwarp();
            const uint32_t tile_at = ring + (stage % Cfg::kStages) * Cfg::kStageBytes;
            const uint32_t meta = tile_at + 2 * Cfg::kCodes;
            const uint32_t at[2] = {ld_shared_u32(meta + 16), ld_shared_u32(meta + 20)};
            if (min(at[0], at[1]) < farthest) {   // (else no row sees any of it)
                // ---- S = Q K^T: four n-tiles of 8 tokens
                float s[MT][4][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[mt][n][e] = 0.0f;
#pragma unroll
                for (int half = 0; half < kHalves; ++half) {
                    uint32_t kw[4][kKeyBytes / 4];
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        if constexpr (H >= 64) ld_codes<16>(tile_at + key_chunk<H>(n * 8 + g, half * 4 + t4), kw[n]);
                        else ld_codes<kKeyBytes>(tile_at + (n * 8 + g) * H + t4 * kKeyBytes, kw[n]);
                    uint32_t kf[4][kKeyBytes / 4][2];
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int j = 0; j < kKeyBytes / 4; ++j) e4m3x4_to_half2(kw[n][j], kf[n][j][0], kf[n][j][1]);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        constexpr int kRegs = kKeyBytes / 2;   // fp16 pairs of a row's half
                        uint32_t qa[2][kRegs];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int part = 0; part < kParts; ++part) {
                                const uint32_t item = ((mt * kHalves + half) * 2 + u) * kParts + part;
                                const uint32_t from = smem_u32(q_frag) + (item * 32 + lane) * kPart;
                                uint32_t w[kPart / 4];
                                ld_codes<kPart>(from, w);
#pragma unroll
                                for (int e = 0; e < kPart / 4; ++e) qa[u][part * 4 + e] = w[e];
                            }
#pragma unroll
                        for (int j = 0; j < kKeyBytes / 4; ++j) {
                            const uint32_t a[4] = {qa[0][2 * j], qa[1][2 * j], qa[0][2 * j + 1], qa[1][2 * j + 1]};
#pragma unroll
                            for (int n = 0; n < 4; ++n) mma_m16n8k16(s[mt][n], a, kf[n][j][0], kf[n][j][1]);
                        }
                    }
                }
                // ---- exponents, weights, row sums
                float ks[2], vlog[2], vinv[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    ks[u] = scale_or_nan(__uint_as_float(ld_shared_u32(meta + 4 * u)));
                    const float vs = scale_or_nan(__uint_as_float(ld_shared_u32(meta + 8 + 4 * u)));
                    const float held_up = vs < 0x1p-100f ? 0x1p-100f : vs;   // (a scale of zero has no logarithm)
                    vlog[u] = __log2f(held_up);
                    vinv[u] = exp2f(-vlog[u]);   // of the rounded logarithm, so that the two cancel
                    if (held_up != held_up) vinv[u] = held_up;
                }
                vtop = max3(vtop, vlog[0], vlog[1]);
                const bool wide = fminf(vlog[0], vlog[1]) < vtop - kSpanOfScales;   // a page of the stage is far below that
                const bool whole = max(at[0], at[1]) < kNoToken && max(at[0], at[1]) + 16 <= nearest;
                uint32_t pf[MT][4][2], rest[MT][4][2];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    // exponents against M, a whole number, so that with scales that are powers of two nothing is rounded but the result
                    float top[2] = {-INFINITY, -INFINITY}, cu[2][2], add[2][2];
#pragma unroll
                    for (int u = 0; u < kU; ++u) {
                        const float ref = m[mt][u] == -INFINITY ? 0.0f : m[mt][u];
#pragma unroll
                        for (int h2 = 0; h2 < 2; ++h2) cu[u][h2] = coef[mt][u] * ks[h2], add[u][h2] = vlog[h2] - ref;
                    }
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int e = 0; e < kE; ++e) s[mt][n][e] = fmaf(s[mt][n][e], cu[e >> 1][n >> 1], add[e >> 1][n >> 1]);
                    if (!whole) {
#pragma unroll
                        for (int n = 0; n < 4; ++n)
#pragma unroll
                            for (int e = 0; e < kE; ++e) {
                                const uint32_t pos = at[n >> 1] + (n & 1) * 8 + 2 * t4 + (e & 1);
                                if (at[n >> 1] == kNoToken || pos >= limit[mt][e >> 1]) s[mt][n][e] = -INFINITY;
                            }
                    }
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int u = 0; u < kU; ++u) top[u] = max3(top[u], s[mt][n][2 * u], s[mt][n][2 * u + 1]);
#pragma unroll
                    for (int u = 0; u < kU; ++u) {
                        top[u] = fmaxf(top[u], __shfl_xor_sync(0xFFFFFFFFu, top[u], 1));
                        top[u] = fmaxf(top[u], __shfl_xor_sync(0xFFFFFFFFu, top[u], 2));
                    }
                    const bool moves[2] = {top[0] > kRowsSlack || (m[mt][0] == -INFINITY && top[0] > -INFINITY),
                                           top[1] > kRowsSlack || (m[mt][1] == -INFINITY && top[1] > -INFINITY)};
                    if (__any_sync(0xFFFFFFFFu, moves[0] || moves[1])) {
                        float f[2], by[2];
#pragma unroll
                        for (int u = 0; u < kU; ++u) {
                            by[u] = moves[u] ? ceilf(top[u]) : 0.0f;
                            f[u] = !moves[u] ? 1.0f : m[mt][u] == -INFINITY ? 0.0f : ex2_approx(-by[u]);
                            if (moves[u]) m[mt][u] = (m[mt][u] == -INFINITY ? 0.0f : m[mt][u]) + by[u];
                            l[mt][u] = times_power(l[mt][u], -by[u]);   // (0 before anything has been seen)
                        }
#pragma unroll
                        for (int n = 0; n < 4; ++n)
#pragma unroll
                            for (int e = 0; e < kE; ++e) s[mt][n][e] -= by[e >> 1];
#pragma unroll
                        for (int j = 0; j < kTilesN; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[mt][j][e] *= f[kAbove ? 0 : e >> 1];
                    }
                    if (wide) {
#pragma unroll
                        for (int n = 0; n < 4; ++n)
#pragma unroll
                            for (int e = 0; e < kE; ++e) l[mt][e >> 1] += ex2_approx(s[mt][n][e] + (kSumLift - vlog[n >> 1])) * kSumUnlift;
                    }
                    float sum[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
#pragma unroll
                        for (int e = 0; e < kE; ++e) {
                            s[mt][n][e] = ex2_approx(s[mt][n][e]);
                            sum[n >> 1][e >> 1] += s[mt][n][e];
                        }
                        pf[mt][n][0] = pack_half2(s[mt][n][0], s[mt][n][1]);
                        if (!kAbove) pf[mt][n][1] = pack_half2(s[mt][n][2], s[mt][n][3]);
                        if (kAbove) {
                            const float2 x = unpack_half2(pf[mt][n][0]);
                            pf[mt][n][1] = pack_half2(s[mt][n][0] - x.x, s[mt][n][1] - x.y);
                        }
                        if (kRest == kRestApart) {
                            const float2 x = unpack_half2(pf[mt][n][0]), y = unpack_half2(pf[mt][n][1]);
                            rest[mt][n][0] = pack_half2(s[mt][n][0] - x.x, s[mt][n][1] - x.y);
                            rest[mt][n][1] = pack_half2(s[mt][n][2] - y.x, s[mt][n][3] - y.y);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < kU; ++u)
#pragma unroll
                        for (int h2 = 0; h2 < 2; ++h2)   // (a page none of whose tokens the row sees adds nothing, whatever its scale)
                            l[mt][u] += sum[h2][u] == 0.0f || wide ? 0.0f : sum[h2][u] * vinv[h2];
                }
                // ---- O += P V: 16 tokens at a time
#pragma unroll
                for (int k16 = 0; k16 < 2; ++k16) {
                    uint32_t vw[4][kValueBytes / 4 > 0 ? kValueBytes / 4 : 1];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t r = k16 * 16 + (i >> 1) * 8 + 2 * t4 + (i & 1);
                        uint32_t from = tile_at + Cfg::kCodes;
                        if constexpr (H == 128) from += value_chunk<H>(r, g);
                        else if constexpr (H == 64) from += value_chunk<H>(r, g >> 1) + (g & 1u) * 8;
                        else from += r * H + g * kValueBytes;
                        ld_codes<kValueBytes>(from, vw[i]);
                    }
#pragma unroll
                    for (int w = 0; w < (kValueBytes + 3) / 4; ++w) {
                        // byte j of the words of two tokens side by side -> one register of fp16 pairs a dimension
                        uint32_t b0[4], b1[4];
                        e4m3x4_to_half2(__byte_perm(vw[0][w], vw[1][w], 0x5140), b0[0], b0[1]);
                        e4m3x4_to_half2(__byte_perm(vw[2][w], vw[3][w], 0x5140), b1[0], b1[1]);
                        if constexpr (kValueBytes >= 4) {
                            e4m3x4_to_half2(__byte_perm(vw[0][w], vw[1][w], 0x7362), b0[2], b0[3]);
                            e4m3x4_to_half2(__byte_perm(vw[2][w], vw[3][w], 0x7362), b1[2], b1[3]);
                        }
#pragma unroll
                        for (int j = 0; j < (kValueBytes < 4 ? kValueBytes : 4); ++j)
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                const uint32_t a[4] = {pf[mt][2 * k16][0], pf[mt][2 * k16][1], pf[mt][2 * k16 + 1][0], pf[mt][2 * k16 + 1][1]};
                                mma_m16n8k16(o[mt][4 * w + j], a, b0[j], b1[j]);
                                if (kRest == kRestApart) {
                                    const uint32_t r[4] = {rest[mt][2 * k16][0], rest[mt][2 * k16][1], rest[mt][2 * k16 + 1][0], rest[mt][2 * k16 + 1][1]};
                                    mma_m16n8k16(o[mt][4 * w + j], r, b0[j], b1[j]);
                                }
                            }
                    }
                }
            }
            __syncwarp();   // the stage may be filled again
        }
        cp_async_wait_all();

        // ---- the four warps' sums together, through the ring's memory
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                l[mt][u] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][u], 1);
                l[mt][u] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][u], 2);
                if (t4 == 0) s_ml[warp * Cfg::kRows + mt * 16 + u * 8 + g] = make_float2(m[mt][u], l[mt][u]);
            }
        __syncthreads();   // every warp has read its last stage
        if (tid < kRowsWarps * Cfg::kRows) {   // the warps' row sums, against the largest M of a row (which is read from the other half of the entries)
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, s_ml[w * Cfg::kRows + tid % Cfg::kRows].x);
            s_ml[tid].y = times_power(s_ml[tid].y, s_ml[tid].x - top);
        }
        float* const area = reinterpret_cast<float*>(smem) + warp * (Cfg::kRows * H);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const uint32_t r = mt * 16 + u * 8 + g;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, s_ml[w * Cfg::kRows + r].x);
                const float f = m[mt][u] == -INFINITY ? 0.0f : ex2_approx(m[mt][u] - top);
                // n-tile j, column 2 t4 + e: dimension (2 t4 + e) * kTilesN + j
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < kTilesN; j += 2) {
                        const uint32_t d = (2 * t4 + e) * kTilesN + j;
                        float2* const to = reinterpret_cast<float2*>(area + r * H + (d ^ (H >= 64 ? (g & 3u) * 2 : 0u)));
                        if (kAbove) *to = make_float2((o[mt][j][e] + o[mt][j][2 + e]) * f, (o[mt][j + 1][e] + o[mt][j + 1][2 + e]) * f);
                        else *to = make_float2(o[mt][j][2 * u + e] * f, o[mt][j + 1][2 * u + e] * f);
                    }
            }
        __syncthreads();
        const bool alone = s_now[3] != 0;
        for (uint32_t i = tid; i < n_rows * (H / 2); i += kThreads) {
            const uint32_t r = i / (H / 2), d = 2 * (i % (H / 2));
            float top = -INFINITY, sum = 0.0f;
            float2 x = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, s_ml[w * Cfg::kRows + r].x);
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                sum += s_ml[w * Cfg::kRows + r].y;
                const float2 y = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(smem) + (w * Cfg::kRows + r) * H +
                                                                  (d ^ (H >= 64 ? (r & 3u) * 2 : 0u)));
                x.x += y.x, x.y += y.y;
            }
            if (alone) {
                const uint32_t t = (row0 + r) / p.group, h = head * p.group + (row0 + r) % p.group;
                const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
                if (!FA_CACHE_OK(p.c.status, kDbgRow, b < p.s.B && t < p.s.T && h < p.c.heads * p.group)) continue;
                uint8_t* const to = p.y + ((static_cast<uint64_t>(b) * p.s.T + t) * (p.c.heads * p.group) + h) * (2 * H) + 2 * d;
                *reinterpret_cast<uint32_t*>(to) = pack_16(x.x * f, x.y * f, bf16);
            } else {
                const uint32_t s_at = s_now[5];
                if (!FA_CACHE_OK(p.c.status, kDbgScratch, s_at < p.slots)) continue;
                *reinterpret_cast<float2*>(p.part_o + (static_cast<uint64_t>(s_at) * Cfg::kRows + r) * H + d) = x;
                if (d == 0) p.part_ml[static_cast<uint64_t>(s_at) * Cfg::kRows + r] = make_float2(top, sum);
            }
        }
        if (tid == 0 && s_now[2] == 0 && p.min_units != 0 && FA_CACHE_OK(p.c.status, kDbgScratch, static_cast<uint64_t>(b) * per_seq + s_now[10] < p.problems)) {   // who has a share of the problem, for fa_cache_join
            p.shares[static_cast<uint64_t>(b) * per_seq + s_now[10]] = make_int2(alone ? -1 : static_cast<int>(s_now[5]), static_cast<int>(share_owner(s_share, s_now[4])));
        }
        unit = s_now[6], unit_end = s_now[7], before = s_now[8], b = s_now[9];
        first_segment = false;
        __syncthreads();   // the sums have been read: the ring, the rows' data and the fragments may be written again
    }
}

#ifdef FA_DEBUG
__device__ __forceinline__ bool share_inside(const RowsArgs& p, uint64_t index, int2 share) {
    return index < p.problems && share.y >= 0 && static_cast<uint32_t>(share.x) <= 2u * static_cast<uint32_t>(share.y) + 1u && 2ull * static_cast<uint32_t>(share.y) < p.slots;
}
#endif
// Puts the parts of divided problems together: a CTA per problem and row, a warp per part in turn, several parts in flight.
constexpr int kJoinWarps = 8;
template <int H, int MT>
__global__ void __launch_bounds__(kJoinWarps * 32) fa_cache_join(const RowsArgs p) {
    constexpr int kRows = 16 * MT, kThreads = kJoinWarps * 32;
    constexpr int kWide = H >= 64 ? H / 32 : 2;   // dimensions of a lane
    __shared__ __align__(16) float s_o[kJoinWarps][H];
    __shared__ float s_top[kJoinWarps], s_sum[kJoinWarps], s_f[kThreads];
    grid_dep_wait();
    grid_dep_launch();
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint64_t index = blockIdx.x / p.rows;
    const uint32_t r = blockIdx.x % p.rows;
    const int2 share = p.shares[index];
    if (share.x < 0 || !FA_CACHE_OK(p.c.status, kDbgScratch, share_inside(p, index, share))) return;
    const uint32_t per_seq = p.c.heads * p.row_tiles;
    const uint32_t b = static_cast<uint32_t>(index / per_seq), problem = static_cast<uint32_t>(index % per_seq);
    const uint32_t head = problem / p.row_tiles, row = problem % p.row_tiles * p.rows + r;
    if (row >= p.s.T * p.group) return;
    const uint32_t first = static_cast<uint32_t>(share.x), last = 2 * static_cast<uint32_t>(share.y);   // slots: first, then the even ones behind it
    const uint32_t n = (last - (first & ~1u)) / 2 + 1;
    auto slot = [&](uint32_t i) { return static_cast<uint64_t>(i == 0 ? first : (first & ~1u) + 2 * i) * kRows + r; };
    float top = -INFINITY, sum = 0.0f, x[kWide];
#pragma unroll
    for (int d = 0; d < kWide; ++d) x[d] = 0.0f;
    for (uint32_t i0 = 0; i0 < n; i0 += kThreads) {   // (more than one turn only where a problem has more parts than threads)
        const uint32_t i = i0 + tid;
        const float2 ml = i < n ? p.part_ml[slot(i)] : make_float2(-INFINITY, 0.0f);
        float mine = ml.x;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) mine = fmaxf(mine, __shfl_xor_sync(0xFFFFFFFFu, mine, d));
        if (i0 > 0) __syncthreads();
        if (lane == 0) s_top[warp] = mine;
        __syncthreads();
        float now = top;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) now = fmaxf(now, s_top[w]);
        const float f = ml.x == -INFINITY ? 0.0f : ex2_approx(ml.x - now);
        const float again = top == now || top == -INFINITY ? 1.0f : ex2_approx(top - now);   // for what the turns before have added up
        s_f[tid] = f;
        sum = times_power(sum, top - now) + times_power(ml.y, ml.x - now);
#pragma unroll
        for (int d = 0; d < kWide; ++d) x[d] *= again;
        top = now;
        __syncthreads();
        const uint32_t here = min(n - i0, static_cast<uint32_t>(kThreads));
        if (lane * kWide < H)
#pragma unroll 4
            for (uint32_t k = warp; k < here; k += kJoinWarps) {
                const float* const from = p.part_o + slot(i0 + k) * H + lane * kWide;
                const float fk = s_f[k];
                if constexpr (kWide == 4) {
                    const float4 y = *reinterpret_cast<const float4*>(from);
                    x[0] += y.x * fk, x[1] += y.y * fk, x[2] += y.z * fk, x[3] += y.w * fk;
                } else {
                    const float2 y = *reinterpret_cast<const float2*>(from);
                    x[0] += y.x * fk, x[1] += y.y * fk;
                }
            }
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (lane == 0) s_sum[warp] = sum;
    if (lane * kWide < H)
#pragma unroll
        for (int d = 0; d < kWide; ++d) s_o[warp][lane * kWide + d] = x[d];
    __syncthreads();
    if (tid < H / 2) {
        const uint32_t d = 2 * tid;
        float total = 0.0f, lo = 0.0f, hi = 0.0f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) total += s_sum[w], lo += s_o[w][d], hi += s_o[w][d + 1];
        const float f = total == 0.0f ? 0.0f : 1.0f / total;
        const uint32_t t = row / p.group, h = head * p.group + row % p.group;
        uint8_t* const to = p.y + ((static_cast<uint64_t>(b) * p.s.T + t) * (p.c.heads * p.group) + h) * (2 * H) + 2 * d;
        *reinterpret_cast<uint32_t*>(to) = pack_16(lo * f, hi * f, p.bf16 != 0);
    }
}

// The same for problems of few parts: a warp per problem and row.
template <int H, int MT>
__global__ void __launch_bounds__(kJoinWarps * 32) fa_cache_join_few(const RowsArgs p) {
    constexpr int kRows = 16 * MT;
    constexpr int kWide = H >= 64 ? H / 32 : 2;   // dimensions of a lane
    grid_dep_wait();
    grid_dep_launch();
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * kJoinWarps + (threadIdx.x >> 5);
    const uint32_t per_seq = p.c.heads * p.row_tiles, r = static_cast<uint32_t>(at % p.rows);
    const uint64_t index = at / p.rows;
    if (index >= static_cast<uint64_t>(p.s.B) * per_seq) return;
    const int2 share = p.shares[index];
    if (share.x < 0 || !FA_CACHE_OK(p.c.status, kDbgScratch, share_inside(p, index, share))) return;
    const uint32_t b = static_cast<uint32_t>(index / per_seq), problem = static_cast<uint32_t>(index % per_seq);
    const uint32_t head = problem / p.row_tiles, row = problem % p.row_tiles * p.rows + r;
    if (row >= p.s.T * p.group) return;
    const uint32_t first = static_cast<uint32_t>(share.x), last = 2 * static_cast<uint32_t>(share.y);
    const uint32_t n = (last - (first & ~1u)) / 2 + 1;
    auto slot = [&](uint32_t i) { return static_cast<uint64_t>(i == 0 ? first : (first & ~1u) + 2 * i) * kRows + r; };
    float top = -INFINITY, sum = 0.0f, x[kWide];
#pragma unroll
    for (int d = 0; d < kWide; ++d) x[d] = 0.0f;
    for (uint32_t i0 = 0; i0 < n; i0 += 32) {
        const float2 ml = i0 + lane < n ? p.part_ml[slot(i0 + lane)] : make_float2(-INFINITY, 0.0f);
        float now = fmaxf(top, ml.x);
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) now = fmaxf(now, __shfl_xor_sync(0xFFFFFFFFu, now, d));
        const float f = ml.x == -INFINITY ? 0.0f : ex2_approx(ml.x - now);
        const float again = top == now || top == -INFINITY ? 1.0f : ex2_approx(top - now);
        sum = times_power(sum, top - now) + times_power(ml.y, ml.x - now);
#pragma unroll
        for (int d = 0; d < kWide; ++d) x[d] *= again;
        top = now;
        const uint32_t here = min(n - i0, 32u);
#pragma unroll 4
        for (uint32_t k = 0; k < here; ++k) {
            const float fk = __shfl_sync(0xFFFFFFFFu, f, k);
            if (lane * kWide < H) {
                const float* const from = p.part_o + slot(i0 + k) * H + lane * kWide;
                if constexpr (kWide == 4) {
                    const float4 y = *reinterpret_cast<const float4*>(from);
                    x[0] += y.x * fk, x[1] += y.y * fk, x[2] += y.z * fk, x[3] += y.w * fk;
                } else {
                    const float2 y = *reinterpret_cast<const float2*>(from);
                    x[0] += y.x * fk, x[1] += y.y * fk;
                }
            }
        }
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t t = row / p.group, h = head * p.group + row % p.group;
    uint8_t* const to = p.y + ((static_cast<uint64_t>(b) * p.s.T + t) * (p.c.heads * p.group) + h) * (2 * H);
    if (lane * kWide < H)
#pragma unroll
        for (int d = 0; d < kWide; d += 2) *reinterpret_cast<uint32_t*>(to + 2 * (lane * kWide + d)) = pack_16(x[d] * f, x[d + 1] * f, p.bf16 != 0);
}

}  // namespace fa
