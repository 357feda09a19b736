// Attention over the cache of latent vectors, the absorbed form: queries that have been multiplied into the latent space.
//
//   s = scale * (q_latent . c + q_rope . r),  p = softmax(s),  y = sum of p c        for every head, over the same rows (c, r)
//
// Rows of the problem are the query heads of a sequence's tokens (row t * heads + h); a group is N of them (16, 32, 48 or 64) of one
// sequence.  The keys of all sequences, in tiles of 64, are dealt out evenly to `parts` CTAs a group, so that a sequence may be divided:
// its parts leave numerators, maxima and sums in scratch, which fa_latent_join puts together.
//
// Both products are tcgen05 MMAs on the same tile in shared memory, and both are kept transposed: S^T[64 keys, N] = C Q^T, and Y^T[128
// dimensions, N] += C^T P^T.  Keys and dimensions are what an MMA's M is filled with, rows are its N, of which there may be few: four such
// tiles hold 512 dimensions in 4 N columns of tensor memory, where Y[128 rows, 512] would need all 512 columns and leave none for the scores.
// (Measured, clocks an MMA: M = 64 N = 16 or 32 27, N = 64 32; M = 128 N = 16 39, N = 32 40, N = 64 48.)  512 threads:
//
//   warps 0-7    softmax: a warp 16 keys and half of the rows, eight threads a row and 16 keys (tcgen05.ld.16x256b hands out scores that way).
//                All share a row's reference; it is looked at again only where a score exceeds it by more than 2^8, so that a tile passes with
//                no maximum being formed.  P into shared memory; at the end of a segment (a sequence's tiles in this CTA) the division and Y,
//                a thread a dimension
//   warps 8-11   fetch tiles by TMA: 64 keys of 128 dimensions a slot of one ring, of the rotary part a slot of another.  (Four, because what a
//                thread asks of a barrier behind a TMA copy takes 280 clocks: one warp alone brings in a tile of 512 dimensions in 2550)
//   warp 12, 13  issue the MMAs of the scores, of the results.  (One warp for both, as slots arrive: 94 us for 64 sequences of 100 to 8192
//                tokens, 16 rows, where two took 72: a barrier's answer reaches a thread only behind the MMAs that it has queued)
//   warps 14-15  queries into shared memory, a segment ahead; of the first segment the softmax warps do most
//
// Measured: 64 sequences of 100 to 8192 tokens, 16 rows, 64 to 69 us from box to box (306 MB, 4.4 to 4.8 TB/s; steady tiles of 73.7 KB take 2900 to 3000 clocks, the memory's
// share 2830; the rest is the way to the first tile, 4 us, CTAs that the memory serves later than others, 5, and the join); 32 of 1000 to 8192, 128
// rows in two groups, 82 to 90 us (tiles take 3000 clocks where their MMAs take 1920: with 74 KB of queries the ring has two tiles, and what one passes
// through from its slots' asking to their letting go, 5700 clocks, is the bound).
//
// What must not happen: a key that a row does not see reaching it, as 0 * NaN.  Tiles that some row of the group sees in part only (the
// last ones of a sequence) are gone over in shared memory between the two products: keys behind the last that any row sees become zeros;
// a key that some rows see and that holds an infinity or a NaN becomes zeros too, and rows that see it get a weight that is NaN.
#pragma once

#include <cuda.h>

#include "fa_latent.cuh"

namespace fa {

constexpr int kLatentThreads = 512;
constexpr uint32_t kLatentSoftmax = 256;              // threads of the softmax warps
constexpr uint32_t kLatentTile = 64;
constexpr uint32_t kLatentSlot = kLatentTile * 128;   // bytes of 64 keys by 64 dimensions
constexpr float kLatentSlack = 8.0f;                  // the reference moves when an exponent exceeds it by more: weights stay below 2^8
constexpr uint32_t kSeesAll = 0xFFFFFFFFu;

struct LatentRowsArgs {
    LatentView c;
    CacheSeqs s;
    const uint8_t* q_latent;
    const uint8_t* q_rope;
    uint8_t* y;              // [B, T, heads, latent] contiguous
    int64_t ql_b, ql_t, ql_h, qr_b, qr_t, qr_h;   // strides in bytes
    uint32_t heads, rows, groups, group_rows;     // rows: T * heads, in `groups` of group_rows (the last may have fewer)
    uint32_t parts, least;                        // CTAs a group; tiles that one has at least (0: a CTA has a sequence, none is divided)
    uint32_t causal, bf16;
    float scale_log2;        // scale * log2(e)
    float* part_o;           // [parts * groups * 2, N, latent]
    float2* part_ml;         // [parts * groups * 2, N]
    int2* shares;            // [B]: first and last part of a sequence
};

template <int LC, int N>
struct LatentCfg {
    static constexpr int kPairs = LC / 2;                     // of 64-dimension chunks: slots of a tile
    static constexpr int kPitch = N == 16 ? 32 : N == 32 ? 64 : 128;   // bytes of a key's weights: a swizzle span
    static constexpr int kPBuffers = N <= 32 ? 2 : 1;
    static constexpr uint32_t kQChunk = N * 128, kQBytes = (LC + 1) * kQChunk, kPBytes = kLatentTile * kPitch;
    // Slots: what is left of shared memory, three tiles' rotary parts (two, eight) and the rest for the other ring
    static constexpr int kChunks = (229376 - kQBytes - kPBuffers * kPBytes) / kLatentSlot;
    static constexpr int kRopeSlots = LC == 8 ? (kChunks >= 23 ? 3 : 2) : LC == 4 ? 4 : 8;
    static constexpr int kPairSlots = (kChunks - kRopeSlots) / 2 < 12 ? (kChunks - kRopeSlots) / 2 : 12;
    static_assert(kPairSlots >= kPairs && kPairSlots >= 2, "room for a tile");
    static constexpr uint32_t kOffPair = kQBytes, kOffRope = kOffPair + kPairSlots * 2 * kLatentSlot, kOffP = kOffRope + kRopeSlots * kLatentSlot;
    static_assert(kOffPair % 1024 == 0 && kOffP % 1024 == 0 && kPBytes % 1024 == 0, "tiles on swizzle atoms");
    static constexpr uint32_t kTiles = kOffP + kPBuffers * kPBytes;
    static constexpr int kSmemBytes = kTiles + 1024;
    static constexpr uint32_t kColS = kPairs * N, kCols = 512;   // scores of even tiles at kColS, of odd ones N behind
    static_assert(kColS + 2 * N <= 512, "tensor memory");
    // barriers
    static constexpr int FULL = 0, EMPTY = FULL + kPairSlots, RFULL = EMPTY + kPairSlots, REMPTY = RFULL + kRopeSlots, QFULL = REMPTY + kRopeSlots, QEMPTY = QFULL + 1,
                         S = QEMPTY + 1, P = S + 2, PV = P + 2, FINAL = PV + 2, kBarriers = FINAL + 2;
};

// Instruction descriptors (see make_idesc_f16): fp16 or bf16 operands, fp32 sums.
__device__ __forceinline__ uint32_t idesc_16bit(uint32_t m, uint32_t n, bool a_mn, bool b_mn, bool bf16) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// 16 lanes x 8 columns: thread t receives of lane t / 4 (v[0], v[1]) and of lane t / 4 + 8 (v[2], v[3]) columns 2 (t % 4) and the next.
__device__ __forceinline__ void tmem_ld_16x8(uint32_t taddr, float* v) {
    FA_DBG_TMEM(taddr, 8u);
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(taddr) : "memory");
}
// Of warps 0-7: all there, and whether any thread says so.
__device__ __forceinline__ bool softmax_any(bool x) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"(static_cast<uint32_t>(x)) : "memory");
    return r != 0;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); }

// What rows see.  A sequence holds `held` tokens, of the call's T it has `count`, the last of those that it holds.
struct LatentSeq {
    uint32_t held, count;
};
__device__ __forceinline__ LatentSeq latent_seq(const LatentRowsArgs& p, uint32_t b) {
    const CacheView c = plain_view(p.c);
    return LatentSeq{cache_length(c, p.s, b), cache_count(p.s, b)};
}
// Keys [0, ...) that token t sees; 0 also where the sequence does not have it.
__device__ __forceinline__ uint32_t latent_limit(const LatentRowsArgs& p, const LatentSeq& q, uint32_t t) {
    if (t >= q.count) return 0;
    if (!p.causal) return q.held;
    return q.held + t >= q.count ? min(q.held, q.held + t - q.count + 1u) : 0u;
}
// Keys that some row of a group sees (its last token's, of those that the sequence has).
__device__ __forceinline__ uint32_t latent_farthest(const LatentRowsArgs& p, const LatentSeq& q, uint32_t group) {
    if (p.s.T == 1) return q.count == 0 ? 0u : q.held;   // (in front of two divisions that stand in a token's way)
    const uint32_t row0 = group * p.group_rows, t_first = row0 / p.heads, t_last = (min(p.rows, row0 + p.group_rows) - 1u) / p.heads;
    if (t_first >= q.count) return 0;
    return latent_limit(p, q, min(t_last, q.count - 1u));
}
__device__ __forceinline__ uint32_t latent_units(const LatentRowsArgs& p, uint32_t b) {
    const LatentSeq q = latent_seq(p, b);
    return q.count == 0 ? 0u : (q.held + kLatentTile - 1u) / kLatentTile;
}

// A CTA's way through its tiles, segment by segment.  All lanes of a warp.
struct LatentWalk {
    uint32_t unit, unit_end, b, before;   // next tile, end, its sequence, tiles of the sequences in front of that
    uint32_t each, more;
    // the segment at hand: tiles [t0, t1) of sequence `seq`, of which the group sees [t0, end)
    uint32_t seq, t0, t1, end, farthest, first_unit, units;
    bool whole, begins;                   // all of the sequence's tiles; its first among them
    LatentSeq q;
};
__device__ __forceinline__ bool latent_start(const LatentRowsArgs& p, uint32_t part, LatentWalk& w) {
    const uint32_t lane = threadIdx.x & 31u;
    if (p.least == 0) {
        w.unit = w.before = 0, w.b = part, w.each = 1, w.more = 0;
        w.unit_end = latent_units(p, part);
        return w.unit_end != 0;
    }
    uint32_t total = 0, kept = 0;
    for (uint32_t b = lane; b < p.s.B; b += 32) total += kept = latent_units(p, b);
    if (lane >= p.s.B) kept = 0;
    total = __reduce_add_sync(0xFFFFFFFFu, total);
    const uint32_t parts = min(p.parts, (total + p.least - 1u) / p.least);
    if (part >= parts) return false;
    w.each = total / parts, w.more = total - w.each * parts;
    w.unit = part * w.each + min(part, w.more);
    w.unit_end = (part + 1u) * w.each + min(part + 1u, w.more);
    w.before = 0, w.b = 0;
    for (uint32_t b0 = 0; b0 < p.s.B; b0 += 32) {
        const uint32_t mine = p.s.B <= 32 ? kept : b0 + lane < p.s.B ? latent_units(p, b0 + lane) : 0u;
        uint32_t upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += x;
        }
        const uint32_t behind = __ballot_sync(0xFFFFFFFFu, w.before + upto > w.unit);
        if (behind != 0) {
            const uint32_t at = __ffs(behind) - 1;
            w.b = b0 + at;
            w.before += __shfl_sync(0xFFFFFFFFu, upto - mine, at);
            break;
        }
        w.before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    return true;
}
__device__ __forceinline__ uint32_t latent_owner(const LatentWalk& w, uint32_t unit) {
    const uint32_t longer = w.more * (w.each + 1u);
    return unit < longer ? unit / (w.each + 1u) : w.more + (unit - longer) / w.each;
}
// False: none is left.
__device__ __forceinline__ bool latent_next(const LatentRowsArgs& p, uint32_t group, LatentWalk& w) {
    while (w.unit < w.unit_end) {
        const LatentSeq q = latent_seq(p, w.b);
        const uint32_t units = q.count == 0 ? 0u : (q.held + kLatentTile - 1u) / kLatentTile;
        if (units == 0) {
            ++w.b;
            continue;
        }
        w.q = q, w.seq = w.b, w.first_unit = w.before, w.units = units;
        w.t0 = w.unit - w.before;
        w.t1 = min(units, w.unit_end - w.before);
        w.begins = w.t0 == 0, w.whole = w.begins && w.t1 == units;
        w.farthest = latent_farthest(p, q, group);
        w.end = max(w.t0, min(w.t1, (w.farthest + kLatentTile - 1u) / kLatentTile));
        w.unit = w.before + w.t1;
        if (w.t1 == units) w.before += units, ++w.b;
        return true;
    }
    return false;
}

// 16 bytes of eight 16-bit values: whether one is an infinity or a NaN.
__device__ __forceinline__ bool not_finite(const uint32_t (&w)[4], bool bf16) {
    const uint32_t mask = bf16 ? 0x7F80u : 0x7C00u;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (w[i] & mask) == mask || (w[i] >> 16 & mask) == mask;
    return bad;
}

template <int LC, int N>
__global__ void __launch_bounds__(kLatentThreads, 1) fa_latent_rows(const __grid_constant__ CUtensorMap map, const LatentRowsArgs p) {
    using C = LatentCfg<LC, N>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[C::kBarriers];
    // (shared memory is full: what is needed at a segment's end takes the places of what is not any more)
    __shared__ float s_max[4][N], s_alpha[N];
    __shared__ uint32_t s_limit[N];
    float (&s_sum)[4][N] = s_max;
    float (&s_m)[N] = s_alpha;
    float* const s_l = reinterpret_cast<float*>(s_limit);
    __shared__ uint32_t s_absent[16];        // of tile g in entry g % 16 (more than the ring has tiles): its 16-key groups without a page
    __shared__ uint32_t s_bad[2][2];         // of the partly seen tile n in entry n % 2: keys that hold no finite numbers
    __shared__ uint32_t tmem_slot, abort_flag;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    auto pair_addr = [&](uint32_t n) { return base + C::kOffPair + (n % C::kPairSlots) * (2 * kLatentSlot); };
    auto rope_addr = [&](uint32_t n) { return base + C::kOffRope + (n % C::kRopeSlots) * kLatentSlot; };
    auto p_addr = [&](uint32_t g) { return base + C::kOffP + (g % C::kPBuffers) * C::kPBytes; };
    const WaitCtl ctl{p.c.status, &abort_flag, kWaitCapCycles, nullptr, 0};
    const uint32_t group = blockIdx.x % p.groups, part = blockIdx.x / p.groups;
    const uint32_t row0 = group * p.group_rows, n_rows = min(p.group_rows, p.rows - row0);
    const bool bf16 = p.bf16 != 0;

    if (tid == 0) {
        for (int i = 0; i < C::kBarriers; ++i) mbar_init(bar(i), i == C::QFULL ? 64u : i >= C::P && i < C::PV ? 8u : 1u);
        abort_flag = 0;
        fence_mbar_init();
        prefetch_tensormap(&map);
    }
    if (tid < 4) s_bad[tid >> 1][tid & 1] = 0;
#ifdef FA_DEBUG
    if (tid == 0) {
        g_dbg.smem_lo = base, g_dbg.smem_hi = base + C::kTiles, g_dbg.F = p.c.latent + p.c.rope, g_dbg.L = p.c.page, g_dbg.B = p.c.n_pages + 1;
        g_dbg.tmem_base = 0, g_dbg.tmem_cols = 512, g_dbg.ctl = ctl;
    }
    FA_CACHE_POISON(base, C::kTiles);
    fence_proxy_async_smem();
#endif
    if (warp == 12) {
        tmem_alloc(smem_u32(&tmem_slot), C::kCols);
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

    // Rows [0, rows) of a sequence's queries, as thread `who` of `of` (a multiple of 64; rows that are not there: zeros).
    auto copy_queries = [&](uint32_t seq, uint32_t who, uint32_t of, uint32_t rows) {
        auto copy = [&](const uint8_t* from, int64_t t_stride, int64_t h_stride, uint32_t pieces, uint32_t to) {   // `pieces` of 16 bytes each: a power of two, 64 at most
            const uint32_t j = who & (pieces - 1u), step = of / pieces;
            uint32_t r = who / pieces, t = (row0 + r) / p.heads, h = row0 + r - t * p.heads;
            const uint32_t chunk = to + (j >> 3) * C::kQChunk;
#pragma unroll 4
            for (; r < rows; r += step) {
                const bool in = r < n_rows && FA_CACHE_OK(p.c.status, kDbgRow, seq < p.s.B && t < p.s.T && h < p.heads);
                cp_async_16_zero(chunk + r * 128 + (((j & 7u) ^ (r & 7u)) << 4), in ? from + t * t_stride + h * h_stride + 16 * j : from, in);
                for (h += step; h >= p.heads; h -= p.heads) ++t;
            }
        };
        copy(p.q_latent + seq * p.ql_b, p.ql_t, p.ql_h, 8 * LC, base);
        copy(p.q_rope + seq * p.qr_b, p.qr_t, p.qr_h, p.c.rope / 8, base + LC * C::kQChunk);
    };

    LatentWalk w;
    const bool any = latent_start(p, part, w) && latent_next(p, group, w);   // (the first segment is worked out by all roles together: one way through the code)
    if (warp < 8) {
        // ---------------------------------------------------------------- softmax
        const uint32_t lanes = warp & 3u, side = warp >> 2, lane_off = (lanes * 32u) << 16;
        // this thread's keys of a tile: key_a and key_a + 8; its rows: first + 8 j + 2 quad + e
        const uint32_t quad = lane & 3u, key_a = 16 * lanes + lane / 4, first = side * (N / 2);
        constexpr int kBlocks = N / 16;
        uint32_t g = 0, partly = 0;
        bool helped = false;   // with the first segment's queries
        for (uint32_t b = part; b < p.s.B; b += p.parts) {   // sequences without tokens
            if (latent_units(p, b) != 0) continue;
            if (group == 0 && tid == 0 && !cache_length_ok(plain_view(p.c), p.s, b)) cache_report(p.c.status, kCacheBadPosition);
            uint8_t* const to = p.y + (static_cast<uint64_t>(b) * p.rows + row0) * (128 * LC);
            for (uint32_t i = tid; i < n_rows * (8 * LC); i += kLatentSoftmax) *reinterpret_cast<uint4*>(to + 16 * i) = make_uint4(0, 0, 0, 0);
        }
        for (bool more = any; more; more = latent_next(p, group, w)) {
            if (!helped && w.end > w.t0) {
                copy_queries(w.seq, tid, kLatentSoftmax + 64u, N);
                cp_async_wait_all();
                fence_proxy_async_smem();
                asm volatile("barrier.cta.arrive 2, 320;" ::: "memory");
                helped = true;
            }
            if (group == 0 && w.begins && tid == 0)
                p.shares[w.seq] = make_int2(static_cast<int>(part), static_cast<int>(latent_owner(w, w.first_unit + w.units - 1u)));
            if (tid < N) {   // (what becomes of a row that sees nothing is not used)
                const uint32_t x = tid < n_rows ? latent_limit(p, w.q, p.s.T == 1 ? 0u : (row0 + tid) / p.heads) : 0u;
                s_limit[tid] = x == 0 ? kSeesAll : x;
            }
            float m[2 * kBlocks], l[2 * kBlocks];
#pragma unroll
            for (int i = 0; i < 2 * kBlocks; ++i) m[i] = -INFINITY, l[i] = 0.0f;
            // keys that all rows see that see any: up to the first row's
            uint32_t least = p.s.T == 1 ? w.farthest : latent_limit(p, w.q, row0 / p.heads);
            if (least == 0) {   // (tokens in front of the first key: found by every thread, rows are few)
                least = w.farthest;
                for (uint32_t t = row0 / p.heads; t <= (row0 + n_rows - 1u) / p.heads; ++t) {
                    const uint32_t x = latent_limit(p, w.q, t);
                    if (x != 0) {
                        least = x;
                        break;
                    }
                }
            }
            softmax_sync();   // s_limit
            for (uint32_t tile = w.t0; tile < w.end; ++tile, ++g) {
                const uint32_t key0 = tile * kLatentTile;
                mbar_wait(bar(C::S + (g & 1u)), (g >> 1) & 1u, ctl, kCacheTimeout | C::S);
                tc_fence_after();
                __syncwarp();
                float s[4 * kBlocks];
#pragma unroll
                for (int j = 0; j < kBlocks; ++j) tmem_ld_16x8(tmem + lane_off + C::kColS + N * (g & 1u) + first + 8 * j, s + 4 * j);
                // (the first slot's barrier: what the fetching warp has written about this tile is there)
                mbar_wait(bar(C::FULL + g * C::kPairs % C::kPairSlots), (g * C::kPairs / C::kPairSlots) & 1u, ctl, kCacheTimeout | C::FULL);
                const uint32_t absent = *reinterpret_cast<volatile uint32_t*>(&s_absent[g & 15u]);
                tmem_wait_ld();
                if (key0 + kLatentTile > least || absent != 0) {
                    uint32_t bad_lo = 0, bad_hi = 0;
                    if (key0 + kLatentTile > least) {
                        // four threads a key: pieces of 16 bytes, two of each 64 dimensions
                        const uint32_t key = tid >> 2, part4 = tid & 3u, at = key0 + key, swz = key & 7u;
                        const bool behind = at >= w.farthest, some = !behind && at >= least;
                        bool bad = false;
#pragma unroll
                        for (int c = 0; c < C::kPairs; ++c) mbar_wait(bar(C::FULL + (g * C::kPairs + c) % C::kPairSlots), ((g * C::kPairs + c) / C::kPairSlots) & 1u, ctl, kCacheTimeout | C::FULL);
                        auto piece = [&](uint32_t c, uint32_t j) {
                            return pair_addr(g * C::kPairs + c / 2) + (c & 1u) * kLatentSlot + key * 128 + (((2 * part4 + j) ^ swz) << 4);
                        };
                        if (some)
#pragma unroll 1
                            for (uint32_t c = 0; c < 2 * LC; ++c) {
                                uint32_t x[4];
                                ld_shared_v4(piece(c >> 1, c & 1u), x);
                                bad |= not_finite(x, bf16);
                            }
                        bad |= __shfl_xor_sync(0xFFFFFFFFu, bad, 1) != 0;
                        bad |= __shfl_xor_sync(0xFFFFFFFFu, bad, 2) != 0;
                        if (behind || bad)
#pragma unroll 1
                            for (uint32_t c = 0; c < 2 * LC; ++c) st_shared_v4(piece(c >> 1, c & 1u), 0, 0, 0, 0);
                        if (bad && part4 == 0) atomicOr(&s_bad[partly & 1u][key >> 5], 1u << (key & 31u));
                        fence_proxy_async_smem();
                        softmax_sync();
                        bad_lo = *reinterpret_cast<volatile uint32_t*>(&s_bad[partly & 1u][0]);
                        bad_hi = *reinterpret_cast<volatile uint32_t*>(&s_bad[partly & 1u][1]);
                        ++partly;
                        // (the other entry was last read two barriers ago)
                        if (tid < 2) s_bad[partly & 1u][tid] = 0;
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        const uint32_t key = key_a + 8 * i, at = key0 + key;
                        const bool gone = (absent >> (key >> 4) & 1u) || at >= w.farthest, bad = (key < 32 ? bad_lo >> key : bad_hi >> (key - 32)) & 1u;
#pragma unroll
                        for (uint32_t j = 0; j < kBlocks; ++j) {
#pragma unroll
                            for (uint32_t e = 0; e < 2; ++e) {
                                if (gone || at >= s_limit[first + 8 * j + 2 * quad + e]) s[4 * j + 2 * i + e] = -INFINITY;
                                else if (bad) s[4 * j + 2 * i + e] = __int_as_float(0x7FC00000);
                            }
                        }
                    }
                }
                // ---- whether some score asks for another reference
                bool above = tile == w.t0;
                if (!above) {
#pragma unroll
                    for (int j = 0; j < kBlocks; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            above |= fmaxf(s[4 * j + e], s[4 * j + 2 + e]) * p.scale_log2 > (m[2 * j + e] == -INFINITY ? -INFINITY : m[2 * j + e] + kLatentSlack);
                    above = softmax_any(above);
                }
                if (above) {   // the largest score of every row; a new reference where it exceeds the old one by too much
#pragma unroll
                    for (int j = 0; j < kBlocks; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = fmaxf(s[4 * j + e], s[4 * j + 2 + e]);
#pragma unroll
                            for (int d = 4; d <= 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
                            if (lane < 4) s_max[lanes][first + 8 * j + 2 * quad + e] = top;
                        }
                    softmax_sync();
#pragma unroll
                    for (int j = 0; j < kBlocks; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t r = first + 8 * j + 2 * quad + e;
                            const float top = fmaxf(fmaxf(s_max[0][r], s_max[1][r]), fmaxf(s_max[2][r], s_max[3][r])) * p.scale_log2;
                            float alpha = 1.0f;
                            if (top > (m[2 * j + e] == -INFINITY ? -INFINITY : m[2 * j + e] + kLatentSlack)) {
                                alpha = ex2_approx(m[2 * j + e] - top);
                                m[2 * j + e] = top;
                                l[2 * j + e] *= alpha;
                            }
                            if (lanes == 0 && lane < 4) s_alpha[r] = alpha;
                        }
                    softmax_sync();
                    if (tile > w.t0) {   // rows are columns of Y^T: every warp multiplies all of them, in its dimensions, its side every other 16 columns
                        mbar_wait(bar(C::PV + ((g - 1u) & 1u)), ((g - 1u) >> 1) & 1u, ctl, kCacheTimeout | C::PV);
                        tc_fence_after();
                        __syncwarp();
#pragma unroll 1
                        for (uint32_t c = 16 * side; c < C::kPairs * N; c += 32) {
                            float o[16];
                            uint32_t x[16];
                            tmem_ld16(tmem + lane_off + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (uint32_t e = 0; e < 16; ++e) x[e] = __float_as_uint(o[e] * s_alpha[c % N + e]);
                            tmem_st16(tmem + lane_off + c, x);
                        }
                        tmem_wait_st();
                    }
                }
                // the last P V that read this buffer of P
                if (g >= C::kPBuffers) {
                    const uint32_t h = g - C::kPBuffers;
                    mbar_wait(bar(C::PV + (h & 1u)), (h >> 1) & 1u, ctl, kCacheTimeout | C::PV);
                }
                // ---- weights, rounded to the rows' type: an MMA takes one type of both operands, and a second product for what that takes away
                // would double P V.  (The result is off by 1.2 times its own rounding)
                uint32_t pk[2 * kBlocks];
#pragma unroll
                for (uint32_t j = 0; j < kBlocks; ++j) {
                    const float r0 = m[2 * j] == -INFINITY ? 0.0f : m[2 * j], r1 = m[2 * j + 1] == -INFINITY ? 0.0f : m[2 * j + 1];
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        pk[2 * j + i] = pack_16(ex2_approx(fmaf(s[4 * j + 2 * i], p.scale_log2, -r0)), ex2_approx(fmaf(s[4 * j + 2 * i + 1], p.scale_log2, -r1)), bf16);
                        const uint32_t row = key_a + 8 * i;
                        st_shared_u32(p_addr(g) + row * C::kPitch + (((first / 8 + j) ^ (row * C::kPitch >> 7 & (C::kPitch / 16 - 1))) << 4) + 4 * quad, pk[2 * j + i]);
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(C::P + (g & 1u)));
                // sums of the weights as they are rounded
#pragma unroll
                for (int j = 0; j < kBlocks; ++j) {
                    const float2 x = unpack_16(pk[2 * j], bf16), y = unpack_16(pk[2 * j + 1], bf16);
                    l[2 * j] += x.x + y.x;
                    l[2 * j + 1] += x.y + y.y;
                }
            }
            // ---- the segment's end
            softmax_sync();   // (s_alpha, s_limit are not read any more)
#pragma unroll
            for (int j = 0; j < kBlocks; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = l[2 * j + e];
#pragma unroll
                    for (int d = 4; d <= 16; d <<= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
                    if (lane < 4) s_sum[lanes][first + 8 * j + 2 * quad + e] = x;
                    if (lanes == 0 && lane < 4) s_m[first + 8 * j + 2 * quad + e] = m[2 * j + e];
                }
            softmax_sync();
            if (tid < N) {
                const float x = (s_sum[0][tid] + s_sum[1][tid]) + (s_sum[2][tid] + s_sum[3][tid]);
                const bool none = s_limit[tid] == kSeesAll || x == 0.0f;
                s_l[tid] = none ? 0.0f : w.whole ? 1.0f / x : x;
                if (none) s_m[tid] = -INFINITY;
            }
            const bool tiles = w.end > w.t0;
            if (tiles) {
                mbar_wait(bar(C::PV + ((g - 1u) & 1u)), ((g - 1u) >> 1) & 1u, ctl, kCacheTimeout | C::PV);
                tc_fence_after();
            }
            softmax_sync();
            const uint32_t slot = 2u * blockIdx.x + (w.begins ? 1u : 0u);
            if (!w.whole && tid < n_rows) p.part_ml[static_cast<uint64_t>(slot) * N + tid] = make_float2(s_m[tid], s_l[tid]);
            const bool inside = w.whole ? FA_CACHE_OK(p.c.status, kDbgRow, w.seq < p.s.B && row0 + n_rows <= p.rows) : FA_CACHE_OK(p.c.status, kDbgScratch, slot < 2u * p.parts * p.groups);
            if ((tiles || w.whole) && inside) {
#pragma unroll 1
                for (uint32_t c = 16 * side; c < C::kPairs * N; c += 32) {
                    float o[16];
                    if (tiles) {
                        tmem_ld16(tmem + lane_off + c, o);
                        tmem_wait_ld();
                    }
                    const uint32_t r0 = c % N, d = c / N * 128 + lanes * 32 + lane;
                    if (w.whole) {
                        uint8_t* const to = p.y + ((static_cast<uint64_t>(w.seq) * p.rows + row0 + r0) * (64 * LC) + d) * 2;
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e) {
                            const float f = s_l[r0 + e];
                            const uint32_t x = f == 0.0f ? 0u : pack_16(o[e] * f, 0.0f, bf16);
                            if (r0 + e < n_rows) *reinterpret_cast<uint16_t*>(to + e * (2 * 64 * LC)) = static_cast<uint16_t>(x);
                        }
                    } else {
                        float* const to = p.part_o + (static_cast<uint64_t>(slot) * N + r0) * (64 * LC) + d;
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e)
                            if (r0 + e < n_rows) to[e * (64 * LC)] = o[e];
                    }
                }
            }
            tc_fence_before();
            softmax_sync();   // s_l and s_m are read
        }
    } else if (warp < 12) {
        // ---------------------------------------------------------------- tiles: 128 dimensions of each, the last warp the rotary part too
        const bool rear = warp == 11;
        const uint32_t c_first = min(warp - 8u, static_cast<uint32_t>(C::kPairs)), c_end = min(warp - 7u, static_cast<uint32_t>(C::kPairs));
        const bool leader = elect_one();
        const uint32_t per_tile = p.c.page < kLatentTile ? kLatentTile >> p.c.page_shift : 1u;   // pages of a tile
        const uint32_t box_rows = min(p.c.page, kLatentTile), box_bytes = box_rows * 128;
        uint32_t g = 0, reports = 0, asked = 0;   // (asked: slots with a copy under way or done, up to this tile's)
        bool ok = true;
        for (bool more = any; ok && more; more = latent_next(p, group, w)) {
            const int32_t* const table = p.s.table + w.seq * p.s.table_stride;
            if (warp == 8 && w.begins && group == 0 && lane == 0 && !cache_length_ok(plain_view(p.c), p.s, w.seq)) cache_report(p.c.status, kCacheBadPosition);
            const uint32_t blocks = (w.q.held + p.c.page - 1u) >> p.c.page_shift;
            uint32_t known = 0, from = 0;   // entries [from, from + known) are in the lanes
            int32_t entry = -1;
            for (uint32_t tile = w.t0; ok && tile < w.end; ++tile, ++g) {
                const uint32_t key0 = tile * kLatentTile, first = key0 >> p.c.page_shift;
                if (known == 0 || first + per_tile > from + known) {
                    from = first, known = 32;
                    entry = from + lane < blocks && FA_CACHE_OK(p.c.status, kDbgEntry, w.seq < p.s.B && from + lane < p.s.width) ? table[from + lane] : -1;
                    const bool wrong = from + lane < blocks && static_cast<uint32_t>(entry) >= p.c.n_pages && (from + lane) * p.c.page < w.end * kLatentTile;
                    if (wrong && warp == 8) ++reports;
                    if (static_cast<uint32_t>(entry) >= p.c.n_pages) entry = static_cast<int32_t>(p.c.n_pages);   // outside: TMA fills with zeros
                }
                uint32_t gone = 0;   // a bit for each 16 keys
                for (uint32_t i = 0; i < per_tile; ++i)
                    if (static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, entry, first + i - from)) >= p.c.n_pages) gone |= (per_tile == 1 ? 15u : per_tile == 2 ? 3u : 1u) << (i * (4 / per_tile));
                const uint32_t y = per_tile == 1 ? key0 & (p.c.page - 1u) : 0u;
                if (rear) {   // (its slot is let go of before the others)
                    if (g >= C::kRopeSlots) ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar(C::REMPTY + g % C::kRopeSlots), (g / C::kRopeSlots - 1u) & 1u, ctl, kCacheTimeout | C::REMPTY));
                    if (!ok) break;
                    asked = g + 1;
                    if (leader) mbar_expect_tx(bar(C::RFULL + g % C::kRopeSlots), kLatentSlot);
                    for (uint32_t i = 0; i < per_tile; ++i) {
                        const int32_t page = __shfl_sync(0xFFFFFFFFu, entry, first + i - from);
                        if (leader) tma_load_3d(rope_addr(g) + i * box_bytes, &map, bar(C::RFULL + g % C::kRopeSlots), 64 * LC, static_cast<int32_t>(y), page);
                    }
                }
                for (uint32_t c = c_first; c < c_end; ++c) {
                    const uint32_t n = g * C::kPairs + c;
                    if (n >= C::kPairSlots) ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar(C::EMPTY + n % C::kPairSlots), (n / C::kPairSlots - 1u) & 1u, ctl, kCacheTimeout | C::EMPTY));
                    if (!ok) break;
                    asked = g + 1;
                    if (leader) {
                        if (c == 0) *reinterpret_cast<volatile uint32_t*>(&s_absent[g & 15u]) = gone;
                        mbar_expect_tx(bar(C::FULL + n % C::kPairSlots), 2 * kLatentSlot);
                    }
                    for (uint32_t i = 0; i < per_tile; ++i) {
                        const int32_t page = __shfl_sync(0xFFFFFFFFu, entry, first + i - from);
                        if (leader) {
                            tma_load_3d(pair_addr(n) + i * box_bytes, &map, bar(C::FULL + n % C::kPairSlots), static_cast<int32_t>(128 * c), static_cast<int32_t>(y), page);
                            tma_load_3d(pair_addr(n) + kLatentSlot + i * box_bytes, &map, bar(C::FULL + n % C::kPairSlots), static_cast<int32_t>(128 * c + 64), static_cast<int32_t>(y), page);
                        }
                    }
                }
                if (!ok) break;
                __syncwarp();
            }
        }
        if (reports != 0) cache_report(p.c.status, kCacheBadPage);
        // What was asked for lands before the CTA ends: the MMAs have waited for it, unless a wait gave up.
        if (*ctl.abort_flag != 0u) {
            for (uint32_t tile = asked > C::kPairSlots ? asked - C::kPairSlots : 0; tile < asked; ++tile) {   // (what has landed answers at once)
                for (uint32_t c = c_first; c < c_end; ++c) {
                    const uint32_t n = tile * C::kPairs + c;
                    if (n + C::kPairSlots >= asked * C::kPairs) mbar_wait_certain(bar(C::FULL + n % C::kPairSlots), (n / C::kPairSlots) & 1u, ctl, kCacheTimeout | C::FULL);
                }
                if (rear && tile + C::kRopeSlots >= asked) mbar_wait_certain(bar(C::RFULL + tile % C::kRopeSlots), (tile / C::kRopeSlots) & 1u, ctl, kCacheTimeout | C::RFULL);
            }
        }
    } else if (warp < 14) {
        // ---------------------------------------------------------------- MMAs: scores, results
        const bool leader = elect_one();
        bool ok = true;   // once a wait has given up nothing more is issued
        auto wait = [&](int x, uint32_t parity) { ok &= mbar_wait(bar(x), parity, ctl, kCacheTimeout | static_cast<uint32_t>(x)); };
        const uint32_t idesc_s = idesc_16bit(kLatentTile, N, false, false, bf16), idesc_y = idesc_16bit(128, N, true, true, bf16);
        const uint32_t rope_steps = p.c.rope / 16;
        uint32_t g = 0, k = 0;   // tiles; segments with tiles
        for (bool more = any; more; more = latent_next(p, group, w)) {
            if (w.end == w.t0) continue;
            if (warp == 12) wait(C::QFULL, k & 1u);
            for (uint32_t tile = w.t0; tile < w.end; ++tile, ++g) {
                if (warp == 12) {
                    // (whoever read the scores two tiles ago has given P)
                    if (g >= 2) wait(C::P + (g & 1u), ((g >> 1) - 1u) & 1u);
                    const uint32_t tS = tmem + C::kColS + N * (g & 1u);
                    // In two halves: the first goes on while the second's slots arrive (32 sequences, 128 heads: 84 us, 88 in one, 90 slot by slot).
                    constexpr uint32_t kFront = (C::kPairs + 1) / 2;
#pragma unroll
                    for (uint32_t half = 0; half < 2; ++half) {
                        const uint32_t c0 = half ? kFront : 0, c1 = half ? C::kPairs : kFront;
                        for (uint32_t c = c0; c < c1; ++c) wait(C::FULL + (g * C::kPairs + c) % C::kPairSlots, ((g * C::kPairs + c) / C::kPairSlots) & 1u);
                        if (half) wait(C::RFULL + g % C::kRopeSlots, (g / C::kRopeSlots) & 1u);
                        tc_fence_after();
                        if (!leader || !ok) continue;
#pragma unroll
                        for (uint32_t c = c0; c < c1; ++c) {
                            const uint64_t dk = make_smem_desc<128>(pair_addr(g * C::kPairs + c), 16), dq = make_smem_desc<128>(base + c * (2 * C::kQChunk), 16);
#pragma unroll
                            for (uint32_t ks = 0; ks < 8; ++ks)
                                mma_ss(tS, dk + (ks >> 2) * (kLatentSlot >> 4) + 2 * (ks & 3u), dq + (ks >> 2) * (C::kQChunk >> 4) + 2 * (ks & 3u), idesc_s, c + ks > 0 ? 1u : 0u);
                        }
                        if (half == 0) continue;
                        const uint64_t dk = make_smem_desc<128>(rope_addr(g), 16), dq = make_smem_desc<128>(base + LC * C::kQChunk, 16);
                        for (uint32_t ks = 0; ks < rope_steps; ++ks) mma_ss(tS, dk + 2 * ks, dq + 2 * ks, idesc_s, 1u);
                        tc_commit(bar(C::REMPTY + g % C::kRopeSlots));
                    }
                    if (leader && ok) {
                        tc_commit(bar(C::S + (g & 1u)));
                        if (tile + 1 == w.end) tc_commit(bar(C::QEMPTY));
                    }
                } else {
                    wait(C::P + (g & 1u), (g >> 1) & 1u);
                    tc_fence_after();
                    if (leader && ok) {
                        const uint64_t dp = make_smem_desc<C::kPitch>(p_addr(g), 16);
#pragma unroll
                        for (uint32_t d = 0; d < C::kPairs; ++d) {
                            const uint32_t n = g * C::kPairs + d;
                            const uint64_t dc = make_smem_desc<128>(pair_addr(n), kLatentSlot);
#pragma unroll
                            for (uint32_t ks = 0; ks < kLatentTile / 16; ++ks)
                                mma_ss(tmem + d * N, dc + ks * (2048 >> 4), dp + ks * (16 * C::kPitch >> 4), idesc_y, tile > w.t0 || ks > 0 ? 1u : 0u);
                            tc_commit(bar(C::EMPTY + n % C::kPairSlots));
                        }
                        tc_commit(bar(C::PV + (g & 1u)));
                    }
                }
                __syncwarp();
            }
            ++k;
        }
        // every product issued has to retire before tensor and shared memory are let go of
        const int last = C::FINAL + (warp == 12 ? 0 : 1);
        if (leader) tc_commit(bar(last));
        __syncwarp();
        mbar_wait_certain(bar(last), 0, ctl, kCacheTimeout | static_cast<uint32_t>(last));
    } else {
        // ---------------------------------------------------------------- queries
        uint32_t k = 0;
        for (bool more = any; more; more = latent_next(p, group, w)) {
            if (w.end == w.t0) continue;
            if (k > 0) mbar_wait(bar(C::QEMPTY), (k - 1u) & 1u, ctl, kCacheTimeout | C::QEMPTY);
            if (k == 0) {
                copy_queries(w.seq, kLatentSoftmax + tid - 448u, kLatentSoftmax + 64u, N);
                cp_async_wait_all();
                fence_proxy_async_smem();
                asm volatile("barrier.cta.sync 2, 320;" ::: "memory");   // the softmax warps' share is there
            } else {
                copy_queries(w.seq, tid - 448u, 64u, n_rows);
                cp_async_wait_all();
                fence_proxy_async_smem();
            }
            mbar_arrive(bar(C::QFULL));
            ++k;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0) report_expired(ctl);
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, C::kCols);
    }
}

// Puts the parts of divided sequences together: 128 dimensions of a row at a time.  By a warp (kWide false), where there are few parts, or by a
// CTA whose warps take the parts in turn.
constexpr int kLatentJoinWarps = 8;
template <int LC, int N, bool kWide>
__global__ void __launch_bounds__(kLatentJoinWarps * 32) fa_latent_join(const LatentRowsArgs p) {
    __shared__ float4 s_o[kWide ? kLatentJoinWarps : 1][32];
    __shared__ float s_sum[kLatentJoinWarps], s_top[kLatentJoinWarps];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint64_t item = kWide ? blockIdx.x : static_cast<uint64_t>(blockIdx.x) * kLatentJoinWarps + warp;
    const uint32_t dims = static_cast<uint32_t>(item % (LC / 2)) * 128 + 4 * lane;
    const uint64_t at = item / (LC / 2);
    const uint32_t b = static_cast<uint32_t>(at / p.rows), row = static_cast<uint32_t>(at - static_cast<uint64_t>(b) * p.rows), group = row / p.group_rows, r = row - group * p.group_rows;
    grid_dep_wait();
    grid_dep_launch();
    if (b >= p.s.B) return;
    // (what a sequence without tokens has for its share is not used: both are asked for at once)
    const int2 share = p.shares[b];
    if (latent_units(p, b) == 0 || share.x == share.y) return;   // written where it was worked out
    auto slot = [&](int part) { return ((static_cast<uint64_t>(part) * p.groups + group) * 2u + (part == share.x ? 1u : 0u)) * N + r; };
    float top = -INFINITY;
    for (int i = share.x + static_cast<int>(kWide ? threadIdx.x : lane); i <= share.y; i += kWide ? kLatentJoinWarps * 32 : 32) top = fmaxf(top, p.part_ml[slot(i)].x);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    if (kWide) {
        if (lane == 0) s_top[warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kLatentJoinWarps; ++i) top = fmaxf(top, s_top[i]);
    }
    if (top == -INFINITY) top = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    float sum = 0.0f;
#pragma unroll 4
    for (int i = share.x + static_cast<int>(kWide ? warp : 0); i <= share.y; i += kWide ? kLatentJoinWarps : 1) {
        const float2 ml = p.part_ml[slot(i)];
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + slot(i) * (64 * LC) + dims);
        if (ml.y == 0.0f) continue;   // nothing seen there: what was read is nothing
        const float f = ex2_approx((ml.x == -INFINITY ? 0.0f : ml.x) - top);
        o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
        sum = fmaf(ml.y, f, sum);
    }
    if (kWide) {
        s_o[warp][lane] = o;
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        if (warp != 0) return;
        for (int i = 1; i < kLatentJoinWarps; ++i) {
            const float4 x = s_o[i][lane];
            o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w, sum += s_sum[i];
        }
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<uint2*>(p.y + (at * (64 * LC) + dims) * 2) = make_uint2(pack_16(o.x * f, o.y * f, p.bf16 != 0), pack_16(o.z * f, o.w * f, p.bf16 != 0));
}

}  // namespace fa
