// The pages of a cache: who holds them, sharing, pages of one's own, moving to the front; and copying what they hold.
//
// refs[p] is the number of table entries that hold page p, 0: it is free.  A table entry is a page or -1; anything else is reported and
// taken for -1.  All results are whole numbers that depend on nothing but the inputs: counts change by atomic additions, whose order
// does not matter, and where one of several has to be chosen it is by a minimum, likewise.
//
// These kernels read and write a few kilobytes to a megabyte: what bounds them is the chain of dependent accesses and the launch, so that
// each call is one launch (compacting, and reserving in a large table: two) and no value crosses to the host.  Copying is bound by memory.
// Measured in a graph: a step of 8 beams of an 8-bit cache (fork, reserve, copy of 4 pages) 11 us, of 256 beams of two latent caches (141 pages of
// 147 KB) 21, of which copying takes 7.6 (5.5 TB/s); 10000 pages planned in 11 us, 2381 of 133 KB moved in 115 (5.5 TB/s, 84 % of a plain copy's).
#pragma once

#include "fa_cache.cuh"

namespace fa {

// Status codes (kCacheBadPage, kCacheBadPosition beside them).
constexpr uint32_t kPagesNone = 3u;    // a sequence needed a page and none was free
constexpr uint32_t kPagesCount = 4u;   // counts that do not fit the table: a page was let go of that nobody held

struct PagesView {
    int32_t* refs;
    uint32_t* status;   // first code, number of reports; pools of one cache may share them
    uint32_t n;
};
struct PagesTable {
    int32_t* at;        // [B, width], rows `stride` apart
    int64_t stride;
    uint32_t width, B;
};

__device__ __forceinline__ int32_t ld_cg(const int32_t* p) {
    int32_t v;
    asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ int4 ld_cg(const int4* p) {
    int4 v;
    asm volatile("ld.global.cg.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ bool is_page(const PagesView& v, int32_t entry) { return static_cast<uint32_t>(entry) < v.n; }
__device__ __forceinline__ void let_go(const PagesView& v, int32_t entry) {
    if (!is_page(v, entry)) {
        if (entry != -1) cache_report(v.status, kCacheBadPage);
        return;
    }
    if (atomicSub(v.refs + entry, 1) <= 0) cache_report(v.status, kPagesCount);
}

// ----------------------------------------------------------------------------- fork
// Columns of the table are independent: a CTA takes `cols` of them, holds all their entries in shared memory and puts them where they
// belong, so the table can be changed in place.  The last CTA does so with the lengths.
struct ForkArgs {
    PagesView v;
    PagesTable t;
    int32_t* lengths;
    const int32_t* parents;
    uint32_t cols;
};
constexpr int kForkThreads = 256;
__global__ void __launch_bounds__(kForkThreads) fa_pages_fork(const ForkArgs p) {
    extern __shared__ int32_t s_old[];   // [B, cols]
    grid_dep_wait();
    grid_dep_launch();
    const bool is_lengths = blockIdx.x == gridDim.x - 1;
    const uint32_t col0 = blockIdx.x * p.cols, cols = is_lengths ? 1u : min(p.cols, p.t.width - col0);
    int32_t* const base = is_lengths ? p.lengths : p.t.at + col0;
    const int64_t stride = is_lengths ? 1 : p.t.stride;
    const uint32_t all = p.t.B * cols;
    auto parent_of = [&](uint32_t b) {
        const int32_t parent = p.parents[b];
        if (parent >= -1 && parent < static_cast<int32_t>(p.t.B)) return parent;
        if (is_lengths) cache_report(p.v.status, kCacheBadPosition);   // stays as it is
        return static_cast<int32_t>(b);
    };
    const int32_t first = threadIdx.x < all ? p.parents[threadIdx.x / cols] : 0;   // (asked for with the entries)
    for (uint32_t i = threadIdx.x; i < all; i += kForkThreads) s_old[i] = base[(i / cols) * stride + i % cols];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < all; i += kForkThreads) {
        const uint32_t b = i / cols, c = i % cols;
        const int32_t parent = i < kForkThreads && first >= -1 && first < static_cast<int32_t>(p.t.B) ? first : parent_of(b);
        const int32_t before = s_old[i];
        int32_t now = parent < 0 ? (is_lengths ? 0 : -1) : s_old[static_cast<uint32_t>(parent) * cols + c];
        if (!is_lengths && now != -1 && !is_page(p.v, now)) {
            cache_report(p.v.status, kCacheBadPage);
            now = -1;
        }
        if (now == before) continue;
        base[b * stride + c] = now;
        if (is_lengths) continue;
        let_go(p.v, before);
        if (now >= 0) atomicAdd(p.v.refs + now, 1);
    }
}

// ----------------------------------------------------------------------------- reserve
// First, blocks behind those that are needed are let go of.  Where the table is small the one CTA that does the rest does that too; otherwise CTAs
// take sequences, a warp each, in a launch of their own.  (Finding the last CTA of one launch takes a counter that is zero beforehand, and calls on
// several tables must not meet there.  In a graph two launches are no slower: 256 sequences of 20 blocks in a table of 2048 11.2 us, 11.6 with a
// counter; 1000 in one of 64 7.7 and 8.9.  The second launch costs the host 5 us, so that an eager call of the latter takes 14, not 9.)
// One CTA does the rest, with `lanes` threads a sequence (as many as its tokens touch blocks, up to 32):
//
//   1  the free pages (count 0), in ascending order, as many as blocks are written to
//   2  entries that are written to and whose page is held by others too let go of it.  What is left of a page's count is the number of
//      those that hold it and do not write to it
//   3  where that is none all that hold the page write to it, and the sequence with the most tokens on it keeps it, the lowest of several: the
//      count becomes the least of their numbers (keeper_number).  The others may find no page and stay on this one, and where the keeper goes on
//      none of them has a token
//   4  an entry keeps its page if it finds its own number there; the others want one.  (Without shared pages 2 to 4 are passed over)
//   5  each takes the page of its rank, in order of sequences and blocks; where there is none left, the entry stays as it was and its
//      sequence is granted fewer tokens
struct ReserveArgs {
    PagesView v;
    PagesTable t;
    const int32_t* lengths;
    const int32_t* counts;   // null: `count` of each
    int32_t* granted;        // [B]
    int32_t* sources;        // [B]
    int32_t* targets;
    int32_t* list;           // [n]: free pages
    uint32_t count, page_shift, alone;   // alone: the one CTA lets go of blocks as well
};
constexpr int kReserveThreads = 1024, kReserveWarps = kReserveThreads / 32;
constexpr uint32_t kNoBlock = 0xFFFFFFFFu;

struct Window {   // of the blocks that a sequence's new tokens touch
    uint32_t held, count, first, need;
    bool ok;
};
__device__ __forceinline__ Window reserve_window(const ReserveArgs& p, uint32_t b) {
    Window w;
    const int32_t held = p.lengths[b], count = p.counts ? p.counts[b] : static_cast<int32_t>(p.count);
    const uint64_t room = min(static_cast<uint64_t>(p.t.width) << p.page_shift, static_cast<uint64_t>(0x7FFFFFFF));
    w.ok = held >= 0 && count >= 0 && static_cast<uint64_t>(held) + static_cast<uint64_t>(count) <= room;
    w.held = static_cast<uint32_t>(min(static_cast<uint64_t>(max(held, 0)), room));
    w.count = static_cast<uint32_t>(min(static_cast<uint64_t>(max(count, 0)), room - w.held));
    w.first = w.held >> p.page_shift;
    w.need = (w.held + w.count + (1u << p.page_shift) - 1u) >> p.page_shift;
    if (w.count == 0) w.first = w.need;   // nothing is written
    return w;
}
// A sequence's number among those that might keep the page of block i: the lower, the more tokens it has there, and among several the lower it is.
// Below zero, and none twice.  (The page is written to, so that it has room: 127 tokens at most, and with up to 2^24 sequences 128 B is 2^31.)
__device__ __forceinline__ int32_t keeper_number(const ReserveArgs& p, const Window& w, uint32_t b, uint32_t i) {
    const uint32_t begins = i << p.page_shift, tokens = w.held > begins ? w.held - begins : 0u;
    return static_cast<int32_t>(0u - (tokens * p.t.B + (p.t.B - b)));
}
// What takes a count from such a number to one, whatever is added beside it (the count passes 2^31 on the way, which additions do not mind).
__device__ __forceinline__ int32_t keeper_to_one(int32_t number) { return static_cast<int32_t>(1u - static_cast<uint32_t>(number)); }
// Sum of x over the threads in front of this one; `all`: of all threads.  All threads of the CTA.
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t* s_warp, uint32_t& all) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t upto = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += y;
    }
    __syncthreads();   // (s_warp may still be read from the last time)
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    const uint32_t w = s_warp[lane];   // as many warps as lanes
    uint32_t sums = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, sums, d);
        if (lane >= d) sums += y;
    }
    all = __shfl_sync(0xFFFFFFFFu, sums, 31);
    return __shfl_sync(0xFFFFFFFFu, sums - w, warp) + upto - x;
}

// Which of pages [q, q + 16) are free.
__device__ __forceinline__ uint32_t free_of_16(const PagesView& v, uint32_t q) {
    uint32_t free = 0;
    if (q + 16 <= v.n && (reinterpret_cast<uintptr_t>(v.refs) & 15u) == 0) {
        int4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = ld_cg(reinterpret_cast<const int4*>(v.refs + q) + k);
#pragma unroll
        for (int k = 0; k < 4; ++k) free |= ((x[k].x == 0) | (x[k].y == 0) << 1 | (x[k].z == 0) << 2 | (x[k].w == 0) << 3) << (4 * k);
    } else {
        for (uint32_t k = 0; k < 16 && q + k < v.n; ++k) free |= static_cast<uint32_t>(ld_cg(v.refs + q + k) == 0) << k;
    }
    return free;
}
// A table of this many entries and sequences is gone over by one CTA, eight entries of a thread at a time.
constexpr uint32_t kAloneEntries = 32768, kAloneRows = 2048;

__global__ void __launch_bounds__(kReserveThreads) fa_pages_release(const ReserveArgs p) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    grid_dep_wait();
    grid_dep_launch();
    for (uint32_t b = blockIdx.x * kReserveWarps + warp; b < p.t.B; b += gridDim.x * kReserveWarps) {
        const Window w = reserve_window(p, b);
        if (lane == 0 && !w.ok) cache_report(p.v.status, kCacheBadPosition);
        int32_t* const row = p.t.at + b * p.t.stride;
        for (uint32_t i = w.need + lane; i < p.t.width; i += 128) {   // four loads of a lane in flight
            int32_t e[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) e[k] = i + 32 * k < p.t.width ? row[i + 32 * k] : -1;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (e[k] != -1) {
                    let_go(p.v, e[k]);
                    row[i + 32 * k] = -1;
                }
        }
    }
}

__global__ void __launch_bounds__(kReserveThreads) fa_pages_reserve(const ReserveArgs p) {
    __shared__ uint32_t s_warp[32], s_most, s_need[kAloneRows];
    __shared__ int32_t s_list[kReserveThreads];
    const uint32_t tid = threadIdx.x, lane = tid & 31u;
    if (tid == 0) s_most = 0;
    grid_dep_wait();
    grid_dep_launch();
    uint32_t free = free_of_16(p.v, 16 * tid), most = 0, bound = 0;   // (asked for along with the lengths)
    auto count_in = [&](const Window& w) {
        most = max(most, w.need - w.first);
        bound += w.need - w.first;
    };
    bool let = false;
    if (p.alone) {
        for (uint32_t b = tid; b < p.t.B; b += kReserveThreads) {
            const Window w = reserve_window(p, b);
            if (!w.ok) cache_report(p.v.status, kCacheBadPosition);
            count_in(w);
            s_need[b] = w.need;
        }
        __syncthreads();
        const uint32_t entries = p.t.B * p.t.width;
        for (uint32_t i = tid; i < entries; i += 8 * kReserveThreads) {
            int32_t e[8];
            int32_t* at[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                const uint32_t j = i + k * kReserveThreads, b = j / p.t.width, c = j - b * p.t.width;
                at[k] = p.t.at + b * p.t.stride + c;
                e[k] = j < entries && c >= s_need[b] ? *at[k] : -1;
            }
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (e[k] != -1) {
                    let_go(p.v, e[k]);
                    *at[k] = -1;
                    let = true;
                }
        }
    } else {
        for (uint32_t b = tid; b < p.t.B; b += kReserveThreads) count_in(reserve_window(p, b));
        __syncthreads();   // s_most
    }

    // how many blocks a sequence's tokens touch at most decides how many threads it gets
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if (lane == 0) atomicMax(&s_most, most);
    if (__syncthreads_or(let)) free = free_of_16(p.v, 16 * tid);
    most = s_most;
    uint32_t shift = 0;
    while (shift < 5 && (1u << shift) < most) ++shift;
    const uint32_t lanes = 1u << shift, per = (most + lanes - 1) >> shift, at_once = kReserveThreads >> shift;
    const uint32_t mine = tid >> shift, l = tid & (lanes - 1u);   // which of the sequences at hand, and of its lanes
    // this thread's blocks [i0, i1) of sequence b
    auto blocks = [&](uint32_t b, Window& w, uint32_t& i0, uint32_t& i1) {
        i0 = i1 = 0;
        if (b >= p.t.B) return;
        w = reserve_window(p, b);
        i0 = min(w.need, w.first + l * per), i1 = min(w.need, i0 + per);
    };
    // Where no sequence's tokens touch more than a block for each of its threads, and all are at hand at once, entries stay in registers
    // and the free pages in shared memory: the calls between two tokens of a decoder.
    const bool at_hand = per <= 1 && p.t.B <= at_once;
    Window own_w = {};
    uint32_t own_i = 0;
    bool writes = false;
    int32_t own_e = -1;
    if (at_hand && mine < p.t.B) {
        own_w = reserve_window(p, mine);
        own_i = own_w.first + l;
        writes = own_i < own_w.need;
        if (writes) own_e = p.t.at[mine * p.t.stride + own_i];
    }
    int32_t* const list = at_hand ? s_list : p.list;
    // 1: 16 of a thread at a time
    uint32_t all_bound, found = 0;
    (void)sum_before(bound, s_warp, all_bound);
    for (uint32_t q0 = 0; q0 < p.v.n && found < all_bound; q0 += 16 * kReserveThreads) {
        const uint32_t q = q0 + 16 * tid;
        if (q0 > 0) free = free_of_16(p.v, q);
        uint32_t all, at = found + sum_before(__popc(free), s_warp, all);
        for (; free != 0 && at < all_bound; free &= free - 1u) list[at++] = static_cast<int32_t>(q + __ffs(free) - 1);   // (`at` stays below n)
        found += all;
    }
    if (at_hand) {
        bool is_shared = false, keeps = false;
        if (writes && own_e != -1) {
            if (!is_page(p.v, own_e)) {
                cache_report(p.v.status, kCacheBadPage);
                own_e = -1;
            } else {
                const int32_t holders = ld_cg(p.v.refs + own_e);
                is_shared = holders > 1, keeps = !is_shared;
                if (holders < 1) cache_report(p.v.status, kPagesCount);
            }
        }
        if (__syncthreads_or(is_shared)) {
            const int32_t own = keeper_number(p, own_w, mine, own_i);
            if (is_shared) atomicSub(p.v.refs + own_e, 1);
            __syncthreads();
            const bool all_write = is_shared && ld_cg(p.v.refs + own_e) <= 0;
            if (all_write) atomicMin(p.v.refs + own_e, own);
            __syncthreads();
            if (all_write && ld_cg(p.v.refs + own_e) == own) {
                keeps = true;
                is_shared = false;
            }
            __syncthreads();   // everyone has looked
            if (keeps && all_write) atomicAdd(p.v.refs + own_e, keeper_to_one(own));   // (refused entries add theirs)
        }
        uint32_t demand;
        const uint32_t rank = sum_before(writes && !keeps, s_warp, demand), there = min(found, demand);
        uint32_t refused = kNoBlock;
        int32_t source = -1, target = -1;
        if (writes && !keeps) {
            int32_t* const entry = p.t.at + mine * p.t.stride + own_i;
            if (rank < there) {
                const int32_t page = s_list[rank];
                *entry = page;
                p.v.refs[page] = 1;
                if (own_e >= 0 && l == 0 && (own_w.held & ((1u << p.page_shift) - 1u)) != 0) source = own_e, target = page;
            } else {
                if (own_e >= 0) atomicAdd(p.v.refs + own_e, 1);
                else *entry = -1;
                refused = own_i;
                cache_report(p.v.status, kPagesNone);
            }
        }
        for (uint32_t d = lanes >> 1; d >= 1; d >>= 1) refused = min(refused, __shfl_xor_sync(0xFFFFFFFFu, refused, d));
        if (mine < p.t.B && l == 0) {
            const uint32_t room = refused == kNoBlock ? own_w.count : max(refused << p.page_shift, own_w.held) - own_w.held;
            p.granted[mine] = static_cast<int32_t>(min(own_w.count, room));
            p.sources[mine] = source;
            p.targets[mine] = target;
        }
        return;
    }
    // 2 to 4; what is kept is marked in the table, where nobody else looks: -2 - page if it was held alone, -2 - n - page if all that hold it write
    // to it (n is below 2^30).  How many pages are wanted
    uint32_t wanted = 0;
    bool shared = false;
    for (uint32_t b0 = 0; b0 < p.t.B; b0 += at_once) {
        const uint32_t b = b0 + mine;
        Window w;
        uint32_t i0, i1;
        blocks(b, w, i0, i1);
        for (uint32_t i = i0; i < i1; ++i) {
            int32_t* const entry = p.t.at + b * p.t.stride + i;
            const int32_t e = *entry;
            if (!is_page(p.v, e)) {
                if (e != -1) {
                    cache_report(p.v.status, kCacheBadPage);
                    *entry = -1;
                }
                ++wanted;
            } else {
                const int32_t holders = ld_cg(p.v.refs + e);
                if (holders > 1) shared = true;
                else *entry = -2 - e;
                if (holders < 1) cache_report(p.v.status, kPagesCount);
            }
        }
    }
    if (__syncthreads_or(shared)) {
        for (int step = 2; step <= 4; ++step) {
            for (uint32_t b0 = 0; b0 < p.t.B; b0 += at_once) {
                const uint32_t b = b0 + mine;
                Window w;
                uint32_t i0, i1;
                blocks(b, w, i0, i1);
                for (uint32_t i = i0; i < i1; ++i) {
                    int32_t* const entry = p.t.at + b * p.t.stride + i;
                    const int32_t e = *entry, own = keeper_number(p, w, b, i);
                    if (e < 0) continue;   // wanted, or kept already
                    if (step == 2) atomicSub(p.v.refs + e, 1);
                    else if (step == 3 && ld_cg(p.v.refs + e) <= 0) atomicMin(p.v.refs + e, own);
                    else if (step == 4) {
                        if (ld_cg(p.v.refs + e) == own) *entry = -2 - static_cast<int32_t>(p.v.n) - e;
                        else ++wanted;
                    }
                }
            }
            __syncthreads();
        }
    }
    uint32_t demand;
    (void)sum_before(wanted, s_warp, demand);
    const uint32_t there = min(found, demand);
    // 5
    uint32_t in_front = 0;
    for (uint32_t b0 = 0; b0 < p.t.B; b0 += at_once) {
        const uint32_t b = b0 + mine;
        Window w;
        uint32_t i0, i1, n = 0, all;
        blocks(b, w, i0, i1);
        for (uint32_t i = i0; i < i1; ++i) n += p.t.at[b * p.t.stride + i] >= -1;
        uint32_t rank = in_front + sum_before(n, s_warp, all), refused = kNoBlock;
        in_front += all;
        int32_t source = -1, target = -1;
        for (uint32_t i = i0; i < i1; ++i) {
            int32_t* const entry = p.t.at + b * p.t.stride + i;
            const int32_t e = *entry;
            if (e < -1) {   // kept
                const int32_t page = -2 - e, n_pages = static_cast<int32_t>(p.v.n);
                if (page < n_pages) {
                    *entry = page;
                } else {
                    *entry = page - n_pages;
                    atomicAdd(p.v.refs + (page - n_pages), keeper_to_one(keeper_number(p, w, b, i)));
                }
                continue;
            }
            if (rank < there) {
                const int32_t page = p.list[rank];
                *entry = page;
                atomicAdd(p.v.refs + page, 1);
                if (e >= 0 && i == w.held >> p.page_shift && (w.held & ((1u << p.page_shift) - 1u)) != 0) source = e, target = page;
            } else {
                if (e >= 0) atomicAdd(p.v.refs + e, 1);
                refused = min(refused, i);
                cache_report(p.v.status, kPagesNone);
            }
            ++rank;
        }
        for (uint32_t d = lanes >> 1; d >= 1; d >>= 1) refused = min(refused, __shfl_xor_sync(0xFFFFFFFFu, refused, d));
        if (b < p.t.B && l == 0) {   // (the first of a sequence's lanes has the block that may be copied)
            const uint32_t room = refused == kNoBlock ? w.count : max(refused << p.page_shift, w.held) - w.held;
            p.granted[b] = static_cast<int32_t>(min(w.count, room));
            p.sources[b] = source;
            p.targets[b] = target;
        }
    }
}

// ----------------------------------------------------------------------------- compact
// With n_used pages held, those from n_used on move to the free ones in front of it, the k-th to the k-th.  A CTA works out 4096 pages;
// it counts those in front of them itself, from all of refs (13333 pages are 53 KB), so that no CTA waits for another.  What is read
// grows with the square of the pages: a call takes 21 us for 10000 and for 100000 of them, 170 for a million, 2 ms for 4 and 32 for 16 million.
struct CompactArgs {
    PagesView v;
    PagesTable t;
    int32_t* new_refs;    // [n]
    int32_t* new_table;   // [B, width] contiguous
    int32_t* sources;     // [n]
    int32_t* targets;
    int32_t* rank;        // [n]: which of the moves a page is, -1: it stays or is free
    uint32_t* totals;     // used pages, moves
};
constexpr int kCompactThreads = 1024, kCompactPages = 4 * kCompactThreads;
__global__ void __launch_bounds__(kCompactThreads) fa_pages_plan(const CompactArgs p) {
    __shared__ uint32_t s_warp[32];
    const uint32_t tid = threadIdx.x, n = p.v.n, base = blockIdx.x * kCompactPages;
    grid_dep_wait();
    grid_dep_launch();
    // used pages among [0, end) and how many of them are in front of `cut`; eight of a thread in flight
    auto count = [&](uint32_t end, uint32_t cut, uint32_t& front, uint32_t& all) {
        uint32_t x = 0, y = 0;
        for (uint32_t q = tid; q < end; q += 8 * kCompactThreads) {
            int32_t r[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) r[k] = q + k * kCompactThreads < end ? p.v.refs[q + k * kCompactThreads] : 0;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) x += r[k] > 0 && q + k * kCompactThreads < cut, y += r[k] > 0;
        }
        (void)sum_before(x, s_warp, front);
        (void)sum_before(y, s_warp, all);
    };
    uint32_t used_front, n_used, low_used, same;
    count(n, base, used_front, n_used);
    count(n_used, 0, same, low_used);
    const uint32_t moves = n_used - low_used;
    if (blockIdx.x == 0 && tid == 0) p.totals[0] = n_used, p.totals[1] = moves;
    int32_t r[4];
    uint32_t used = 0, all;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t q = base + 4 * tid + k;
        r[k] = q < n ? p.v.refs[q] : 0;
        used += r[k] > 0;
    }
    uint32_t before = used_front + sum_before(used, s_warp, all);   // used pages in front of q
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t q = base + 4 * tid + k;
        if (q >= n) break;
        const bool is_used = r[k] > 0;
        const bool moves_on = is_used && q >= n_used;
        p.rank[q] = moves_on ? static_cast<int32_t>(before - low_used) : -1;
        if (moves_on) p.sources[before - low_used] = static_cast<int32_t>(q);
        else if (!is_used && q < n_used) p.targets[q - before] = static_cast<int32_t>(q);
        if (q >= n_used) p.new_refs[q] = 0;
        else if (is_used) p.new_refs[q] = r[k];   // (the others: fa_pages_renumber)
        if (q >= moves) p.sources[q] = -1, p.targets[q] = -1;
        before += is_used;
    }
}
__global__ void __launch_bounds__(256) fa_pages_renumber(const CompactArgs p) {
    grid_dep_wait();
    grid_dep_launch();
    const uint64_t entries = static_cast<uint64_t>(p.t.B) * p.t.width;
    const uint32_t n_used = p.totals[0], moves = p.totals[1];
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < entries || i < moves; i += gridDim.x * 256ull) {
        if (i < moves) p.new_refs[p.targets[i]] = p.v.refs[p.sources[i]];
        if (i >= entries) continue;
        const uint64_t b = i / p.t.width;
        int32_t e = p.t.at[static_cast<int64_t>(b) * p.t.stride + static_cast<int64_t>(i - b * p.t.width)];
        if (!is_page(p.v, e)) {
            if (e != -1) cache_report(p.v.status, kCacheBadPage);
            e = -1;
        } else if (p.v.refs[e] <= 0) {   // an entry that is not counted
            cache_report(p.v.status, kPagesCount);
            e = -1;
        } else if (static_cast<uint32_t>(e) >= n_used) {
            e = p.targets[p.rank[e]];
        }
        p.new_table[i] = e;
    }
}

// ----------------------------------------------------------------------------- copy
// Contents of pages, source to target, for up to kCopyAreas arrays: a page of an array is n0 x n1 rows of `row` bytes (one row where it
// lies in one piece), taken 16 or 4 bytes at a time.  CTAs are dealt out by parts of a page, `parts` equal ones of each array, first: CTA (x, y)
// has part y of the pairs x, x + gridDim.x, ...  Every thread has eight pieces of 16 bytes in flight.
struct CopyArea {
    uint8_t* base;
    int64_t page, stride0, stride1;   // bytes
    uint32_t n0, n1, row, parts;
    uint32_t unit;                    // 16 if base, strides and row are multiples of that, else 4
};
constexpr int kCopyAreas = 32;
struct CopyArgs {
    CopyArea area[kCopyAreas];
    const int32_t* sources;
    const int32_t* targets;
    uint32_t* status;
    uint32_t areas, pairs, n;   // n: pages of every array
};
constexpr int kCopyThreads = 256;
constexpr int kCopyFlight = 8;

template <typename Piece>
__device__ __forceinline__ void copy_part(const CopyArea& a, uint32_t source, uint32_t target, uint32_t part) {
    const uint32_t in_row = a.row / sizeof(Piece);
    const uint64_t pieces = static_cast<uint64_t>(a.n0) * a.n1 * in_row, begin = pieces * part / a.parts, end = pieces * (part + 1) / a.parts;
    const uint8_t* const from = a.base + source * a.page;
    uint8_t* const to = a.base + target * a.page;
    if (a.n0 * a.n1 == 1) {
        for (uint64_t i = begin + threadIdx.x; i < end; i += kCopyThreads * kCopyFlight) {
            Piece x[kCopyFlight];
#pragma unroll
            for (int k = 0; k < kCopyFlight; ++k)
                if (i + k * kCopyThreads < end) x[k] = reinterpret_cast<const Piece*>(from)[i + k * kCopyThreads];
#pragma unroll
            for (int k = 0; k < kCopyFlight; ++k)
                if (i + k * kCopyThreads < end) reinterpret_cast<Piece*>(to)[i + k * kCopyThreads] = x[k];
        }
        return;
    }
    auto place = [&](uint64_t i) {
        const uint32_t r = static_cast<uint32_t>(i / in_row), c = static_cast<uint32_t>(i - static_cast<uint64_t>(r) * in_row), r0 = r / a.n1;
        return r0 * a.stride0 + (r - r0 * a.n1) * a.stride1 + static_cast<int64_t>(c * sizeof(Piece));
    };
    for (uint64_t i = begin + threadIdx.x; i < end; i += kCopyThreads * 4) {
        Piece x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * kCopyThreads < end) x[k] = *reinterpret_cast<const Piece*>(from + place(i + k * kCopyThreads));
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * kCopyThreads < end) *reinterpret_cast<Piece*>(to + place(i + k * kCopyThreads)) = x[k];
    }
}

__global__ void __launch_bounds__(kCopyThreads, 3) fa_cache_copy(const __grid_constant__ CopyArgs p) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t k = 0, part = blockIdx.y;
    while (part >= p.area[k].parts) part -= p.area[k++].parts;   // (gridDim.y is their sum)
    const CopyArea& a = p.area[k];
    grid_dep_wait();
    grid_dep_launch();
    for (uint64_t i0 = blockIdx.x; i0 < p.pairs; i0 += 32ull * gridDim.x) {   // every warp looks at 32 of the CTA's pairs
        const uint64_t i = i0 + static_cast<uint64_t>(lane) * gridDim.x;
        const int32_t s = i < p.pairs ? p.sources[i] : -1, t = i < p.pairs ? p.targets[i] : -1;
        const bool good = static_cast<uint32_t>(s) < p.n && static_cast<uint32_t>(t) < p.n;
        if (!good && ((s != -1 && static_cast<uint32_t>(s) >= p.n) || (t != -1 && static_cast<uint32_t>(t) >= p.n)) && threadIdx.x < 32 && blockIdx.y == 0)
            cache_report(p.status, kCacheBadPage);
        for (uint32_t left = __ballot_sync(0xFFFFFFFFu, good && s != t); left != 0; left &= left - 1u) {
            const int from = __ffs(left) - 1;
            const uint32_t source = static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, s, from)), target = static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, t, from));
            if (a.unit == 16) copy_part<uint4>(a, source, target, part);
            else copy_part<uint32_t>(a, source, target, part);
        }
    }
}

}  // namespace fa
