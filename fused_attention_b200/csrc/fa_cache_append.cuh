// Appending keys and values to the cache, with the position rotation of keys and queries on the way.
//
// A task is one page and head of the keys or of the values that a sequence's new tokens touch.  Its new tokens are read and
// (keys) rotated in fp32, x1 c - x2 s and x2 c + x1 s with every product and sum rounded by itself.  The largest magnitude `a`
// gives the scale, the smallest power of two with a / scale <= 448, 2^-100 at least.  A page that held tokens keeps its scale
// unless the new tokens need a larger one; its old codes are then moved to it, which loses nothing but bits of the smallest
// (subnormal) codes, since both scales are powers of two: a page that is filled token by token ends as close to its values as
// one that is filled at once.  A value that is not finite makes the page's scale NaN and its codes zero.
//
// Prompts: 4 of up to 2048 tokens, 8 heads of 128 with 32 of queries, ask for 94 MB and take 25 to 29 us, 3.2 to 3.7 TB/s (73 MB of that
// reach DRAM in a launch by itself, 30 us); without queries, a third of the bytes, 14.6 us.  What holds either half below the memory's rate
// has not been found out.  Single tokens are bound by the chain length -> table entry -> old scale -> codes, which is why a task is a
// warp there: B=256 sequences of 8 heads are 4096 tasks (7.8 us; 17.6 with a CTA each).
#pragma once

#include "fa_cache.cuh"

namespace fa {

struct AppendArgs {
    CacheView c;
    CacheSeqs s;
    const uint8_t* keys;      // 16-bit rows of heads * H values
    const uint8_t* values;
    const uint8_t* queries;   // null: none
    uint8_t* rotated;         // [B, T, q_heads * H] contiguous
    const float* cos;         // [positions, H / 2]; null: no rotation
    const float* sin;
    int64_t keys_b, keys_t, values_b, values_t, queries_b, queries_t;   // strides in bytes
    uint32_t positions, q_heads, blocks, bf16, interleaved;
    uint32_t tasks, query_ctas;
};

// The 16 values of a head that one thread works on: dimensions [8 j, 8 j + 8) and [H/2 + 8 j, H/2 + 8 j + 8).
struct Sixteen {
    float a[8], b[8];
};
struct RawSixteen {
    uint4 x, y;
};
template <int H>
__device__ __forceinline__ RawSixteen load_sixteen(const uint8_t* row, uint32_t j) {
    return RawSixteen{*reinterpret_cast<const uint4*>(row + 16 * j), *reinterpret_cast<const uint4*>(row + H + 16 * j)};
}
__device__ __forceinline__ Sixteen unpack_sixteen(const RawSixteen& w, bool bf16) {
    const uint32_t xs[4] = {w.x.x, w.x.y, w.x.z, w.x.w}, ys[4] = {w.y.x, w.y.y, w.y.z, w.y.w};
    Sixteen r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = unpack_16(xs[i], bf16), q = unpack_16(ys[i], bf16);
        r.a[2 * i] = p.x, r.a[2 * i + 1] = p.y, r.b[2 * i] = q.x, r.b[2 * i + 1] = q.y;
    }
    return r;
}
__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
    const float u = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
    y = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
    x = u;
}
// cos and sin of the eight pairs that the sixteen values form: (i, i + H/2), or neighbours (2i, 2i + 1).
struct Angles {
    float c[8], s[8];
};
template <int H>
__device__ __forceinline__ Angles load_angles(const AppendArgs& p, uint32_t position, uint32_t j) {
    Angles a = {};
    if (!FA_CACHE_OK(p.c.status, kDbgRow, position < p.positions && 8 * j + 8 <= H / 2)) return a;
    const size_t at = static_cast<size_t>(position) * (H / 2);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const size_t from = at + (p.interleaved ? q * (H / 4) + 4 * j : 8 * j + 4 * q);
        const float4 c = *reinterpret_cast<const float4*>(p.cos + from), s = *reinterpret_cast<const float4*>(p.sin + from);
        a.c[4 * q] = c.x, a.c[4 * q + 1] = c.y, a.c[4 * q + 2] = c.z, a.c[4 * q + 3] = c.w;
        a.s[4 * q] = s.x, a.s[4 * q + 1] = s.y, a.s[4 * q + 2] = s.z, a.s[4 * q + 3] = s.w;
    }
    return a;
}
__device__ __forceinline__ void rotate(Sixteen& r, const Angles& a, bool interleaved) {
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            turn(r.a[2 * i], r.a[2 * i + 1], a.c[i], a.s[i]);
            turn(r.b[2 * i], r.b[2 * i + 1], a.c[4 + i], a.s[4 + i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(r.a[i], r.b[i], a.c[i], a.s[i]);
    }
}

// The smallest power of two, 2^-100 at least, that brings `most` to 448 or below; NaN if `most` is not finite.
__device__ __forceinline__ float append_scale(float most) {
    if (!(most < __int_as_float(0x7F800000))) return __int_as_float(0x7FC00000);
    const uint32_t bits = __float_as_uint(most);
    const int32_t k = static_cast<int32_t>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);   // 448 = 1.75 * 2^8
    return __uint_as_float(static_cast<uint32_t>(max(k, 27)) << 23);
}
// (the larger of the two, NaN if one is)
__device__ __forceinline__ float larger_scale(float x, float y) { return x > y || x != x ? x : y; }

// NaN if one is.
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float min_nan(float x, float y) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ uint32_t half2_min(uint32_t x, uint32_t y) {
    const __half2 r = __hmin2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half2_max(uint32_t x, uint32_t y) {
    const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Four codes, their values multiplied by a power of two <= 1.
__device__ __forceinline__ uint32_t moved_codes(uint32_t four, float shrink) {
    uint32_t lo, hi;
    e4m3x4_to_half2(four, lo, hi);
    const float2 x = unpack_half2(lo), y = unpack_half2(hi);
    return floats_to_e4m3x2(x.x * shrink, x.y * shrink) | (floats_to_e4m3x2(y.x * shrink, y.y * shrink) << 16);
}

constexpr int kAppendThreads = 128;
constexpr uint32_t kAppendHeads = 4;   // query heads of a thread: they share the angles

// kTask threads a task (32: a warp, 128: the CTA).
template <int H, int kTask>
__global__ void __launch_bounds__(kAppendThreads, 5) fa_cache_append(const AppendArgs p) {
    constexpr int kPerToken = H / 16;                    // threads that share a token
    constexpr int kTokens = kTask / kPerToken;           // tokens at a time
    __shared__ float s_most[kAppendThreads / 32];
    __shared__ uint32_t s_low[kAppendThreads / 32][H / 2], s_high[kAppendThreads / 32][H / 2];
    grid_dep_wait();
    grid_dep_launch();
    const bool bf16 = p.bf16 != 0;

    const uint32_t task_ctas = gridDim.x - p.query_ctas;
    if (blockIdx.x >= task_ctas) {   // ---- queries: 16 values of up to four heads a thread
        const uint32_t fours = (p.q_heads + kAppendHeads - 1) / kAppendHeads, i = (blockIdx.x - task_ctas) * kAppendThreads + threadIdx.x;
        const uint32_t j = i % kPerToken, four = i / kPerToken % fours, row = i / kPerToken / fours, b = row / p.s.T, t = row - b * p.s.T;
        if (b >= p.s.B || !FA_CACHE_OK(p.c.status, kDbgRow, t < p.s.T && four * kAppendHeads < p.q_heads && 16 * j + 16 <= H)) return;
        const uint32_t head = four * kAppendHeads, n = min(kAppendHeads, p.q_heads - head);
        const uint8_t* const from = p.queries + b * p.queries_b + t * p.queries_t + static_cast<int64_t>(head) * (2 * H);
        uint8_t* const out = p.rotated + (static_cast<uint64_t>(row) * p.q_heads + head) * (2 * H) + 16 * j;
        const uint64_t at = static_cast<uint64_t>(max(p.s.lengths[b], 0)) + t;
        const bool there = t < cache_count(p.s, b) && (p.cos == nullptr || at < p.positions);
        RawSixteen raw[kAppendHeads];
#pragma unroll
        for (uint32_t h = 0; h < kAppendHeads; ++h)
            if (there && h < n) raw[h] = load_sixteen<H>(from + h * (2 * H), j);
        Angles angles;
        if (there && p.cos != nullptr) angles = load_angles<H>(p, static_cast<uint32_t>(at), j);
#pragma unroll
        for (uint32_t h = 0; h < kAppendHeads; ++h) {
            if (h >= n) break;
            uint4 x = make_uint4(0, 0, 0, 0), y = x;
            if (there) {
                Sixteen r = unpack_sixteen(raw[h], bf16);
                if (p.cos != nullptr) rotate(r, angles, p.interleaved != 0);
                x = make_uint4(pack_16(r.a[0], r.a[1], bf16), pack_16(r.a[2], r.a[3], bf16), pack_16(r.a[4], r.a[5], bf16), pack_16(r.a[6], r.a[7], bf16));
                y = make_uint4(pack_16(r.b[0], r.b[1], bf16), pack_16(r.b[2], r.b[3], bf16), pack_16(r.b[4], r.b[5], bf16), pack_16(r.b[6], r.b[7], bf16));
            }
            *reinterpret_cast<uint4*>(out + h * (2 * H)) = x;
            *reinterpret_cast<uint4*>(out + h * (2 * H) + H) = y;
        }
        return;
    }

    // ---- one page and head of the keys or the values
    const uint32_t tid = threadIdx.x % kTask, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t task = blockIdx.x * (kAppendThreads / kTask) + threadIdx.x / kTask;
    if (task >= p.tasks) return;   // (whole warps; whole CTAs where a task is one)
    const bool is_v = task & 1u;
    uint32_t rest = task >> 1;
    const uint32_t head = rest % p.c.heads;
    rest /= p.c.heads;
    const uint32_t b = rest / p.blocks, nth = rest % p.blocks;
    const int32_t held_signed = p.s.lengths[b];
    const uint32_t n = cache_count(p.s, b);
    if (n == 0) return;
    const uint32_t held = held_signed < 0 ? 0u : static_cast<uint32_t>(held_signed);
    const uint64_t block = (held >> p.c.page_shift) + static_cast<uint64_t>(nth);
    const uint64_t first = block << p.c.page_shift;               // position of the block's first token
    if (first >= static_cast<uint64_t>(held) + n) return;
    const uint32_t begin = nth == 0 ? held & (p.c.page - 1) : 0u;   // slots [begin, end) are new
    const uint32_t all = static_cast<uint32_t>(min(static_cast<uint64_t>(p.c.page), static_cast<uint64_t>(held) + n - first));
    // (tokens behind the rotation's last position are not appended, neither their keys nor their values)
    const uint32_t end = p.cos == nullptr ? all : static_cast<uint32_t>(min(static_cast<uint64_t>(all), max(static_cast<uint64_t>(p.positions), first) - first));
    int32_t page = -1;
    const bool fits = held_signed >= 0 && block < p.s.width;
    if (fits && FA_CACHE_OK(p.c.status, kDbgEntry, b < p.s.B && block < p.s.width)) page = p.s.table[b * p.s.table_stride + block];   // (asked for ahead of the tokens, used behind them)
    const uint32_t j = tid % kPerToken, sub = tid / kPerToken;
    const uint8_t* rows = is_v ? p.values + b * p.values_b : p.keys + b * p.keys_b;
    const int64_t row_pitch = is_v ? p.values_t : p.keys_t;
    rows += static_cast<int64_t>(head) * (2 * H);
    // Tokens are read for the scale and, from the caches, again for the codes: holding them takes registers that are worth more as
    // CTAs (34 us against 39 with four prompts of up to 2048); the first of each thread is asked for ahead of all else.
    RawSixteen raw;
    auto from = [&](uint32_t slot) {
        if (!FA_CACHE_OK(p.c.status, kDbgRow, b < p.s.B && first + slot >= held && first + slot - held < p.s.T && 16 * j + 16 <= H)) return RawSixteen{};
        return load_sixteen<H>(rows + static_cast<uint32_t>(first + slot - held) * row_pitch, j);
    };
    if (begin + sub < end) raw = from(begin + sub);
    const bool known = static_cast<uint32_t>(page) < p.c.n_pages;
    if (tid == 0 && (!known || end < all)) cache_report(p.c.status, fits && end == all ? kCacheBadPage : kCacheBadPosition);
    if (!known || end <= begin) return;
    const bool turned = !is_v && p.cos != nullptr;
    auto values_of = [&](const RawSixteen& w, uint32_t slot) {
        Sixteen r = unpack_sixteen(w, bf16);
        if (turned) rotate(r, load_angles<H>(p, static_cast<uint32_t>(first) + slot, j), p.interleaved != 0);
        return r;
    };
    auto each = [&](auto&& f) {   // f(slot, values) for this thread's new tokens
        for (uint32_t slot = begin + sub; slot < end; slot += kTokens) f(slot, values_of(slot == begin + sub ? raw : from(slot), slot));
    };
    float* const scale_at = (is_v ? p.c.v_scale : p.c.k_scale) + static_cast<size_t>(page) * p.c.heads + head;
    const float before = begin != 0 ? *scale_at : 0.0f;

    // the largest magnitude, NaN if a value is; for keys from the lowest and highest value by dimension, whose codes are the bounds
    // (rounding keeps their order)
    float most = 0.0f;
    float lowest[16], highest[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) lowest[i] = __int_as_float(0x7F800000), highest[i] = __int_as_float(0xFF800000);
    if (is_v) {
        each([&](uint32_t, const Sixteen& r) {
#pragma unroll
            for (int i = 0; i < 8; ++i) most = max_nan(max_nan(most, fabsf(r.a[i])), fabsf(r.b[i]));
        });
    } else {
        each([&](uint32_t, const Sixteen& r) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                lowest[i] = min_nan(lowest[i], r.a[i]), highest[i] = max_nan(highest[i], r.a[i]);
                lowest[8 + i] = min_nan(lowest[8 + i], r.b[i]), highest[8 + i] = max_nan(highest[8 + i], r.b[i]);
            }
        });
        if (begin + sub < end)
#pragma unroll
            for (int i = 0; i < 16; ++i) most = max_nan(max_nan(most, -lowest[i]), highest[i]);
    }
    if (!(most < __int_as_float(0x7F800000))) most = __int_as_float(0x7F800000);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
    if (kTask > 32) {
        if (lane == 0) s_most[warp] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kAppendThreads / 32; ++w) most = fmaxf(most, s_most[w]);
    }
    float scale = append_scale(most);
    if (begin != 0) scale = larger_scale(before, scale);
    const bool good = scale == scale;
    // (a power of two: the product is the quotient)
    const float inverse = good ? 1.0f / scale : 0.0f;

    uint8_t* const base = (is_v ? p.c.v + static_cast<int64_t>(page) * p.c.v_page + static_cast<int64_t>(head) * p.c.v_head
                                : p.c.k + static_cast<int64_t>(page) * p.c.k_page + static_cast<int64_t>(head) * p.c.k_head);
    const int64_t pitch = is_v ? p.c.v_token : p.c.k_token;
    const bool grown = begin != 0 && !(before == scale);
    const float shrink = good ? before * inverse : 0.0f;
    if (grown) {   // the tokens that the page held move to the larger scale
        for (uint32_t slot = sub; slot < begin; slot += kTokens) {
            if (!FA_CACHE_OK(p.c.status, kDbgCodes, slot < p.c.page && static_cast<uint32_t>(page) < p.c.n_pages)) break;
            uint4* const at = reinterpret_cast<uint4*>(base + slot * pitch + 16 * j);
            uint4 w = *at;
            w.x = good ? moved_codes(w.x, shrink) : 0u;
            w.y = good ? moved_codes(w.y, shrink) : 0u;
            w.z = good ? moved_codes(w.z, shrink) : 0u;
            w.w = good ? moved_codes(w.w, shrink) : 0u;
            *at = w;
        }
    }
    each([&](uint32_t slot, const Sixteen& r) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = good ? floats_to_e4m3x2(r.a[2 * i] * inverse, r.a[2 * i + 1] * inverse) : 0u;
            w[4 + i] = good ? floats_to_e4m3x2(r.b[2 * i] * inverse, r.b[2 * i + 1] * inverse) : 0u;
        }
        if (!FA_CACHE_OK(p.c.status, kDbgCodes, slot < p.c.page && static_cast<uint32_t>(page) < p.c.n_pages && 16 * j + 16 <= H)) return;
        uint8_t* const at = base + slot * pitch + 8 * j;
        *reinterpret_cast<uint2*>(at) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
        *reinterpret_cast<uint2*>(at + H / 2) = make_uint2(w[4] | (w[5] << 16), w[6] | (w[7] << 16));
    });
    if (!is_v) {
        uint32_t low[8], high[8];   // fp16 pairs: the bounds of the thread's dimensions
        const bool some = begin + sub < end;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            low[i] = some ? (good ? e4m3x2_to_half2(floats_to_e4m3x2(lowest[2 * i] * inverse, lowest[2 * i + 1] * inverse)) : 0u) : 0x7C007C00u;
            high[i] = some ? (good ? e4m3x2_to_half2(floats_to_e4m3x2(highest[2 * i] * inverse, highest[2 * i + 1] * inverse)) : 0u) : 0xFC00FC00u;
#pragma unroll
            for (int d = 16; d >= kPerToken; d >>= 1) {
                low[i] = half2_min(low[i], __shfl_xor_sync(0xFFFFFFFFu, low[i], d));
                high[i] = half2_max(high[i], __shfl_xor_sync(0xFFFFFFFFu, high[i], d));
            }
        }
        if (kTask > 32) {
            if (lane < kPerToken)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t d2 = (i < 4 ? 0 : H / 4) + 4 * lane + (i & 3);   // pair of dimensions
                    s_low[warp][d2] = low[i];
                    s_high[warp][d2] = high[i];
                }
            __syncthreads();
        }
        if (tid < kPerToken && FA_CACHE_OK(p.c.status, kDbgCodes, static_cast<uint32_t>(page) < p.c.n_pages && head < p.c.heads)) {
            uint8_t* const bounds = p.c.bounds + (static_cast<size_t>(page) * p.c.heads + head) * (2 * H);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t lo[4], hi[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    lo[i] = low[4 * half + i], hi[i] = high[4 * half + i];
                    if (kTask > 32) {
                        const uint32_t d2 = half * (H / 4) + 4 * j + i;
#pragma unroll
                        for (int w = 0; w < kAppendThreads / 32; ++w) lo[i] = half2_min(lo[i], s_low[w][d2]), hi[i] = half2_max(hi[i], s_high[w][d2]);
                    }
                }
                uint2* const lo_at = reinterpret_cast<uint2*>(bounds + half * (H / 2) + 8 * j);
                uint2* const hi_at = reinterpret_cast<uint2*>(bounds + H + half * (H / 2) + 8 * j);
                if (begin != 0) {
                    const uint2 ol = *lo_at, oh = *hi_at;
                    uint32_t was[4], x[4];
                    was[0] = ol.x, was[1] = ol.y, was[2] = oh.x, was[3] = oh.y;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (grown) was[i] = good ? moved_codes(was[i], shrink) : 0u;
                    }
                    e4m3x4_to_half2(was[0], x[0], x[1]);
                    e4m3x4_to_half2(was[1], x[2], x[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) lo[i] = half2_min(lo[i], x[i]);
                    e4m3x4_to_half2(was[2], x[0], x[1]);
                    e4m3x4_to_half2(was[3], x[2], x[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) hi[i] = half2_max(hi[i], x[i]);
                }
                auto codes = [](uint32_t x, uint32_t y) {
                    const float2 u = unpack_half2(x), v = unpack_half2(y);
                    return floats_to_e4m3x2(u.x, u.y) | (floats_to_e4m3x2(v.x, v.y) << 16);
                };
                *lo_at = make_uint2(codes(lo[0], lo[1]), codes(lo[2], lo[3]));
                *hi_at = make_uint2(codes(hi[0], hi[1]), codes(hi[2], hi[3]));
            }
        }
    }
    if (tid == 0) *scale_at = scale;   // (every thread of the task has read the old one: the reductions lie in between)
}

}  // namespace fa
