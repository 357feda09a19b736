// The paged 8-bit key/value cache: what its kernels share.
//
// A page holds `page` tokens (16, 32, 64 or 128) of every key/value head: e4m3 codes, and per page and head one fp32 scale for
// the keys and one for the values; a value is code * scale.  Beside the keys lie their bounds, the lowest and the highest code
// by dimension.  What is read from device memory to find a page (a table entry, a length, a count, a selected page) is looked
// at before it is used: a page outside the cache is not touched, its tokens are left out, and the cache's status word says so.
#pragma once

#include <cuda_bf16.h>

#include "fa_ptx.cuh"

namespace fa {

// What a kernel writes into the first word of the cache's status block (the second counts the reports).
constexpr uint32_t kCacheBadPage = 1u;       // a table entry or selected page outside the cache or the table
constexpr uint32_t kCacheBadPosition = 2u;   // a token behind the table's or the rotation's last position, or a negative length
constexpr uint32_t kCacheTimeout = 0x100u;   // a bounded wait expired (the role and barrier in the bits above and below)

struct CacheView {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;      // [n_pages, heads]
    float* v_scale;
    uint8_t* bounds;     // [n_pages, heads, 2, H]
    uint32_t* status;    // two words
    int64_t k_page, k_head, k_token;   // strides in bytes
    int64_t v_page, v_head, v_token;
    uint32_t n_pages, heads, page, page_shift;
};

// Where the tokens of the sequences are.
struct CacheSeqs {
    const int32_t* table;     // [B, width], rows `table_stride` apart
    const int32_t* lengths;   // [B]
    const int32_t* counts;    // [B] or null: T of each
    int64_t table_stride;
    uint32_t width, B, T;
};

__device__ __forceinline__ void cache_report(uint32_t* status, uint32_t code) {
    atomicCAS(status, 0u, code);
    atomicAdd(status + 1, 1u);
}

// ----------------------------------------------------------------------------- checked build (-DFA_DEBUG)
// Where an address is formed, of a table entry, a list, a scale, bounds or codes, a row of a tensor, a place of a tile in shared memory or of
// scratch, the checked build looks at its indexes first.  A failed check leaves kRoleDebug | <what> in the cache's status word and skips
// the access.  Tiles in shared memory are filled with NaN before anything is copied there, and the launcher fills outputs and scratch
// with NaN before the launch.  (Tensor memory: fa_ptx.cuh.)  Normal builds contain none of this.
#ifdef FA_DEBUG
enum : uint32_t {
    kDbgEntry = 0x20,   // of a table or a list of pages
    kDbgCodes,          // codes, scales or bounds outside the cache
    kDbgRow,            // a row of queries, keys, values, angles or results outside its tensor
    kDbgTile,           // outside a tile in shared memory
    kDbgScratch         // outside the call's scratch
};
__device__ __forceinline__ bool cache_checked(uint32_t* status, uint32_t what, bool ok) {
    if (!ok) cache_report(status, kRoleDebug | what);
    return ok;
}
__device__ __forceinline__ void cache_poison(uint32_t base, uint32_t bytes) {   // all threads of the CTA
    for (uint32_t off = threadIdx.x * 16u; off + 16u <= bytes; off += blockDim.x * 16u)
        st_shared_v4(base + off, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu);
    __syncthreads();
}
#define FA_CACHE_OK(status, what, cond) cache_checked(status, what, cond)
#define FA_CACHE_POISON(base, bytes) cache_poison(base, bytes)
#else
#define FA_CACHE_OK(status, what, cond) true
#define FA_CACHE_POISON(base, bytes) do {} while (0)
#endif

// Tokens that sequence b holds, as far as the table has room for them.
__device__ __forceinline__ uint32_t cache_length(const CacheView& c, const CacheSeqs& s, uint32_t b) {
    const int32_t n = s.lengths[b];
    const uint64_t room = static_cast<uint64_t>(s.width) << c.page_shift;
    return n < 0 ? 0u : static_cast<uint32_t>(min(static_cast<uint64_t>(n), room));
}
__device__ __forceinline__ bool cache_length_ok(const CacheView& c, const CacheSeqs& s, uint32_t b) {
    return s.lengths[b] >= 0 && static_cast<uint64_t>(s.lengths[b]) <= (static_cast<uint64_t>(s.width) << c.page_shift);
}
__device__ __forceinline__ uint32_t cache_count(const CacheSeqs& s, uint32_t b) {
    if (s.counts == nullptr) return s.T;
    const int32_t n = s.counts[b];
    return n < 0 ? 0u : min(static_cast<uint32_t>(n), s.T);
}

// ----------------------------------------------------------------------------- work dealt out by the device
// Sequences have units of work (below 2^32 in all), sequence b units(b) * per_seq; CTA c of C takes `each` from c * each +
// min(c, more) on, the first `more` CTAs one more.  C is the grid, or fewer so that each has `least`.  Lengths are only known on the
// device, so every CTA adds up the units itself.  s_share (8 + kWarps words): what share_owner needs to know.
constexpr int kShareWords = 8;
__device__ __forceinline__ uint32_t share_owner(const uint32_t* s_share, uint32_t unit) {
    const uint32_t each = s_share[3], more = s_share[4], longer = more * (each + 1);
    return unit < longer ? unit / (each + 1) : more + (unit - longer) / each;
}
// False: this CTA has none.  b: the sequence of its first unit; before: units in front of b.  `alike`: all sequences have as many.
template <int kWarps, typename Units>
__device__ __forceinline__ bool share_of(const Units& units, bool alike, uint32_t B, uint32_t per_seq, uint32_t least, uint32_t* s_share, uint32_t& unit,
                                         uint32_t& unit_end, uint32_t& b, uint32_t& before) {
    constexpr uint32_t kThreads = kWarps * 32;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    uint32_t* const s_sum = s_share + kShareWords;
    // the units of all sequences; with up to kThreads of them every thread keeps what lies in front of its own
    uint32_t total = 0, mine = 0, upto = 0;
    if (alike) {
        mine = units(0) * per_seq;
        total = mine * B;
    } else {
        for (uint32_t i = tid; i < B; i += kThreads) mine += units(i);
        mine *= per_seq;
        upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += x;
        }
        if (lane == 31) s_sum[warp] = upto;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
            if (w < warp) upto += s_sum[w];
            total += s_sum[w];
        }
    }
    const uint32_t ctas = min(gridDim.x, (total + least - 1) / least), each = total / ctas, more = total - each * ctas, c = blockIdx.x;
    if (c >= ctas) return false;
    if (tid == 0) s_share[3] = each, s_share[4] = more;
    unit = c * each + min(c, more);
    unit_end = (c + 1) * each + min(c + 1, more);
    before = 0;
    if (alike) {
        b = unit / mine;
        before = b * mine;
    } else if (B <= kThreads) {
        if (tid < B && unit < upto && unit >= upto - mine) s_share[0] = tid, s_share[1] = upto - mine;
        __syncthreads();
        b = s_share[0], before = s_share[1];
    } else {
        for (uint32_t b0 = 0; b0 < B; b0 += 32) {   // every warp adds up 32 sequences at a time
            const uint32_t mine32 = b0 + lane < B ? units(b0 + lane) * per_seq : 0u;
            uint32_t upto32 = mine32;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, upto32, d);
                if (lane >= d) upto32 += x;
            }
            const uint32_t behind = __ballot_sync(0xFFFFFFFFu, before + upto32 > unit);
            if (behind != 0) {
                const uint32_t at = __ffs(behind) - 1;
                b = b0 + at;
                before += __shfl_sync(0xFFFFFFFFu, upto32 - mine32, at);
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, upto32, 31);
        }
    }
    return true;
}

// ----------------------------------------------------------------------------- e4m3 <-> fp16
// Two codes (the lower 16 bits) -> two fp16 values; every e4m3 value is one of fp16.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo;\n\tcvt.u16.u32 lo, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(four));
}
// To nearest even; beyond the range to its end.  `lo` in the lower byte.
__device__ __forceinline__ uint32_t floats_to_e4m3x2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b16 t;\n\tcvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}

// ----------------------------------------------------------------------------- sums of weights whose value scales lie far apart
// The value scale is part of a weight's exponent, w = 2^(s + log2 scale - M), and the row's sum takes it out again, w / scale.  Where scales
// lie further apart than this many bits (pages of zeros, 2^-100, beside values of 100 and more) a weight that counts in the sum can be
// less than the smallest fp32 number: 2^(s - M) is then an exponential of its own.  (95: what is lost up to there is below 2^-29 of the
// largest weight; where the weights are multiplied, in fp16, all below 2^-25 is.)
constexpr int kSpanOfScales = 95;
// s - M lies between -121 and 108 for scales of 2^-100 to 2^120: exponentials are taken of it and 12, near the middle.
constexpr float kSumLift = 12.0f, kSumUnlift = 0x1p-12f;
// A scale; one below zero, which no append writes, is not a number.
__device__ __forceinline__ float scale_or_nan(float x) { return x < 0.0f ? __int_as_float(0x7FC00000) : x; }
// x * 2^d for d <= 0, also where 2^d is less than the smallest fp32 number.  (A d that is not a number counts as a small one.)
__device__ __forceinline__ float times_power(float x, float d) {
    const float y = x * ex2_approx(fmaxf(d, -126.0f));
    return d < -126.0f ? y * ex2_approx(d + 126.0f) : y;
}

__device__ __forceinline__ float2 unpack_half2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 unpack_16(uint32_t w, bool bf16) {
    if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return unpack_half2(w);
}
// Two floats rounded once to the tensor's type.
__device__ __forceinline__ uint32_t pack_16(float lo, float hi, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&p);
    }
    return pack_half2(lo, hi);
}

}  // namespace fa
