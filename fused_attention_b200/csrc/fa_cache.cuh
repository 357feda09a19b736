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
