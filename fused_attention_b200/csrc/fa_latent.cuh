// The paged cache of latent vectors: what its kernels share, and appending to it.
//
// A token has one row of 16-bit values for all heads: `latent` dimensions that are key and value at once, behind them `rope` more that
// are rotated by the token's position and belong to the key alone.  A page holds `page` rows (16, 32, 64 or 128).  Table entries, lengths
// and counts are looked at before they are used, as in fa_cache.cuh.
#pragma once

#include "fa_cache.cuh"

namespace fa {

struct LatentView {
    uint8_t* data;
    uint32_t* status;
    int64_t page_stride, token_stride;   // bytes
    uint32_t n_pages, page, page_shift, latent, rope;
};
// (for cache_length and its like)
__device__ __forceinline__ CacheView plain_view(const LatentView& v) {
    CacheView c = {};
    c.status = v.status, c.n_pages = v.n_pages, c.page = v.page, c.page_shift = v.page_shift;
    return c;
}

// ----------------------------------------------------------------------------- append
// Bound by memory for prompts (4 of up to 2048 tokens, 32 heads of 64, 60 MB with the zeros of queries past `counts`: 15 to 19 us, 3 to 4 TB/s;
// asking for the rows ahead of the length, and so for absent tokens' too, took 18), by the launch and length -> table entry -> row for single
// tokens (128 of them 2.3 us in a graph, 6.7 a call).
//
// A CTA a token, a thread 16 bytes of the latent vector or 16 values of a rotary part: one of the key's, one of a query head's.  Products
// and sums of the rotation are rounded one by one in fp32, its results once to the tensors' type.
struct LatentAppendArgs {
    LatentView c;
    CacheSeqs s;
    const uint8_t* latents;
    const uint8_t* keys;
    const uint8_t* queries;   // null: none
    uint8_t* keys_out;        // [B, T, rope] contiguous
    uint8_t* queries_out;     // [B, T, heads, rope] contiguous
    const float* cos;         // [positions, rope / 2]; null: no rotation
    const float* sin;
    int64_t latents_b, latents_t, keys_b, keys_t, queries_b, queries_t, queries_h;   // strides in bytes
    uint32_t positions, heads, bf16, interleaved;
};

__device__ __forceinline__ void turn_pair(float& x, float& y, float c, float s) {
    const float u = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
    y = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
    x = u;
}
// 16 values of a rotary part of `rope`: [8 j, 8 j + 8) and [rope / 2 + 8 j, ...) as halves, [16 j, 16 j + 16) as neighbours.
__device__ __forceinline__ void latent_turn(uint4 (&w)[2], const LatentAppendArgs& p, uint32_t position, uint32_t j) {
    float x[16];
    const uint32_t in[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 y = unpack_16(in[i], p.bf16 != 0);
        x[2 * i] = y.x, x[2 * i + 1] = y.y;
    }
    const size_t at = static_cast<size_t>(position) * (p.c.rope / 2) + 8 * j;
    float c[8], s[8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const float4 a = *reinterpret_cast<const float4*>(p.cos + at + 4 * q), b = *reinterpret_cast<const float4*>(p.sin + at + 4 * q);
        c[4 * q] = a.x, c[4 * q + 1] = a.y, c[4 * q + 2] = a.z, c[4 * q + 3] = a.w;
        s[4 * q] = b.x, s[4 * q + 1] = b.y, s[4 * q + 2] = b.z, s[4 * q + 3] = b.w;
    }
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn_pair(x[2 * i], x[2 * i + 1], c[i], s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn_pair(x[i], x[8 + i], c[i], s[i]);
    }
    uint32_t out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = pack_16(x[2 * i], x[2 * i + 1], p.bf16 != 0);
    w[0] = make_uint4(out[0], out[1], out[2], out[3]);
    w[1] = make_uint4(out[4], out[5], out[6], out[7]);
}

constexpr int kLatentAppendThreads = 256;   // at most
__global__ void __launch_bounds__(kLatentAppendThreads) fa_latent_append(const LatentAppendArgs p) {
    grid_dep_wait();
    grid_dep_launch();
    const uint32_t b = blockIdx.x / p.s.T, t = blockIdx.x - b * p.s.T;
    const uint32_t pieces = p.c.latent / 8, units = p.c.rope / 16, all = pieces + units * (1 + p.heads);
    const int32_t held = p.s.lengths[b];
    const uint64_t at = static_cast<uint64_t>(max(held, 0)) + t;
    const bool mine = t < cache_count(p.s, b), rotated = p.cos != nullptr && at < p.positions, turned = mine && (p.cos == nullptr || rotated);
    int32_t page = -1;
    const bool inside = turned && held >= 0 && at < (static_cast<uint64_t>(p.s.width) << p.c.page_shift);
    if (inside) page = p.s.table[b * p.s.table_stride + static_cast<int64_t>(at >> p.c.page_shift)];
    const bool there = inside && static_cast<uint32_t>(page) < p.c.n_pages;
    if (mine && !there && threadIdx.x == 0) cache_report(p.c.status, inside ? kCacheBadPage : kCacheBadPosition);
    uint8_t* const row = p.c.data + (there ? static_cast<uint32_t>(page) * p.c.page_stride + static_cast<int64_t>(at & (p.c.page - 1)) * p.c.token_stride : 0);
    // where a unit's two pieces lie in their rotary part, in bytes
    for (uint32_t i = threadIdx.x; i < all; i += blockDim.x) {
        if (i < pieces) {
            if (there) *reinterpret_cast<uint4*>(row + 16 * i) = *reinterpret_cast<const uint4*>(p.latents + b * p.latents_b + t * p.latents_t + 16 * i);
            continue;
        }
        const uint32_t u = i - pieces, head = u / units, j = u - head * units;   // (head 0: the key)
        const uint32_t first = p.interleaved ? 32 * j : 16 * j, second = p.interleaved ? 32 * j + 16 : p.c.rope + 16 * j;
        const uint8_t* const from = head == 0 ? p.keys + b * p.keys_b + t * p.keys_t : p.queries + b * p.queries_b + t * p.queries_t + (head - 1) * p.queries_h;
        uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (turned) {
            w[0] = *reinterpret_cast<const uint4*>(from + first);
            w[1] = *reinterpret_cast<const uint4*>(from + second);
            if (rotated) latent_turn(w, p, static_cast<uint32_t>(at), j);
        }
        uint8_t* const to = head == 0 ? p.keys_out + static_cast<uint64_t>(blockIdx.x) * (2 * p.c.rope)
                                      : p.queries_out + (static_cast<uint64_t>(blockIdx.x) * p.heads + head - 1) * (2 * p.c.rope);
        *reinterpret_cast<uint4*>(to + first) = w[0];
        *reinterpret_cast<uint4*>(to + second) = w[1];
        if (head == 0 && there) {
            *reinterpret_cast<uint4*>(row + 2 * p.c.latent + first) = w[0];
            *reinterpret_cast<uint4*>(row + 2 * p.c.latent + second) = w[1];
        }
    }
}

}  // namespace fa
