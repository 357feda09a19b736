// C entry points of the paged cache of latent vectors (include/fa_b200.h): checks, the choice of a kernel, launches.
#include <cuda.h>

#include "fa_b200.h"
#include "fa_host.cuh"
#include "fa_latent.cuh"
#include "fa_latent_prompt.cuh"
#include "fa_latent_rows.cuh"

namespace {

constexpr uint64_t kMostCtas = 0x7FFFFFFFull;
constexpr double kLog2e = 1.4426950408889634;

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
std::atomic<EncodeTiledFn> g_encode{nullptr};

// A map of 16-bit values with 128-byte swizzled boxes, zeros outside.  (The encoder needs a current context, which a thread that has not
// called the runtime yet has none of: the device's is bound to it then.)
template <int kDims>
int make_map(CUtensorMap* map, const void* base, const cuuint64_t (&dims)[kDims], const cuuint64_t (&strides)[kDims - 1], const cuuint32_t (&box)[kDims]) {
    EncodeTiledFn encode = g_encode.load(std::memory_order_acquire);
    if (encode == nullptr) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess || fn == nullptr) {
            (void)cudaGetLastError();
            return FA_B200_ERR_DRIVER;
        }
        encode = reinterpret_cast<EncodeTiledFn>(fn);
        g_encode.store(encode, std::memory_order_release);
    }
    cuuint32_t unit[kDims];
    for (int i = 0; i < kDims; ++i) unit[i] = 1;
    auto once = [&] {
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, kDims, const_cast<void*>(base), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = once();
    int device = 0;
    if (r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) r = once();
    return r == CUDA_SUCCESS ? FA_B200_OK : FA_B200_ERR_DRIVER;
}

int view_of(const fa_b200_latent_cache* c, fa::LatentView* v) {
    if (!c || !c->data || !c->status) return FA_B200_ERR_NULL_POINTER;
    if ((c->latent_dim != 128 && c->latent_dim != 256 && c->latent_dim != 512) || (c->rope_dim != 16 && c->rope_dim != 32 && c->rope_dim != 64)) return FA_B200_ERR_HEAD_DIM;
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return FA_B200_ERR_PAGE;
    if (c->n_pages == 0 || c->n_pages > 0x7FFFFFFEu) return FA_B200_ERR_SHAPE;
    if (!aligned16(c->data) || !multiple16(c->page_stride) || !multiple16(c->token_stride) || (reinterpret_cast<uintptr_t>(c->status) & 3u)) return FA_B200_ERR_ALIGNMENT;
    if (c->page_stride < 0 || c->token_stride < 0 || c->page_stride > 0x7FFFFFFFll || c->token_stride > (1 << 24)) return FA_B200_ERR_SHAPE;
    v->data = static_cast<uint8_t*>(c->data), v->status = c->status;
    v->page_stride = c->page_stride, v->token_stride = c->token_stride;
    v->n_pages = c->n_pages, v->page = c->page_size, v->latent = c->latent_dim, v->rope = c->rope_dim;
    v->page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    return FA_B200_OK;
}
int seqs_of(const fa_b200_sequences* s, const fa::LatentView& c, fa::CacheSeqs* out) {
    if (!s || !s->table || !s->lengths) return FA_B200_ERR_NULL_POINTER;
    if (s->B == 0 || s->T == 0 || s->table_width == 0 || s->B > (1u << 24) || s->T > (1u << 24) || s->table_width > (0x7FFFFFFFu >> c.page_shift)) return FA_B200_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(s->table) | reinterpret_cast<uintptr_t>(s->lengths) | reinterpret_cast<uintptr_t>(s->counts)) & 3u) return FA_B200_ERR_ALIGNMENT;
    out->table = s->table, out->lengths = s->lengths, out->counts = s->counts, out->table_stride = s->table_stride;
    out->width = s->table_width, out->B = s->B, out->T = s->T;
    return FA_B200_OK;
}
int rows_ok(const void* base, std::initializer_list<int64_t> strides) {
    if (!base) return FA_B200_ERR_NULL_POINTER;
    if (!aligned16(base)) return FA_B200_ERR_ALIGNMENT;
    for (const int64_t s : strides)
        if (!multiple16(2 * s)) return FA_B200_ERR_ALIGNMENT;
    return FA_B200_OK;
}

// (so that its product with log2 e is a normal number too)
bool scale_ok(float scale) { return scale >= 0x1p-126f && scale <= 1e38f; }

struct LatentPlan {
    uint32_t n, groups, group_rows, parts, least;
    uint64_t rows, o_bytes, ml_bytes, share_bytes;
    uint64_t scratch() const { return 16 + o_bytes + ml_bytes + share_bytes; }
};
LatentPlan plan_rows(uint32_t latent, uint32_t heads, uint32_t page, uint32_t B, uint32_t T, uint32_t width, uint32_t sms) {
    LatentPlan r = {};
    r.rows = static_cast<uint64_t>(T) * heads;
    // As few groups as there can be, of equal size.
    r.groups = static_cast<uint32_t>((r.rows + 63) / 64);
    r.group_rows = static_cast<uint32_t>((r.rows + r.groups - 1) / r.groups);
    r.n = (r.group_rows + 15) / 16 * 16;
    r.groups = static_cast<uint32_t>((r.rows + r.group_rows - 1) / r.group_rows);
    const uint64_t each = (static_cast<uint64_t>(width) * page + fa::kLatentTile - 1) / fa::kLatentTile, tiles = B * each;   // at most
    // Two tiles a CTA at least (us, with 1, 2, 3 and 4 or 8: 1 sequence of 1000 tokens 16 heads 10.0, 10.4, -, 13.7; 128 heads 14.6, 14.5, 17.1,
    // 18.6; 4 of 2000 32 heads 16.5, 13.7, 17.3, 15.3; 1 of 4000 128 heads 20.8, 17.4, 18.2, 18.6).
    r.least = 2;
    // As many parts as fill the SMs, in one round, or in up to four where fewer would leave more than a tenth of them idle.
    uint64_t parts = 1;
    double best = 0;
    for (uint64_t rounds = 1; rounds <= 4 && best < 0.9; ++rounds) {
        const uint64_t x = rounds * sms / r.groups;
        const double busy = static_cast<double>(x * r.groups) / static_cast<double>(rounds * sms);
        if (x > 0 && busy > best) best = busy, parts = x;
    }
    const uint64_t most = (tiles + r.least - 1) / r.least;
    r.parts = static_cast<uint32_t>(parts < most ? parts : most);
    // Sequences that the table has little room for are not divided where they give a quarter of the SMs something to do: what would be left of them
    // takes less than joining, which costs the more the more rows there are.  It is the table's width that decides, since lengths are known on the
    // device alone: short sequences in a wide table are divided.  (64 of 500 to 1000 tokens, 128 heads, with L2 flushed: 47 us in a table of 1024
    // tokens, 62 in one of 131072; 16 heads 35 and 33.  In tables as wide as the longest, us whole and divided: 64 sequences of 100 to 512 tokens,
    // 16 heads, 16.6 and 19.8, 16 of them 15.7 and 14.8, 1 of 301 12.1 and 9.8, 64 of 500 to 1000 26.7 and 23.7; 128 heads, 64 of 100 to 512 25 and 42, of 500 to
    // 1000 39 and 54.)
    if (each <= (r.n <= 32 ? 8u : 16u) && static_cast<uint64_t>(B) * r.groups >= sms / 4) r.parts = B, r.least = 0;
    const uint64_t slots = r.parts == 1 || r.least == 0 ? 0 : 2ull * r.parts * r.groups;
    r.o_bytes = slots * r.n * latent * 4;
    r.ml_bytes = slots * r.n * 8;
    r.share_bytes = static_cast<uint64_t>(B) * 8;
    return r;
}

template <int LC, int N>
int launch_rows(Device& d, uint32_t bit, const CUtensorMap& map, const fa::LatentRowsArgs& a, cudaStream_t stream) {
    int rc = allow_smem(d, bit, &fa::fa_latent_rows<LC, N>, fa::LatentCfg<LC, N>::kSmemBytes);
    if (rc == FA_B200_OK) rc = launch(&fa::fa_latent_rows<LC, N>, a.parts * a.groups, fa::kLatentThreads, fa::LatentCfg<LC, N>::kSmemBytes, stream, map, a);
    if (rc != FA_B200_OK || a.parts == 1 || a.least == 0) return rc;
    // a sequence has about parts / B parts, and one more
    const uint32_t items = a.s.B * a.rows * (LC / 2);
    if (a.parts >= 8 * a.s.B) return launch(&fa::fa_latent_join<LC, N, true>, items, fa::kLatentJoinWarps * 32, 0, stream, a);
    return launch(&fa::fa_latent_join<LC, N, false>, (items + fa::kLatentJoinWarps - 1) / fa::kLatentJoinWarps, fa::kLatentJoinWarps * 32, 0, stream, a);
}
template <int LC>
int launch_rows(Device& d, uint32_t bit, const CUtensorMap& map, const fa::LatentRowsArgs& a, uint32_t n, cudaStream_t stream) {
    return n == 16   ? launch_rows<LC, 16>(d, bit, map, a, stream)
           : n == 32 ? launch_rows<LC, 32>(d, bit + 1, map, a, stream)
           : n == 48 ? launch_rows<LC, 48>(d, bit + 2, map, a, stream)
                     : launch_rows<LC, 64>(d, bit + 3, map, a, stream);
}

template <int NOPE, bool kBf16>
int launch_prompt(Device& d, uint32_t bit, uint32_t ctas, cudaStream_t stream, const CUtensorMap& q, const CUtensorMap& qr, const CUtensorMap& kv, const CUtensorMap& r,
                  const fa::ExpandArgs& a) {
    const int rc = allow_smem(d, bit, &fa::fa_latent_prompt<NOPE, kBf16>, fa::ExpandCfg<NOPE>::kSmemBytes);
    if (rc != FA_B200_OK) return rc;
    return launch(&fa::fa_latent_prompt<NOPE, kBf16>, ctas, fa::kExpandThreads, fa::ExpandCfg<NOPE>::kSmemBytes, stream, q, qr, kv, r, a);
}

}  // namespace

extern "C" {

int fa_b200_latent_append(const fa_b200_latent_cache* cache, const fa_b200_sequences* sequences, const void* latents, int64_t latents_batch_stride,
                          int64_t latents_token_stride, const void* rope_keys, int64_t keys_batch_stride, int64_t keys_token_stride, const void* queries_or_null,
                          int64_t queries_batch_stride, int64_t queries_token_stride, int64_t queries_head_stride, uint32_t heads, void* rotated_keys,
                          void* rotated_queries, const float* cos_or_null, const float* sin_or_null, uint32_t positions, uint32_t dtype, uint32_t flags, int device,
                          void* cuda_stream) {
    fa::LatentAppendArgs a = {};
    int rc = view_of(cache, &a.c);
    if (rc == FA_B200_OK) rc = seqs_of(sequences, a.c, &a.s);
    if (rc == FA_B200_OK) rc = rows_ok(latents, {latents_batch_stride, latents_token_stride});
    if (rc == FA_B200_OK) rc = rows_ok(rope_keys, {keys_batch_stride, keys_token_stride});
    if (rc == FA_B200_OK) rc = rows_ok(rotated_keys, {});
    if (rc == FA_B200_OK && queries_or_null) rc = rows_ok(queries_or_null, {queries_batch_stride, queries_token_stride, queries_head_stride});
    if (rc == FA_B200_OK && queries_or_null) rc = rows_ok(rotated_queries, {});
    if (rc != FA_B200_OK) return rc;
    if (dtype > FA_B200_BF16) return FA_B200_ERR_DTYPE;
    if (flags & ~FA_B200_CACHE_NEIGHBOURS) return FA_B200_ERR_FLAGS;
    if ((queries_or_null && heads == 0) || heads > (1u << 20)) return FA_B200_ERR_SHAPE;
    if ((cos_or_null == nullptr) != (sin_or_null == nullptr)) return FA_B200_ERR_NULL_POINTER;
    if (cos_or_null && (!aligned16(cos_or_null) || !aligned16(sin_or_null))) return FA_B200_ERR_ALIGNMENT;
    a.latents = static_cast<const uint8_t*>(latents), a.latents_b = 2 * latents_batch_stride, a.latents_t = 2 * latents_token_stride;
    a.keys = static_cast<const uint8_t*>(rope_keys), a.keys_b = 2 * keys_batch_stride, a.keys_t = 2 * keys_token_stride;
    a.queries = static_cast<const uint8_t*>(queries_or_null), a.queries_b = 2 * queries_batch_stride, a.queries_t = 2 * queries_token_stride;
    a.queries_h = 2 * queries_head_stride, a.heads = queries_or_null ? heads : 0;
    a.keys_out = static_cast<uint8_t*>(rotated_keys), a.queries_out = static_cast<uint8_t*>(rotated_queries);
    a.cos = cos_or_null, a.sin = sin_or_null, a.positions = positions;
    a.bf16 = dtype == FA_B200_BF16, a.interleaved = flags & FA_B200_CACHE_NEIGHBOURS;
    const uint64_t ctas = static_cast<uint64_t>(a.s.B) * a.s.T;
    if (ctas > kMostCtas) return FA_B200_ERR_SHAPE;
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    const uint32_t work = a.c.latent / 8 + a.c.rope / 16 * (1 + a.heads), threads = (work + 31) / 32 * 32;
    return launch(&fa::fa_latent_append, static_cast<uint32_t>(ctas), threads < fa::kLatentAppendThreads ? threads : fa::kLatentAppendThreads, 0,
                  static_cast<cudaStream_t>(cuda_stream), a);
}

int fa_b200_latent_attention_scratch(uint32_t latent_dim, uint32_t heads, uint32_t page_size, uint32_t B, uint32_t T, uint32_t table_width, int device, uint64_t out[1]) {
    if (!out) return FA_B200_ERR_NULL_POINTER;
    if (latent_dim != 128 && latent_dim != 256 && latent_dim != 512) return FA_B200_ERR_HEAD_DIM;
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return FA_B200_ERR_PAGE;
    if (heads == 0 || B == 0 || T == 0 || table_width == 0) return FA_B200_ERR_SHAPE;
    Device* d = nullptr;
    const int rc = device_of(device, &d);
    if (rc != FA_B200_OK) return rc;
    out[0] = plan_rows(latent_dim, heads, page_size, B, T, table_width, static_cast<uint32_t>(d->sms.load())).scratch();
    return FA_B200_OK;
}

int fa_b200_latent_attention(const fa_b200_latent_cache* cache, const fa_b200_sequences* sequences, const void* q_latent, int64_t ql_batch_stride,
                             int64_t ql_token_stride, int64_t ql_head_stride, const void* q_rope, int64_t qr_batch_stride, int64_t qr_token_stride,
                             int64_t qr_head_stride, uint32_t heads, float scale, uint32_t dtype, uint32_t flags, void* y, void* scratch, uint64_t scratch_bytes,
                             int device, void* cuda_stream) {
    fa::LatentRowsArgs a = {};
    int rc = view_of(cache, &a.c);
    if (rc == FA_B200_OK) rc = seqs_of(sequences, a.c, &a.s);
    if (rc == FA_B200_OK) rc = rows_ok(q_latent, {ql_batch_stride, ql_token_stride, ql_head_stride});
    if (rc == FA_B200_OK) rc = rows_ok(q_rope, {qr_batch_stride, qr_token_stride, qr_head_stride});
    if (rc == FA_B200_OK) rc = rows_ok(y, {});
    if (rc != FA_B200_OK) return rc;
    if (!scratch) return FA_B200_ERR_NULL_POINTER;
    if (!aligned16(scratch)) return FA_B200_ERR_ALIGNMENT;
    if (dtype > FA_B200_BF16) return FA_B200_ERR_DTYPE;
    if (flags & ~FA_B200_CACHE_ALL_KEYS) return FA_B200_ERR_FLAGS;
    if (heads == 0 || !scale_ok(scale)) return FA_B200_ERR_SHAPE;
    if (static_cast<uint64_t>(a.s.T) * heads > 0x3FFFFFFFull) return FA_B200_ERR_SHAPE;
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    const LatentPlan plan = plan_rows(a.c.latent, heads, a.c.page, a.s.B, a.s.T, a.s.width, static_cast<uint32_t>(d->sms.load()));
    const uint64_t tiles = static_cast<uint64_t>(a.s.B) * ((static_cast<uint64_t>(a.s.width) << a.c.page_shift) / fa::kLatentTile + 1);
    if (tiles > 0xFFFFFFFFull || static_cast<uint64_t>(plan.parts) * plan.groups > kMostCtas || a.s.B * plan.rows * (a.c.latent / 128) > kMostCtas) return FA_B200_ERR_SHAPE;
    if (scratch_bytes < plan.scratch()) return FA_B200_ERR_TOO_LARGE;
    a.q_latent = static_cast<const uint8_t*>(q_latent), a.ql_b = 2 * ql_batch_stride, a.ql_t = 2 * ql_token_stride, a.ql_h = 2 * ql_head_stride;
    a.q_rope = static_cast<const uint8_t*>(q_rope), a.qr_b = 2 * qr_batch_stride, a.qr_t = 2 * qr_token_stride, a.qr_h = 2 * qr_head_stride;
    a.y = static_cast<uint8_t*>(y);
    a.heads = heads, a.rows = static_cast<uint32_t>(plan.rows), a.groups = plan.groups, a.group_rows = plan.group_rows, a.parts = plan.parts, a.least = plan.least;
    a.causal = (flags & FA_B200_CACHE_ALL_KEYS) ? 0u : 1u, a.bf16 = dtype == FA_B200_BF16;
    a.scale_log2 = static_cast<float>(scale * kLog2e);
    uint8_t* const at = static_cast<uint8_t*>(scratch);
    a.part_o = reinterpret_cast<float*>(at);
    a.part_ml = reinterpret_cast<float2*>(at + plan.o_bytes);
    a.shares = reinterpret_cast<int2*>(at + plan.o_bytes + plan.ml_bytes);
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    CUtensorMap map;
    const cuuint64_t dims[3] = {a.c.latent + a.c.rope, a.c.page, a.c.n_pages};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.c.token_stride), static_cast<cuuint64_t>(a.c.page_stride)};
    const cuuint32_t box[3] = {64, a.c.page < fa::kLatentTile ? a.c.page : fa::kLatentTile, 1};
    if ((rc = make_map<3>(&map, a.c.data, dims, strides, box)) != FA_B200_OK) return rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
#ifdef FA_DEBUG
    if (const cudaError_t e = cudaMemsetAsync(y, 0xFF, 2ull * a.s.B * plan.rows * a.c.latent, stream)) return static_cast<int>(e);
    if (const cudaError_t e = cudaMemsetAsync(scratch, 0xFF, plan.scratch(), stream)) return static_cast<int>(e);
#endif
    switch (a.c.latent) {
        case 128: return launch_rows<2>(*d, 0, map, a, plan.n, stream);
        case 256: return launch_rows<4>(*d, 4, map, a, plan.n, stream);
        default: return launch_rows<8>(*d, 8, map, a, plan.n, stream);
    }
}

int fa_b200_latent_prompt(const void* q_nope, int64_t qn_batch_stride, int64_t qn_token_stride, int64_t qn_head_stride, const void* q_rope, int64_t qr_batch_stride,
                          int64_t qr_token_stride, int64_t qr_head_stride, const void* expanded, int64_t kv_batch_stride, int64_t kv_token_stride,
                          int64_t kv_head_stride, const void* rope_keys, int64_t rk_batch_stride, int64_t rk_token_stride, const int32_t* lengths_or_null,
                          const int32_t* counts_or_null, uint32_t B, uint32_t T, uint32_t S, uint32_t heads, uint32_t nope_dim, uint32_t rope_dim, float scale,
                          uint32_t dtype, uint32_t flags, void* y, int device, void* cuda_stream) {
    int rc = rows_ok(q_nope, {qn_batch_stride, qn_token_stride, qn_head_stride});
    if (rc == FA_B200_OK) rc = rows_ok(q_rope, {qr_batch_stride, qr_token_stride, qr_head_stride});
    if (rc == FA_B200_OK) rc = rows_ok(expanded, {kv_batch_stride, kv_token_stride, kv_head_stride});
    if (rc == FA_B200_OK) rc = rows_ok(rope_keys, {rk_batch_stride, rk_token_stride});
    if (rc == FA_B200_OK) rc = rows_ok(y, {});
    if (rc != FA_B200_OK) return rc;
    if ((reinterpret_cast<uintptr_t>(lengths_or_null) | reinterpret_cast<uintptr_t>(counts_or_null)) & 3u) return FA_B200_ERR_ALIGNMENT;
    if ((nope_dim != 64 && nope_dim != 128) || (rope_dim != 16 && rope_dim != 32 && rope_dim != 64)) return FA_B200_ERR_HEAD_DIM;
    if (dtype > FA_B200_BF16) return FA_B200_ERR_DTYPE;
    if (flags & ~FA_B200_CACHE_ALL_KEYS) return FA_B200_ERR_FLAGS;
    if (B == 0 || T == 0 || S == 0 || heads == 0 || B > (1u << 24) || T > 0x3FFFFFFFu || S > 0x3FFFFFFFu || heads > (1u << 20) || !scale_ok(scale)) return FA_B200_ERR_SHAPE;
    const uint64_t pairs = (static_cast<uint64_t>(T) + 2 * fa::kExpandTile - 1) / (2 * fa::kExpandTile), items = pairs * B * heads;
    if (static_cast<uint64_t>(B) * heads > kMostCtas || items > kMostCtas) return FA_B200_ERR_SHAPE;
    fa::ExpandArgs a = {};
    a.lengths = lengths_or_null, a.counts = counts_or_null, a.y = static_cast<uint8_t*>(y);
    a.B = B, a.T = T, a.S = S, a.heads = heads, a.pairs = static_cast<uint32_t>(pairs), a.rope = rope_dim;
    a.causal = (flags & FA_B200_CACHE_ALL_KEYS) ? 0u : 1u, a.scale_log2 = static_cast<float>(scale * kLog2e);
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    // {dimensions, heads, tokens, sequences}; boxes of 64 dimensions of one head by 128 tokens.  An axis of one is nowhere stepped along.
    auto map_of = [&](CUtensorMap* map, const void* base, uint32_t dim, uint32_t n_heads, uint32_t tokens, int64_t batch, int64_t token, int64_t head) {
        const cuuint64_t dims[4] = {dim, n_heads, tokens, B};
        const cuuint64_t strides[3] = {static_cast<cuuint64_t>(n_heads > 1 ? 2 * head : 16), static_cast<cuuint64_t>(tokens > 1 ? 2 * token : 16),
                                       static_cast<cuuint64_t>(B > 1 ? 2 * batch : 16)};
        const cuuint32_t box[4] = {64, 1, fa::kExpandTile, 1};
        return make_map<4>(map, base, dims, strides, box);
    };
    for (const int64_t stride : {B > 1 ? qn_batch_stride : 1, T > 1 ? qn_token_stride : 1, heads > 1 ? qn_head_stride : 1, B > 1 ? qr_batch_stride : 1,
                                 T > 1 ? qr_token_stride : 1, heads > 1 ? qr_head_stride : 1, B > 1 ? kv_batch_stride : 1, S > 1 ? kv_token_stride : 1,
                                 heads > 1 ? kv_head_stride : 1, B > 1 ? rk_batch_stride : 1, S > 1 ? rk_token_stride : 1})
        if (stride <= 0 || stride >= (1ll << 38)) return FA_B200_ERR_SHAPE;
    CUtensorMap q, qr, kv, r;
    rc = map_of(&q, q_nope, nope_dim, heads, T, qn_batch_stride, qn_token_stride, qn_head_stride);
    if (rc == FA_B200_OK) rc = map_of(&qr, q_rope, rope_dim, heads, T, qr_batch_stride, qr_token_stride, qr_head_stride);
    if (rc == FA_B200_OK) rc = map_of(&kv, expanded, 2 * nope_dim, heads, S, kv_batch_stride, kv_token_stride, kv_head_stride);
    if (rc == FA_B200_OK) rc = map_of(&r, rope_keys, rope_dim, 1, S, rk_batch_stride, rk_token_stride, 0);
    if (rc != FA_B200_OK) return rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
#ifdef FA_DEBUG
    if (const cudaError_t e = cudaMemsetAsync(y, 0xFF, 2ull * B * T * heads * nope_dim, stream)) return static_cast<int>(e);
#endif
    const uint32_t ctas = static_cast<uint32_t>(items);
    if (nope_dim == 64) return dtype == FA_B200_BF16 ? launch_prompt<64, true>(*d, 12, ctas, stream, q, qr, kv, r, a) : launch_prompt<64, false>(*d, 13, ctas, stream, q, qr, kv, r, a);
    return dtype == FA_B200_BF16 ? launch_prompt<128, true>(*d, 14, ctas, stream, q, qr, kv, r, a) : launch_prompt<128, false>(*d, 15, ctas, stream, q, qr, kv, r, a);
}

int fa_b200_latent_status(int device, uint32_t out[2]) {
    if (!out) return FA_B200_ERR_NULL_POINTER;
    Device* d = nullptr;
    const int rc = device_of(device, &d);
    if (rc != FA_B200_OK) return rc;
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(out, fa::g_latent_status, 2 * sizeof(uint32_t));
    if (e == cudaSuccess && (out[0] != 0 || out[1] != 0)) {
        const uint32_t zero[2] = {0, 0};
        e = cudaMemcpyToSymbol(fa::g_latent_status, zero, sizeof(zero));
    }
    return static_cast<int>(e);
}

}  // extern "C"
