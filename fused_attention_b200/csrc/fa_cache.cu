// C entry points of the paged 8-bit key/value cache (include/fa_b200.h): checks, the choice of a kernel, launches.
#include <atomic>
#include <cstdint>

#include "fa_b200.h"
#include "fa_cache.cuh"
#include "fa_cache_append.cuh"
#include "fa_cache_prompt.cuh"
#include "fa_cache_rows.cuh"
#include "fa_cache_select.cuh"

namespace {

constexpr int kMaxDevices = 64;

// What is asked of a device once.
struct Device {
    std::atomic<int> sms{0};   // 0: not asked yet
    std::atomic<uint64_t> attr_done{0};   // bit per kernel instance whose shared-memory attribute is set
};
Device g_device[kMaxDevices];

int device_of(int device, Device** out) {
    if (device < 0 || device >= kMaxDevices) return static_cast<int>(cudaErrorInvalidDevice);
    Device& d = g_device[device];
    if (d.sms.load(std::memory_order_acquire) == 0) {
        int major = 0, sms = 0;
        cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return static_cast<int>(e);
        if (major != 10) return FA_B200_ERR_ARCH;
        d.sms.store(sms, std::memory_order_release);
    }
    *out = &d;
    return FA_B200_OK;
}

// Makes `device` current for a call and puts the old one back.
struct OnDevice {
    int before = -1, rc = 0;
    bool changed = false;
    explicit OnDevice(int device) {
        cudaError_t e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != device) {
            e = cudaSetDevice(device);
            changed = e == cudaSuccess;
        }
        rc = static_cast<int>(e);
    }
    ~OnDevice() {
        if (changed) (void)cudaSetDevice(before);
    }
};

// (the kernels wait for the one before them on the stream before they touch memory)
template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), uint32_t grid, uint32_t block, size_t smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

template <typename Kernel>
int allow_smem(Device& d, uint32_t bit, Kernel* kernel, int bytes) {
    if (d.attr_done.load(std::memory_order_acquire) & (1ull << bit)) return FA_B200_OK;   // (setting it twice is harmless)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    d.attr_done.fetch_or(1ull << bit, std::memory_order_release);
    return FA_B200_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool multiple16(int64_t x) { return (x & 15) == 0; }
bool head_dim_ok(uint32_t H) { return H == 16 || H == 32 || H == 64 || H == 128; }
bool page_ok(uint32_t p) { return p == 16 || p == 32 || p == 64 || p == 128; }
// log2(e) / sqrt(H)
float scale_log2(uint32_t H) {
    return static_cast<float>(1.4426950408889634 / (H == 16 ? 4.0 : H == 32 ? 5.656854249492381 : H == 64 ? 8.0 : 11.313708498984761));
}
uint32_t log2_of(uint32_t p) { return p == 16 ? 4 : p == 32 ? 5 : p == 64 ? 6 : 7; }

int view_of(const fa_b200_cache* c, fa::CacheView* v) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->bounds || !c->status) return FA_B200_ERR_NULL_POINTER;
    if (!head_dim_ok(c->head_dim)) return FA_B200_ERR_HEAD_DIM;
    if (!page_ok(c->page_size)) return FA_B200_ERR_PAGE;
    if (c->n_pages == 0 || c->n_pages > 0x7FFFFFFFu || c->kv_heads == 0) return FA_B200_ERR_SHAPE;
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->bounds) || !multiple16(c->k_page_stride) || !multiple16(c->k_head_stride) ||
        !multiple16(c->k_token_stride) || !multiple16(c->v_page_stride) || !multiple16(c->v_head_stride) || !multiple16(c->v_token_stride) ||
        (reinterpret_cast<uintptr_t>(c->k_scale) & 3u) || (reinterpret_cast<uintptr_t>(c->v_scale) & 3u) || (reinterpret_cast<uintptr_t>(c->status) & 3u))
        return FA_B200_ERR_ALIGNMENT;
    // strides that 32 bits hold (offsets are 64-bit numbers): what a page or a token is apart, in bytes
    for (int64_t stride : {c->k_page_stride, c->k_head_stride, c->k_token_stride, c->v_page_stride, c->v_head_stride, c->v_token_stride})
        if (stride < 0 || stride > 0x7FFFFFFFll) return FA_B200_ERR_SHAPE;
    if (c->k_token_stride > (1 << 24) || c->v_token_stride > (1 << 24)) return FA_B200_ERR_SHAPE;
    v->k = static_cast<uint8_t*>(c->k);
    v->v = static_cast<uint8_t*>(c->v);
    v->k_scale = c->k_scale;
    v->v_scale = c->v_scale;
    v->bounds = static_cast<uint8_t*>(c->bounds);
    v->status = c->status;
    v->k_page = c->k_page_stride, v->k_head = c->k_head_stride, v->k_token = c->k_token_stride;
    v->v_page = c->v_page_stride, v->v_head = c->v_head_stride, v->v_token = c->v_token_stride;
    v->n_pages = c->n_pages, v->heads = c->kv_heads, v->page = c->page_size, v->page_shift = log2_of(c->page_size);
    return FA_B200_OK;
}

int seqs_of(const fa_b200_sequences* s, const fa::CacheView& c, fa::CacheSeqs* out) {
    if (!s || !s->table || !s->lengths) return FA_B200_ERR_NULL_POINTER;
    if (s->B == 0 || s->T == 0 || s->table_width == 0 || s->B > (1u << 24) || s->T > (1u << 24) ||
        s->table_width > (0x7FFFFFFFu >> c.page_shift))   // positions are 31-bit numbers
        return FA_B200_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(s->table) | reinterpret_cast<uintptr_t>(s->lengths) | reinterpret_cast<uintptr_t>(s->counts)) & 3u)
        return FA_B200_ERR_ALIGNMENT;
    out->table = s->table, out->lengths = s->lengths, out->counts = s->counts, out->table_stride = s->table_stride;
    out->width = s->table_width, out->B = s->B, out->T = s->T;
    return FA_B200_OK;
}

// Rows of 16-bit values: base and strides in elements, all rows on 16-byte boundaries.
int rows_ok(const void* base, int64_t batch_stride, int64_t token_stride) {
    if (!base) return FA_B200_ERR_NULL_POINTER;
    return aligned16(base) && multiple16(2 * batch_stride) && multiple16(2 * token_stride) ? FA_B200_OK : FA_B200_ERR_ALIGNMENT;
}

constexpr uint64_t kMostCtas = 0x7FFFFFFFull;

// Checked build: what a call writes is filled with NaN (or places far outside) beforehand.
#ifdef FA_DEBUG
int poison(void* p, uint64_t bytes, int value, cudaStream_t stream) { return static_cast<int>(cudaMemsetAsync(p, value, bytes, stream)); }
#define FA_CACHE_FILL(p, bytes, value, stream) if (const int poisoned = poison(p, bytes, value, stream)) return poisoned
#else
#define FA_CACHE_FILL(p, bytes, value, stream) do {} while (0)
#endif

// ----------------------------------------------------------------------------- attention for few rows
struct RowsPlan {
    uint32_t mt, rows, row_tiles, grid, min_units;
    uint64_t problems, units;   // units: of one problem, at most
    uint64_t o_bytes, ml_bytes, share_bytes;
    uint64_t scratch() const { return 16 + o_bytes + ml_bytes + share_bytes; }
};

RowsPlan plan_rows(uint32_t H, uint32_t heads, uint32_t group, uint32_t page, uint32_t B, uint32_t T, uint32_t width, uint32_t keep, uint32_t sms) {
    RowsPlan r = {};
    // One m-tile or two.  With more than 16 rows the second reads the keys once for 32 of them (32 rows on 16 sequences of 2000 tokens:
    // 36 us, 39 with one, which takes the keys twice; 64 rows on 64 of 4000: 305 and 360); with 16 or fewer it is work for nothing
    // (64 sequences of 4000 tokens: 96 us with one, 148 with two).
    if (keep != 0) {   // a problem has rows of one token
        r.rows = group;
        if (group > 32)
            for (r.rows = 32; group % r.rows != 0;) --r.rows;
        r.mt = r.rows > 16 ? 2 : 1;
        r.row_tiles = T * (group / r.rows);
    } else {
        const uint64_t all = static_cast<uint64_t>(T) * group;
        r.mt = all > 16 ? 2 : 1;
        r.rows = static_cast<uint32_t>(all < 16u * r.mt ? all : 16u * r.mt);
        r.row_tiles = static_cast<uint32_t>((all + r.rows - 1) / r.rows);
    }
    const uint64_t tokens = static_cast<uint64_t>(keep != 0 ? keep : width) * page;
    r.units = (tokens + fa::kRowsUnit - 1) / fa::kRowsUnit;
    r.problems = static_cast<uint64_t>(B) * heads * r.row_tiles;   // (below 2^31 in every call that is taken)
    const uint64_t ctas = static_cast<uint64_t>(sms) * (r.mt == 1 ? 3 : 2), all_units = r.problems * r.units;
    // Problems of up to 512 tokens are not divided, those of up to 1024 where there is one for every CTA: joining costs more than what
    // is left of them takes.  (Tables of 512 tokens: 1 sequence of 8 heads 9.7 us, divided 10.5, 16 sequences 10.3 and 14.3; of 1024:
    // 1 sequence 14.7 and 10.4, 32 sequences of any lengths 21.5 and 19.1, 64 27.6 and 29.1, 256 74 and 84; of 2048: 64 41.5 and 41.1.)
    // Two units a CTA at least: with one the same times, with four 12.3 us for 10.2 (1 sequence of 1000).
    r.min_units = r.units <= 4 || (r.units <= 8 && r.problems >= ctas) ? 0 : 2;
    r.grid = static_cast<uint32_t>(r.min_units == 0 ? r.problems : ctas < all_units ? ctas : all_units);
    const uint64_t slots = r.min_units == 0 ? 0 : 2ull * r.grid * 16 * r.mt;
    r.o_bytes = slots * H * 4;
    r.ml_bytes = slots * 8;
    r.share_bytes = r.problems * 8;
    return r;
}

template <int H, int MT>
int launch_rows(Device& d, uint32_t bit, const fa::RowsArgs& a, const RowsPlan& plan, cudaStream_t stream) {
    using Cfg = fa::RowsCfg<H, MT>;
    const int rest = a.bf16 ? fa::kRestNone : MT == 1 && plan.rows <= 8 ? fa::kRestAbove : fa::kRestApart;
    const auto kernel = rest == fa::kRestNone    ? &fa::fa_cache_rows<H, MT, fa::kRestNone>
                        : rest == fa::kRestApart ? &fa::fa_cache_rows<H, MT, fa::kRestApart>
                                                 : &fa::fa_cache_rows<H, MT, MT == 1 ? fa::kRestAbove : fa::kRestApart>;
    int rc = allow_smem(d, bit + 8 * static_cast<uint32_t>(rest), kernel, Cfg::kSmem);
    if (rc == FA_B200_OK) rc = launch(kernel, plan.grid, fa::kRowsWarps * 32, Cfg::kSmem, stream, a);
    if (rc != FA_B200_OK || plan.min_units == 0) return rc;
    const uint64_t rows = plan.problems * plan.rows;
    // a problem has about grid / problems parts, and one more.  A warp a row, or a CTA a row where there are eight or more: 55 parts 32.4
    // us with a warp and 22.6 with a CTA (the whole call, 1 sequence of 32768 tokens), 14 parts 56.3 and 54.4, 7 parts 94.0 and 93.1, 3.5
    // parts 33.6 and 34.8 (16 of 4096).
    if (plan.grid < 8 * plan.problems) rc = launch(&fa::fa_cache_join_few<H, MT>, static_cast<uint32_t>((rows + fa::kJoinWarps - 1) / fa::kJoinWarps), fa::kJoinWarps * 32, 0, stream, a);
    else rc = launch(&fa::fa_cache_join<H, MT>, static_cast<uint32_t>(rows), fa::kJoinWarps * 32, 0, stream, a);
    return rc;
}
template <int H>
int launch_rows(Device& d, uint32_t bit, const fa::RowsArgs& a, const RowsPlan& plan, cudaStream_t stream) {
    return plan.mt == 1 ? launch_rows<H, 1>(d, bit, a, plan, stream) : launch_rows<H, 2>(d, bit + 1, a, plan, stream);
}

// ----------------------------------------------------------------------------- attention for many rows
struct PromptPlan {
    uint32_t pairs, parts, grid;
    uint64_t whole, items;      // that are not cut; all, with their parts
    uint64_t o_bytes, ml_bytes;
    uint64_t scratch() const { return 16 + o_bytes + ml_bytes; }   // (never none: there is an address then)
};

// Rows from which the tensor tiles of fa_cache_prompt.cuh pay, although they are 256 rows high: us by fa_cache_rows.cuh and by it with
// 32, 64, 96, 128 rows: 1 sequence of 16384 tokens 25 and 34, 34 and 36, 43 and 38, 50 and 40; 64 of 3000 tokens 130 and 223, 243 and
// 227, 357 and 233, 467 and 238; 16 of 1300 tokens with 16 heads of 64 30 and 49, 48 and 49, 67 and 51, 84 and 52.
bool use_prompt(uint32_t group, uint32_t T, uint32_t keep) { return keep == 0 && static_cast<uint64_t>(T) * group >= 64; }
// The kernel for many rows knows a page's place as a 32-bit number of 16 bytes.
bool prompt_reaches(const fa::CacheView& c) {
    const auto end = [&](int64_t page, int64_t token) { return static_cast<uint64_t>(c.n_pages) * page + static_cast<uint64_t>(c.page) * token; };
    return end(c.k_page, c.k_token) < (1ull << 36) && end(c.v_page, c.v_token) < (1ull << 36);
}

// The items of the last, partial round (all, where there are fewer than SMs) are cut into parts of their keys.  In key steps, a
// round costs the steps of an item and about two for its beginning and end, with parts three more (their sums go through memory,
// and a kernel that joins them follows).
PromptPlan plan_prompt(uint32_t H, uint32_t heads, uint32_t group, uint32_t page, uint32_t B, uint32_t T, uint32_t width, uint32_t sms) {
    PromptPlan r = {};
    const uint64_t rows = static_cast<uint64_t>(T) * group;
    r.pairs = static_cast<uint32_t>((rows + 2 * fa::kPromptTile - 1) / (2 * fa::kPromptTile));
    const uint64_t all = static_cast<uint64_t>(B) * heads * r.pairs, tail = all % sms;
    const uint64_t steps = (static_cast<uint64_t>(width) * page + fa::kPromptTile - 1) / fa::kPromptTile;
    r.whole = all, r.parts = 1, r.items = all;
    if (tail != 0) {
        uint64_t best = steps + 2;
        for (uint64_t parts = 2; parts <= 32 && parts <= steps && tail * parts <= 2ull * sms; ++parts) {
            const uint64_t cost = (tail * parts + sms - 1) / sms * ((steps + parts - 1) / parts + 2) + 3;
            if (cost < best) best = cost, r.parts = static_cast<uint32_t>(parts), r.whole = all - tail, r.items = all - tail + tail * parts;
        }
    }
    r.grid = static_cast<uint32_t>(r.items < sms ? r.items : sms);
    r.o_bytes = (r.items - r.whole) * 2 * fa::kPromptTile * H * 4;
    r.ml_bytes = (r.items - r.whole) * 2 * fa::kPromptTile * 8;
    return r;
}

template <int H>
int launch_prompt(Device& d, uint32_t bit, const fa::PromptArgs& a, const PromptPlan& plan, cudaStream_t stream) {
    const int same = a.c.page >= 64 ? 2 : a.c.page == 32 ? 1 : 0;
    const auto kernel = same == 2 ? &fa::fa_cache_prompt<H, 4> : same == 1 ? &fa::fa_cache_prompt<H, 2> : &fa::fa_cache_prompt<H, 1>;
    int rc = allow_smem(d, bit + same, kernel, fa::PromptCfg<H>::kSmemBytes);
    if (rc == FA_B200_OK) rc = launch(kernel, plan.grid, fa::kPromptThreads, fa::PromptCfg<H>::kSmemBytes, stream, a);
    if (rc == FA_B200_OK && plan.parts > 1)
        rc = launch(&fa::fa_cache_prompt_join<H>, static_cast<uint32_t>((plan.items - plan.whole) / plan.parts * 2 * fa::kPromptTile / 4), 128, 0, stream, a);
    return rc;
}

// ----------------------------------------------------------------------------- appending
template <int H>
int launch_append(const fa::AppendArgs& a, bool warp_tasks, uint32_t task_ctas, cudaStream_t stream) {
    return warp_tasks ? launch(&fa::fa_cache_append<H, 32>, task_ctas + a.query_ctas, fa::kAppendThreads, 0, stream, a)
                      : launch(&fa::fa_cache_append<H, 128>, task_ctas + a.query_ctas, fa::kAppendThreads, 0, stream, a);
}

}  // namespace

extern "C" {

int fa_b200_cache_append(const fa_b200_cache* cache, const fa_b200_sequences* sequences, const void* keys, int64_t keys_batch_stride,
                         int64_t keys_token_stride, const void* values, int64_t values_batch_stride, int64_t values_token_stride,
                         const void* queries_or_null, int64_t queries_batch_stride, int64_t queries_token_stride, uint32_t q_heads, void* rotated,
                         const float* cos_or_null, const float* sin_or_null, uint32_t positions, uint32_t dtype, uint32_t flags, int device,
                         void* cuda_stream) {
    fa::AppendArgs a = {};
    int rc = view_of(cache, &a.c);
    if (rc == FA_B200_OK) rc = seqs_of(sequences, a.c, &a.s);
    if (rc == FA_B200_OK) rc = rows_ok(keys, keys_batch_stride, keys_token_stride);
    if (rc == FA_B200_OK) rc = rows_ok(values, values_batch_stride, values_token_stride);
    if (rc == FA_B200_OK && queries_or_null) rc = rows_ok(queries_or_null, queries_batch_stride, queries_token_stride);
    if (rc == FA_B200_OK && queries_or_null) rc = rows_ok(rotated, 0, 0);
    if (rc != FA_B200_OK) return rc;
    if (dtype > FA_B200_BF16) return FA_B200_ERR_DTYPE;
    if (flags & ~FA_B200_CACHE_NEIGHBOURS) return FA_B200_ERR_FLAGS;
    if (queries_or_null && q_heads == 0) return FA_B200_ERR_SHAPE;
    if ((cos_or_null == nullptr) != (sin_or_null == nullptr)) return FA_B200_ERR_NULL_POINTER;
    if (cos_or_null && (!aligned16(cos_or_null) || !aligned16(sin_or_null))) return FA_B200_ERR_ALIGNMENT;
    const uint32_t H = cache->head_dim;
    a.keys = static_cast<const uint8_t*>(keys), a.keys_b = 2 * keys_batch_stride, a.keys_t = 2 * keys_token_stride;
    a.values = static_cast<const uint8_t*>(values), a.values_b = 2 * values_batch_stride, a.values_t = 2 * values_token_stride;
    a.queries = static_cast<const uint8_t*>(queries_or_null), a.queries_b = 2 * queries_batch_stride, a.queries_t = 2 * queries_token_stride;
    a.rotated = static_cast<uint8_t*>(rotated);
    a.cos = cos_or_null, a.sin = sin_or_null, a.positions = positions;
    a.q_heads = q_heads, a.bf16 = dtype == FA_B200_BF16, a.interleaved = flags & FA_B200_CACHE_NEIGHBOURS;
    a.blocks = (a.s.T + a.c.page - 2) / a.c.page + 1;   // that T tokens touch at most
    const uint64_t tasks = 2ull * a.s.B * a.blocks * a.c.heads;
    const uint64_t q_threads = queries_or_null ? static_cast<uint64_t>(a.s.B) * a.s.T * ((q_heads + fa::kAppendHeads - 1) / fa::kAppendHeads) * (H / 16) : 0;
    const uint64_t q_ctas = (q_threads + fa::kAppendThreads - 1) / fa::kAppendThreads;
    if (tasks + q_ctas > kMostCtas || q_threads > 0xFFFFFF00ull) return FA_B200_ERR_SHAPE;
    a.tasks = static_cast<uint32_t>(tasks), a.query_ctas = static_cast<uint32_t>(q_ctas);
    // A warp a task, not a CTA of four: where a task has few tokens, or the tasks fill the device many times over in either form.  (Pages
    // of 64 tokens, 8 heads of 128, us as CTAs and as warps: 32 sequences of 4 tokens 5.3 and 4.5, of 16 6.2 and 8.0; 128 of 16 16.6 and
    // 11.4; 64 of 32 13.4 and 15.7; 128 of 32 28 and 24; 32 of 512 82 and 85; 64 of 512 164 and 158; 4 of 4096 82 and 94.)
    const bool warp_tasks = a.s.T <= 4 || tasks >= 128ull * (a.s.T < a.c.page ? a.s.T : a.c.page);
    const uint32_t task_ctas = static_cast<uint32_t>(warp_tasks ? (tasks + 3) / 4 : tasks);
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    if (queries_or_null) FA_CACHE_FILL(rotated, 2ull * a.s.B * a.s.T * q_heads * H, 0xFF, stream);
    switch (H) {
        case 16: return launch_append<16>(a, warp_tasks, task_ctas, stream);
        case 32: return launch_append<32>(a, warp_tasks, task_ctas, stream);
        case 64: return launch_append<64>(a, warp_tasks, task_ctas, stream);
        default: return launch_append<128>(a, warp_tasks, task_ctas, stream);
    }
}

int fa_b200_cache_select(const fa_b200_cache* cache, const fa_b200_sequences* sequences, const void* queries, int64_t queries_batch_stride,
                         int64_t queries_token_stride, uint32_t q_heads, uint32_t dtype, uint32_t keep, uint32_t first, uint32_t last,
                         int32_t* pages, void* scratch, uint64_t scratch_bytes, int device, void* cuda_stream) {
    fa::SelectArgs a = {};
    int rc = view_of(cache, &a.c);
    if (rc == FA_B200_OK) rc = seqs_of(sequences, a.c, &a.s);
    if (rc == FA_B200_OK) rc = rows_ok(queries, queries_batch_stride, queries_token_stride);
    if (rc != FA_B200_OK) return rc;
    if (!pages || !scratch) return FA_B200_ERR_NULL_POINTER;
    if (dtype > FA_B200_BF16) return FA_B200_ERR_DTYPE;
    if (q_heads == 0 || q_heads % a.c.heads != 0 || keep == 0 || keep > 0x7FFFFFFFu || last == 0) return FA_B200_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(scratch)) & 3u) return FA_B200_ERR_ALIGNMENT;
    const uint64_t rows = static_cast<uint64_t>(a.s.B) * a.s.T * a.c.heads;
    if (rows > kMostCtas) return FA_B200_ERR_SHAPE;
    if (scratch_bytes < 4 * rows * a.s.width) return FA_B200_ERR_TOO_LARGE;
    a.q = static_cast<const uint8_t*>(queries), a.q_b = 2 * queries_batch_stride, a.q_t = 2 * queries_token_stride;
    a.keys = static_cast<uint32_t*>(scratch), a.pages = pages;
    a.group = q_heads / a.c.heads, a.keep = keep, a.first = first, a.last = last, a.bf16 = dtype == FA_B200_BF16;
    // Query rows in tiles of 16: the heads of several tokens, or a part of one token's.
    a.per_tile = a.group > 16 ? 1 : 16 / a.group;
    const uint32_t all_tiles = a.group > 16 ? (a.group + 15) / 16 : (a.s.T + a.per_tile - 1) / a.per_tile;
    a.tiles = all_tiles < fa::kScoreTiles ? all_tiles : fa::kScoreTiles;
    a.turns = a.group > 16 ? (all_tiles + a.tiles - 1) / a.tiles : 1;
    a.token_chunks = a.group > 16 ? a.s.T : (all_tiles + a.tiles - 1) / a.tiles;
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    // as many CTAs as are resident at once, if there are as many units of 64 pages
    const uint64_t problems = static_cast<uint64_t>(a.s.B) * a.c.heads * a.token_chunks, resident = static_cast<uint64_t>(fa::kScoreCtas) * d->sms.load();
    const uint64_t units = problems * ((a.s.width + fa::kScoreWarps * fa::kScorePages - 1) / (fa::kScoreWarps * fa::kScorePages));
    if (units > 0xFFFFFFFFull) return FA_B200_ERR_SHAPE;
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    FA_CACHE_FILL(scratch, 4 * rows * a.s.width, 0xFF, stream);
    FA_CACHE_FILL(pages, 4 * rows * keep, 0x7F, stream);
    const uint32_t grid = static_cast<uint32_t>(units < resident ? units : resident);
    const size_t smem = static_cast<size_t>(a.tiles) * (cache->head_dim / 16) * 2 * 32 * sizeof(uint4);   // 32 KB at most
    constexpr uint32_t kBlock = fa::kScoreWarps * 32;
    switch (cache->head_dim) {
        case 16: rc = launch(&fa::fa_cache_scores<16>, grid, kBlock, smem, stream, a); break;
        case 32: rc = launch(&fa::fa_cache_scores<32>, grid, kBlock, smem, stream, a); break;
        case 64: rc = launch(&fa::fa_cache_scores<64>, grid, kBlock, smem, stream, a); break;
        default: rc = launch(&fa::fa_cache_scores<128>, grid, kBlock, smem, stream, a); break;
    }
    if (rc != FA_B200_OK) return rc;
    const uint32_t per = (a.s.width + fa::kTakeThreads - 1) / fa::kTakeThreads;
    // As many keys of a thread in registers as there are at most (32 queries on 2048 pages: 47.8 us so, 52.9 out of memory, 49.2 with 32;
    // on 313 17.3, 19.9 out of memory, 18.2 with 8, 20.5 with 32; on 8192 147, 244 out of memory).
    if (per <= 2) return launch(&fa::fa_cache_take<2>, static_cast<uint32_t>(rows), fa::kTakeThreads, 0, stream, a);
    if (per <= 8) return launch(&fa::fa_cache_take<8>, static_cast<uint32_t>(rows), fa::kTakeThreads, 0, stream, a);
    if (per <= 32) return launch(&fa::fa_cache_take<32>, static_cast<uint32_t>(rows), fa::kTakeThreads, 0, stream, a);
    return launch(&fa::fa_cache_take<0>, static_cast<uint32_t>(rows), fa::kTakeThreads, 0, stream, a);
}

int fa_b200_cache_attention_scratch(uint32_t head_dim, uint32_t kv_heads, uint32_t q_heads, uint32_t page_size, uint32_t B, uint32_t T,
                                    uint32_t table_width, uint32_t keep, int device, uint64_t out[1]) {
    if (!out) return FA_B200_ERR_NULL_POINTER;
    if (!head_dim_ok(head_dim)) return FA_B200_ERR_HEAD_DIM;
    if (!page_ok(page_size)) return FA_B200_ERR_PAGE;
    if (kv_heads == 0 || q_heads == 0 || q_heads % kv_heads != 0 || B == 0 || T == 0 || table_width == 0) return FA_B200_ERR_SHAPE;
    Device* d = nullptr;
    const int rc = device_of(device, &d);
    if (rc != FA_B200_OK) return rc;
    const uint32_t sms = static_cast<uint32_t>(d->sms.load()), group = q_heads / kv_heads;
    // (which kernel has a call for many rows depends on the cache too: room for either)
    out[0] = plan_rows(head_dim, kv_heads, group, page_size, B, T, table_width, keep, sms).scratch();
    if (use_prompt(group, T, keep)) {
        const uint64_t prompt = plan_prompt(head_dim, kv_heads, group, page_size, B, T, table_width, sms).scratch();
        if (prompt > out[0]) out[0] = prompt;
    }
    return FA_B200_OK;
}

int fa_b200_cache_attention(const fa_b200_cache* cache, const fa_b200_sequences* sequences, const void* queries, int64_t queries_batch_stride,
                            int64_t queries_token_stride, uint32_t q_heads, uint32_t dtype, const int32_t* pages_or_null, uint32_t keep,
                            uint32_t flags, void* y, void* scratch, uint64_t scratch_bytes, int device, void* cuda_stream) {
    fa::RowsArgs a = {};
    int rc = view_of(cache, &a.c);
    if (rc == FA_B200_OK) rc = seqs_of(sequences, a.c, &a.s);
    if (rc == FA_B200_OK) rc = rows_ok(queries, queries_batch_stride, queries_token_stride);
    if (rc == FA_B200_OK) rc = rows_ok(y, 0, 0);
    if (rc != FA_B200_OK) return rc;
    if (!scratch) return FA_B200_ERR_NULL_POINTER;
    if (dtype > FA_B200_BF16) return FA_B200_ERR_DTYPE;
    if (flags & ~FA_B200_CACHE_ALL_KEYS) return FA_B200_ERR_FLAGS;
    if (q_heads == 0 || q_heads % a.c.heads != 0 || (pages_or_null != nullptr) != (keep != 0)) return FA_B200_ERR_SHAPE;
    if (static_cast<uint64_t>(keep) * a.c.page > 0x7FFFFFFFull || static_cast<uint64_t>(a.s.T) * q_heads > 0x7FFFFFFFull) return FA_B200_ERR_SHAPE;
    if (!aligned16(scratch) || (reinterpret_cast<uintptr_t>(pages_or_null) & 3u)) return FA_B200_ERR_ALIGNMENT;
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    const uint32_t H = cache->head_dim;
    if (use_prompt(q_heads / a.c.heads, a.s.T, keep) && prompt_reaches(a.c) && q_heads / a.c.heads < 65536) {
        const PromptPlan plan = plan_prompt(H, a.c.heads, q_heads / a.c.heads, a.c.page, a.s.B, a.s.T, a.s.width, static_cast<uint32_t>(d->sms.load()));
        if (plan.items * (2 * fa::kPromptTile) > kMostCtas) return FA_B200_ERR_SHAPE;
        if (scratch_bytes < plan.scratch()) return FA_B200_ERR_TOO_LARGE;
        fa::PromptArgs b = {};
        b.c = a.c, b.s = a.s;
        b.q = static_cast<const uint8_t*>(queries), b.q_b = 2 * queries_batch_stride, b.q_t = 2 * queries_token_stride;
        b.y = static_cast<uint8_t*>(y), b.group = q_heads / a.c.heads, b.by_group = static_cast<uint32_t>((1ull << 32) / b.group + 1);
        b.causal = (flags & FA_B200_CACHE_ALL_KEYS) ? 0u : 1u, b.bf16 = dtype == FA_B200_BF16;
        b.pairs = plan.pairs, b.parts = plan.parts, b.whole = static_cast<uint32_t>(plan.whole), b.items = static_cast<uint32_t>(plan.items), b.scale_log2 = scale_log2(H);
        b.part_o = static_cast<float*>(scratch);
        b.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(scratch) + plan.o_bytes);
        OnDevice on(device);
        if (on.rc != 0) return on.rc;
        const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
        FA_CACHE_FILL(y, 2ull * a.s.B * a.s.T * q_heads * H, 0xFF, stream);
        FA_CACHE_FILL(scratch, plan.scratch(), 0xFF, stream);
        switch (H) {
            case 16: return launch_prompt<16>(*d, 32, b, plan, stream);
            case 32: return launch_prompt<32>(*d, 35, b, plan, stream);
            case 64: return launch_prompt<64>(*d, 38, b, plan, stream);
            default: return launch_prompt<128>(*d, 41, b, plan, stream);
        }
    }
    const RowsPlan plan = plan_rows(H, a.c.heads, q_heads / a.c.heads, a.c.page, a.s.B, a.s.T, a.s.width, keep, static_cast<uint32_t>(d->sms.load()));
    if (plan.problems * plan.rows > kMostCtas || plan.problems * (plan.units + fa::kRowsSetup) > 0xFFFFFFFFull) return FA_B200_ERR_SHAPE;
    if (scratch_bytes < plan.scratch()) return FA_B200_ERR_TOO_LARGE;
    a.q = static_cast<const uint8_t*>(queries), a.q_b = 2 * queries_batch_stride, a.q_t = 2 * queries_token_stride;
    a.y = static_cast<uint8_t*>(y), a.pages = pages_or_null, a.keep = keep;
    a.group = q_heads / a.c.heads, a.causal = (flags & FA_B200_CACHE_ALL_KEYS) ? 0u : 1u, a.bf16 = dtype == FA_B200_BF16;
    a.rows = plan.rows, a.row_tiles = plan.row_tiles, a.min_units = plan.min_units;
    a.scale_log2 = scale_log2(H);
    uint8_t* const at = static_cast<uint8_t*>(scratch);
    a.part_o = reinterpret_cast<float*>(at);
    a.part_ml = reinterpret_cast<float2*>(at + plan.o_bytes);
    a.shares = reinterpret_cast<int2*>(at + plan.o_bytes + plan.ml_bytes);
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    FA_CACHE_FILL(y, 2ull * a.s.B * a.s.T * q_heads * H, 0xFF, stream);
    FA_CACHE_FILL(scratch, plan.scratch(), 0xFF, stream);
#ifdef FA_DEBUG
    a.slots = plan.min_units == 0 ? 0 : 2ull * plan.grid, a.problems = plan.problems;
#endif
    switch (H) {
        case 16: return launch_rows<16>(*d, 0, a, plan, stream);
        case 32: return launch_rows<32>(*d, 2, a, plan, stream);
        case 64: return launch_rows<64>(*d, 4, a, plan, stream);
        default: return launch_rows<128>(*d, 6, a, plan, stream);
    }
}

}  // extern "C"
