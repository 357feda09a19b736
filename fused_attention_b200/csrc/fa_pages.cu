// C entry points of the pages of a cache (include/fa_b200.h): checks and launches.
#include "fa_b200.h"
#include "fa_host.cuh"
#include "fa_pages.cuh"

namespace {

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int pages_of(const fa_b200_pages* pages, fa::PagesView* v) {
    if (!pages || !pages->refs || !pages->status) return FA_B200_ERR_NULL_POINTER;
    if (!aligned4(pages->refs) || !aligned4(pages->status)) return FA_B200_ERR_ALIGNMENT;
    if (pages->n_pages == 0 || pages->n_pages >= (1u << 30)) return FA_B200_ERR_SHAPE;
    v->refs = pages->refs, v->status = pages->status, v->n = pages->n_pages;
    return FA_B200_OK;
}
int table_of(const int32_t* table, int64_t stride, uint32_t width, uint32_t B, fa::PagesTable* t) {
    if (!table) return FA_B200_ERR_NULL_POINTER;
    if (!aligned4(table)) return FA_B200_ERR_ALIGNMENT;
    if (width == 0 || B == 0 || B > (1u << 24) || width > 0x7FFFFFFFu) return FA_B200_ERR_SHAPE;
    t->at = const_cast<int32_t*>(table), t->stride = stride, t->width = width, t->B = B;
    return FA_B200_OK;
}

// Of what every address in an array of pages is a multiple.
uint64_t unit_of(const void* base, int64_t page_stride, uint32_t n0, int64_t stride0, uint32_t n1, int64_t stride1, uint32_t row) {
    const uint64_t all = reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(page_stride) | row | (n0 > 1 ? static_cast<uint64_t>(stride0) : 0) |
                         (n1 > 1 ? static_cast<uint64_t>(stride1) : 0);
    return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
}
// An array in as few rows as it lies in.  What a thread takes at a time is decided by those and where they begin: rows that lie behind one another may
// make one of a multiple of 16 bytes that does not begin on such a boundary.
int area_of(const fa_b200_copy_area& x, fa::CopyArea* y) {
    if (!x.base) return FA_B200_ERR_NULL_POINTER;
    if (x.n0 == 0 || x.n1 == 0 || x.row_bytes == 0 || static_cast<uint64_t>(x.n0) * x.n1 > 0x7FFFFFFFull) return FA_B200_ERR_SHAPE;
    if (unit_of(x.base, x.page_stride, x.n0, x.stride0, x.n1, x.stride1, x.row_bytes) < (x.row_bytes % 16 == 0 ? 16u : 4u)) return FA_B200_ERR_ALIGNMENT;
    y->base = static_cast<uint8_t*>(x.base), y->page = x.page_stride, y->stride0 = x.stride0, y->stride1 = x.stride1;
    y->n0 = x.n0, y->n1 = x.n1, y->row = x.row_bytes;
    if (y->n1 > 1 && y->stride1 == y->row && static_cast<uint64_t>(y->row) * y->n1 < (1u << 31)) y->row *= y->n1, y->n1 = 1;
    if (y->n0 > 1 && y->n1 == 1 && y->stride0 == y->row && static_cast<uint64_t>(y->row) * y->n0 < (1u << 31)) y->row *= y->n0, y->n0 = 1;
    y->unit = static_cast<uint32_t>(unit_of(y->base, y->page, y->n0, y->stride0, y->n1, y->stride1, y->row));
    return FA_B200_OK;
}

constexpr uint32_t kForkMost = 57344;   // sequences whose entries of one column fit shared memory
constexpr int kForkSmem = 4 * kForkMost;

}  // namespace

extern "C" {

int fa_b200_pages_fork(const fa_b200_pages* pages, int32_t* table, int64_t table_stride, uint32_t table_width, uint32_t B, int32_t* lengths,
                       const int32_t* parents, int device, void* cuda_stream) {
    fa::ForkArgs a = {};
    int rc = pages_of(pages, &a.v);
    if (rc == FA_B200_OK) rc = table_of(table, table_stride, table_width, B, &a.t);
    if (rc != FA_B200_OK) return rc;
    if (!lengths || !parents) return FA_B200_ERR_NULL_POINTER;
    if (!aligned4(lengths) || !aligned4(parents)) return FA_B200_ERR_ALIGNMENT;
    if (B > kForkMost) return FA_B200_ERR_TOO_LARGE;
    a.lengths = lengths, a.parents = parents;
    a.cols = 4 * B <= kForkMost ? 4 : 1;
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    if ((rc = allow_smem(*d, 0, &fa::fa_pages_fork, kForkSmem)) != FA_B200_OK) return rc;
    return launch(&fa::fa_pages_fork, (table_width + a.cols - 1) / a.cols + 1, fa::kForkThreads, 4ull * B * a.cols, static_cast<cudaStream_t>(cuda_stream), a);
}

int fa_b200_pages_reserve(const fa_b200_pages* pages, int32_t* table, int64_t table_stride, uint32_t table_width, uint32_t B, const int32_t* lengths,
                          const int32_t* counts_or_null, uint32_t count, uint32_t page_size, int32_t* granted, int32_t* sources, int32_t* targets,
                          void* scratch, uint64_t scratch_bytes, int device, void* cuda_stream) {
    fa::ReserveArgs a = {};
    int rc = pages_of(pages, &a.v);
    if (rc == FA_B200_OK) rc = table_of(table, table_stride, table_width, B, &a.t);
    if (rc != FA_B200_OK) return rc;
    if (!lengths || !granted || !sources || !targets || !scratch) return FA_B200_ERR_NULL_POINTER;
    for (const void* p : {static_cast<const void*>(lengths), static_cast<const void*>(counts_or_null), static_cast<const void*>(granted),
                          static_cast<const void*>(sources), static_cast<const void*>(targets), static_cast<const void*>(scratch)})
        if (!aligned4(p)) return FA_B200_ERR_ALIGNMENT;
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return FA_B200_ERR_PAGE;
    if (count > 0x7FFFFFFFu) return FA_B200_ERR_SHAPE;
    if (scratch_bytes < 4ull * a.v.n) return FA_B200_ERR_TOO_LARGE;
    a.lengths = lengths, a.counts = counts_or_null, a.count = count;
    a.granted = granted, a.sources = sources, a.targets = targets, a.list = static_cast<int32_t*>(scratch);
    a.page_shift = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    a.alone = B <= fa::kAloneRows && static_cast<uint64_t>(B) * table_width <= fa::kAloneEntries;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    if (!a.alone) {
        const uint32_t ctas = (B + fa::kReserveWarps - 1) / fa::kReserveWarps, sms = static_cast<uint32_t>(d->sms.load());
        if ((rc = launch(&fa::fa_pages_release, ctas < sms ? ctas : sms, fa::kReserveThreads, 0, stream, a)) != FA_B200_OK) return rc;
    }
    return launch(&fa::fa_pages_reserve, 1, fa::kReserveThreads, 0, stream, a);
}

int fa_b200_pages_compact(const fa_b200_pages* pages, const int32_t* table, int64_t table_stride, uint32_t table_width, uint32_t B, int32_t* new_refs,
                          int32_t* new_table, int32_t* sources, int32_t* targets, void* scratch, uint64_t scratch_bytes, int device, void* cuda_stream) {
    fa::CompactArgs a = {};
    int rc = pages_of(pages, &a.v);
    if (rc == FA_B200_OK) rc = table_of(table, table_stride, table_width, B, &a.t);
    if (rc != FA_B200_OK) return rc;
    if (!new_refs || !new_table || !sources || !targets || !scratch) return FA_B200_ERR_NULL_POINTER;
    for (const void* p : {static_cast<const void*>(new_refs), static_cast<const void*>(new_table), static_cast<const void*>(sources),
                          static_cast<const void*>(targets), static_cast<const void*>(scratch)})
        if (!aligned4(p)) return FA_B200_ERR_ALIGNMENT;
    if (scratch_bytes < 4ull * a.v.n + 8) return FA_B200_ERR_TOO_LARGE;
    a.new_refs = new_refs, a.new_table = new_table, a.sources = sources, a.targets = targets;
    a.totals = static_cast<uint32_t*>(scratch), a.rank = static_cast<int32_t*>(scratch) + 2;
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    rc = launch(&fa::fa_pages_plan, (a.v.n + fa::kCompactPages - 1) / fa::kCompactPages, fa::kCompactThreads, 0, stream, a);
    if (rc != FA_B200_OK) return rc;
    const uint64_t entries = static_cast<uint64_t>(B) * table_width, items = entries > a.v.n ? entries : a.v.n, ctas = (items + 255) / 256;
    const uint64_t most = 8ull * static_cast<uint64_t>(d->sms.load());
    return launch(&fa::fa_pages_renumber, static_cast<uint32_t>(ctas < most ? ctas : most), 256, 0, stream, a);
}

int fa_b200_cache_copy(const fa_b200_copy_area* areas, uint32_t n_areas, uint32_t n_pages, const int32_t* sources, const int32_t* targets, uint32_t pairs,
                       uint32_t* status, int device, void* cuda_stream) {
    if (!areas || !sources || !targets || !status) return FA_B200_ERR_NULL_POINTER;
    if (!aligned4(sources) || !aligned4(targets) || !aligned4(status)) return FA_B200_ERR_ALIGNMENT;
    if (n_areas == 0 || n_pages == 0 || n_pages > 0x7FFFFFFFu || pairs == 0 || pairs > 0x7FFFFFFFu) return FA_B200_ERR_SHAPE;
    int rc = FA_B200_OK;
    for (uint32_t i = 0; i < n_areas; ++i) {
        fa::CopyArea y = {};
        if ((rc = area_of(areas[i], &y)) != FA_B200_OK) return rc;
    }
    Device* d = nullptr;
    if ((rc = device_of(device, &d)) != FA_B200_OK) return rc;
    OnDevice on(device);
    if (on.rc != 0) return on.rc;
    const uint32_t sms = static_cast<uint32_t>(d->sms.load());
    for (uint32_t first = 0; first < n_areas; first += fa::kCopyAreas) {
        fa::CopyArgs a = {};
        a.sources = sources, a.targets = targets, a.status = status, a.pairs = pairs, a.n = n_pages;
        a.areas = n_areas - first < fa::kCopyAreas ? n_areas - first : fa::kCopyAreas;
        // Eight CTAs an SM in all, if there are as many parts of 16 KB (half of what a CTA has in flight at once) and more.
        const uint32_t ctas = 8 * sms, share = (ctas + pairs - 1) / pairs;
        uint32_t parts = 0;
        for (uint32_t i = 0; i < a.areas; ++i) {
            fa::CopyArea& y = a.area[i];
            (void)area_of(areas[first + i], &y);   // (looked at above)
            const uint64_t most = static_cast<uint64_t>(y.n0) * y.n1 * y.row / 16384;
            y.parts = static_cast<uint32_t>(most < 1 ? 1 : most < share ? most : share);
            if (y.parts > 64) y.parts = 64;
            parts += y.parts;
        }
        const uint32_t most_x = (ctas + parts - 1) / parts, x = pairs < most_x ? pairs : most_x;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(x, parts, 1), cfg.blockDim = dim3(fa::kCopyThreads, 1, 1), cfg.stream = static_cast<cudaStream_t>(cuda_stream);
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr, cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, &fa::fa_cache_copy, a);
        rc = static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
        if (rc != FA_B200_OK) return rc;
    }
    return FA_B200_OK;
}

int fa_b200_describe_copy(const fa_b200_copy_area* area, uint32_t out[4]) {
    if (!area || !out) return FA_B200_ERR_NULL_POINTER;
    fa::CopyArea y = {};
    const int rc = area_of(*area, &y);
    if (rc != FA_B200_OK) return rc;
    out[0] = y.n0, out[1] = y.n1, out[2] = y.row, out[3] = y.unit;
    return FA_B200_OK;
}

}  // extern "C"
