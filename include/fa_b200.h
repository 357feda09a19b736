/*
 * fa_b200.h — C ABI of the B200 (sm_100a) fused multi-head attention forward.
 *
 * One operator:  Y = softmax(Q K^T / sqrt(H)) V  per (batch, head), fp16 in / fp16 out,
 * fp32 accumulation and fp32 online-softmax state, no L x L score matrix in global memory.
 *
 * Tensor contract (same as the reference operator, src/fused_attn_extention.cu:24-70):
 * q, k, v, y are contiguous fp16 device arrays of logical shape [B, L, F] with F = R * head_dim
 * (any B, R, L with ceil(L/128) * R * B below 2^31);
 * head h owns columns [h*head_dim, (h+1)*head_dim) of the last axis
 * (include/fused_attn.cuh:681-696 in the reference).  The optional mask is a contiguous fp16
 * array [B, L, L] that is ADDED to the scaled scores of every head (reference
 * include/fused_attn.cuh:686,735-742; the reference adds it to the first key chunk only, this
 * library adds it to every key tile).
 *
 * Every function is thread-safe.  None of them terminates the process: where the reference
 * launcher prints and calls exit() (include/fused_attn.cuh:17-42) these return a status code.
 */
#ifndef FA_B200_H_
#define FA_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes.  0 = success, negative = rejected before launch, positive = a cudaError_t. */
enum {
    FA_B200_OK = 0,
    FA_B200_ERR_NULL_POINTER = -1,   /* q, k, v or y is NULL                                   */
    FA_B200_ERR_HEAD_DIM = -2,       /* head_dim not in {16, 32, 64, 128}                      */
    FA_B200_ERR_CHUNK = -3,          /* chunk_hint violates the reference's rule set           */
    FA_B200_ERR_SHAPE = -4,          /* B, L or F is zero, F % head_dim != 0, or too large     */
    FA_B200_ERR_ALIGNMENT = -5,      /* a tensor base address is not 16-byte aligned           */
    FA_B200_ERR_ARCH = -6,           /* the device is not compute capability 10.x              */
    FA_B200_ERR_DRIVER = -7,         /* cuTensorMapEncodeTiled unavailable or failed           */
    FA_B200_ERR_FLAGS = -8,          /* contradictory or unknown flag bits                     */
    FA_B200_ERR_DEVICE_TIMEOUT = -9, /* a bounded device-side wait expired (see read_status)   */
    FA_B200_ERR_TOO_LARGE = -10,     /* a fixed-capacity entry point was given too much work, or
                                        a call less scratch than it needs                      */
    FA_B200_ERR_PAGE = -11,          /* page_size not in {16, 32, 64, 128}                     */
    FA_B200_ERR_DTYPE = -12          /* dtype is neither FA_B200_FP16 nor FA_B200_BF16         */
};

/* flags for fa_b200_attention_forward */
enum {
    FA_B200_FLAG_DEFAULT = 0u,
    FA_B200_FLAG_FORCE_SIMPLE = 1u,    /* always use the one-tile-per-CTA kernel                */
    FA_B200_FLAG_FORCE_PIPELINED = 2u, /* always use the warp-specialised kernel (H in {64,128}) */
    FA_B200_FLAG_SYNC = 4u,            /* synchronise the stream before returning and fold the
                                          device status word into the return value; a report is
                                          cleared when it is returned (see fa_b200_read_status) */
    FA_B200_FLAG_NO_OVERLAP = 8u,      /* plain launch.  By default the kernel is launched with the
                                          programmatic-stream-serialization attribute: its CTAs may
                                          become resident and set up their barriers and tensor memory
                                          while the previous kernel of the stream drains; they touch
                                          global memory only once that kernel has completed, so the
                                          stream's ordering guarantees are unchanged             */
    FA_B200_FLAG_FORCE_PAIR = 32u,     /* head_dim 128 (with a mask: one whose rows all start on 16-byte
                                          boundaries, else FA_B200_ERR_FLAGS): always use the kernel
                                          that runs on pairs
                                          of CTAs (one MMA of 256 rows for two SMs); implies whole work
                                          items.  By default it is taken for such calls when their last
                                          round is not divided, the sequence has an even or large
                                          number of 256-row blocks and (without a mask) the pairs of SMs
                                          get more than one work item each                           */
    FA_B200_FLAG_NO_PAIR = 64u,        /* never use that kernel                                      */
    FA_B200_FLAG_NO_SPLIT = 16u        /* never divide the key axis of one (batch, head, query rows)
                                          problem among several CTAs.  By default the warp-specialised
                                          kernel may do so to keep every SM busy when the work items
                                          leave most SMs idle in the last round; the partial results
                                          are merged in fp32, in a fixed order, so a call repeats bit
                                          for bit, but where the cuts fall depends on how many
                                          (batch, head) pairs the call holds, and a divided problem
                                          differs from the undivided one by the kernel's ordinary
                                          rounding error.  With this flag the bits of one
                                          (batch, head) do not depend on what else is in the call (a
                                          shard reproduces the undivided job exactly)                */
};

/*
 * Launch the fused attention forward on `cuda_stream` (a cudaStream_t, NULL = default stream)
 * of CUDA device `device`.  Asynchronous unless FA_B200_FLAG_SYNC is given.
 *
 * Replaces the reference's launcher template
 *   launch_attention_kernel<head_dim, chunk_size>(B, L, F, q, k, v, mask, out, sync)
 * (include/fused_attn.cuh:860-894) together with the 12-way dispatch switch of
 * src/fused_attn_extention.cu:72-111.
 *
 * `chunk_hint` is validated with the reference's rules (power of two in [16,128], <= 2*head_dim,
 * not (16 with head_dim 128); src/fused_attn_extention.cu:45-47) so that existing callers see
 * the same rejections, but the tile sizes are internal and L need NOT be a multiple of it.
 * Pass 0 to skip the check.
 */
int fa_b200_attention_forward(const void* q, const void* k, const void* v,
                              const void* mask_or_null, void* y,
                              uint32_t B, uint32_t L, uint32_t F,
                              uint32_t head_dim, uint32_t chunk_hint,
                              int device, void* cuda_stream, uint32_t flags);

/*
 * Same operator with HOST buffers: copies q, k, v (and mask) to the device, runs the kernel and
 * copies y back, and returns when y is complete.  The work is cut into up to 8 chunks (batch
 * entries, or blocks of query rows of one where there are few) that flow through three internal streams, so the copy-in of one
 * chunk, the kernel of the previous and the copy-out of the one before overlap; pinned host
 * buffers are needed for that overlap.  Device staging buffers are cached per device and grow on
 * demand.  This is the call a torch-free
 * host program makes; it plays the role of the reference's standalone driver
 * (src/test.cu:43-62: cudaMalloc, fill, launch, synchronise).
 */
int fa_b200_attention_forward_host(const void* q, const void* k, const void* v,
                                   const void* mask_or_null, void* y,
                                   uint32_t B, uint32_t L, uint32_t F,
                                   uint32_t head_dim, uint32_t chunk_hint,
                                   int device, uint32_t flags);

/*
 * The same operator for callers that must not allocate.  It has no counterpart in the reference
 * (whose binding always allocates its output and whose launcher has no workspace at all).
 *
 * Who needs it: code that runs where cudaMalloc is off limits or unwanted: a process whose device
 * memory is entirely owned by another allocator or already handed out (an inference server that
 * reserves the whole GPU at start-up), a plugin that may not grow its host's footprint, a
 * latency-critical loop where an allocation would synchronise the device.
 * fa_b200_attention_forward allocates (once per device) a small status buffer for its kernels;
 * this entry point never calls cudaMalloc, cudaFree or any allocating library routine.
 *
 * How: it always runs the one-tile-per-CTA kernel, and that kernel's only scratch (a pair of
 * status words per CTA, written when a bounded device-side wait expires) lives in a fixed array
 * inside the library's device image: 16384 pairs = 128 KiB, held by every GPU that loads the
 * library until the process exits.  Consequences:
 *   - ceil(L/128) * (F/head_dim) * B must not exceed 16384 CTAs, otherwise the call is rejected
 *     with FA_B200_ERR_TOO_LARGE before anything is launched;
 *   - all calls on a device share that array.  Each call zeroes the pairs it is going to use (in
 *     stream order, ahead of its kernel) and the array otherwise keeps what the last call left;
 *     two calls whose kernels overlap on the GPU (different streams) race on it, so serialise them;
 *   - the first call on a device looks up the array's device address and sets the kernel's
 *     shared-memory attribute, two calls into the CUDA runtime that later calls do not make.
 *     Calls on different devices do not wait for one another.
 * flags: 0 or FA_B200_FLAG_SYNC (synchronise the stream and return FA_B200_ERR_DEVICE_TIMEOUT if
 * any CTA reported).  Inputs, outputs, head_dim, chunk_hint, mask: as fa_b200_attention_forward.
 */
int fa_b200_attention_forward_noalloc(const void* q, const void* k, const void* v,
                                      const void* mask_or_null, void* y,
                                      uint32_t B, uint32_t L, uint32_t F,
                                      uint32_t head_dim, uint32_t chunk_hint,
                                      int device, void* cuda_stream, uint32_t flags);

/*
 * Human-readable text for a status code returned by this library (negative codes) or by the
 * CUDA runtime (positive codes).  Replaces the stderr printing of the reference's
 * checkCudaError / checkLastCudaError (include/fused_attn.cuh:17-42).
 */
const char* fa_b200_strerror(int code);

/*
 * Device facts used by harnesses: out[0] = compute capability major, out[1] = minor,
 * out[2] = SM count, out[3] = max opt-in shared memory per block (bytes).
 * No counterpart in the reference (its CMake probes the device instead, CMakeLists.txt:12-39).
 */
int fa_b200_query(int device, int32_t out[4]);

/*
 * Read and clear the per-device status word written by kernels whose bounded waits expired:
 * out[0] = first failure code (0 = none; bits 8.. = role, bits 0..7 = barrier id),
 * out[1] = number of CTAs that reported.  Synchronises the device.
 * The word is shared by every launch on the device and stays set until it is read here, or
 * returned by a call with FA_B200_FLAG_SYNC or by fa_b200_attention_forward_host (both clear it
 * when they return FA_B200_ERR_DEVICE_TIMEOUT).  An asynchronous call never looks at it: after a
 * launch whose wait expired its output is garbage and only this word says so.  A CTA reports as it
 * ends; the CTAs of its launch that start after that leave at once.
 * No counterpart in the reference (it has no device-side error reporting).
 */
int fa_b200_read_status(int device, uint32_t out[2]);

/*
 * Exercise the bounded-wait path without touching the attention kernels: a one-warp kernel waits
 * (for about 10 ms) on a barrier that nothing completes, must give up, report and return.
 * out[0] = status code it recorded (expected 0x67F), out[1] = CTAs that reported (expected 1),
 * out[2] = 2 if the wait returned "gave up", 1 if it claimed success.  The GPU stays usable.
 * No counterpart in the reference (its kernels wait only on __syncthreads).
 */
int fa_b200_selftest_bounded_wait(int device, uint32_t out[3]);

/*
 * The checked build of the library (compiled with -DFA_DEBUG: every TMA copy and tensor-memory access
 * checks its shared-memory operand, its coordinates and its columns first, reports a failed check in
 * the device status word at the CTA's end and skips the access; tile buffers and Y are filled with NaN beforehand) can
 * test its own predicates: they are asked about operands that are in order and operands that are not,
 * with no copy made.  out[0] = status code recorded by the first refusal (expected 0x703: innermost
 * coordinate not a multiple of 8 elements), out[1] = 1, out[2] = 1 in a checked build and 0 in a normal
 * one (where nothing else is done), out[3] = one bit per predicate answered as it should be (expected
 * 0x7FF).  It plays the role of the reference's -g -G build of its smoke test (CMakeLists.txt:43) on
 * a pool where compute-sanitizer cannot be run.
 */
int fa_b200_selftest_debug_checks(int device, uint32_t out[4]);

#ifdef FA_CYCLES
/*
 * Only in the clock-counting build of the library (compiled with -DFA_CYCLES): from now on CTA 0 of the
 * warp-specialised kernels writes, per launch, four 64-bit words into record (launch id mod 64) of the
 * given device buffer of 256 words: the global timer (ns) at its entry, after its wait for the previous
 * kernel of the stream and at its end, and its SM clock count between the last two.  NULL stops the
 * recording.  The buffer must outlive the launches.  A build with -DFA_TIMELINE as well needs a buffer of
 * 9 * 1024 words: behind the 256, lane 0 of one warp per role of CTA 0 of the kernel on pairs of CTAs writes
 * its SM clock at up to eight events of each of the first 256 key steps (word 256 + (role * 256 + step) * 8 +
 * event; the roles and events are listed in csrc/fa_kernels.cuh and csrc/fa_pair.cuh).  No counterpart in the
 * reference.
 */
int fa_b200_debug_cycles(void* device_buffer_of_256_u64);
#endif

/*
 * What a call launches on a device with `sm_count` SMs.  `mask_alignment`: 0 without a mask, else what the
 * mask's address is a multiple of, in bytes (2, 4, 8 or 16).
 * out[0] = the kernel: 0 the one for short sequences, 1 the one with a query tile per CTA, 2 the
 *          warp-specialised one, 3 the warp-specialised one on pairs of CTAs,
 * out[1] = 1 if the call is planned on a stream that has scratch (fa_b200_stream_has_scratch): a kernel
 *          finds out first what the mask leaves to do, and the warp-specialised kernel follows its lists;
 *          for a mask whose rows all start on 16-byte boundaries the kernel of out[0] is launched behind
 *          the two and does the call where the mask leaves too little out (fa_b200_plan_taken).  Without
 *          scratch it is launched alone,
 * out[2] = how many kernels that are (1, 2 or 3).
 * Pure arithmetic, no CUDA call; it is what the launcher itself uses.  No counterpart in the reference.
 */
int fa_b200_describe_call(uint32_t B, uint32_t L, uint32_t F, uint32_t head_dim,
                          uint32_t mask_alignment, uint32_t flags, uint32_t sm_count, uint32_t out[3]);

/*
 * out[0] = 1 if a call on `cuda_stream` would find scratch for a divided or a planned call, 0 if not: four
 * streams of a device get some, the first four that ask, and keep it; a stream that is being captured
 * gets none.  Takes none itself.  No counterpart in the reference.
 */
int fa_b200_stream_has_scratch(int device, void* cuda_stream, uint32_t out[1]);

/*
 * A planned call whose mask's rows all start on 16-byte boundaries is given to the kernel behind the
 * planned one where too little of the mask is -inf.  That is judged first by the beginnings of at most 256
 * of its 128 x 128 tiles: out[0] = batch entry, out[1] = query tile, out[2] = key tile of the one with the
 * given index, out[3] = how many are looked at.  FA_B200_ERR_SHAPE for an index beyond them, or sizes that
 * are not planned.  Pure arithmetic, no CUDA call; it is what the kernel itself uses.  No counterpart in the
 * reference.
 */
int fa_b200_describe_plan_sample(uint32_t B, uint32_t L, uint32_t index, uint32_t out[4]);

/*
 * Leaving a key tile out is only right while its K and V are finite.  Where the rows of a planned call's
 * mask all start on 16-byte boundaries, a key tile that some pairs of query tiles leave out and others work
 * on is looked through by one of the latter: out[0] = which, 0xFFFF if no pair works on it or none leaves it
 * out.  `works`: for each of the `tiles` query tiles of a batch entry 0 if the mask is -inf throughout for it
 * and the key tile, anything else if not.  Pure arithmetic, no CUDA call; it is what the kernel itself uses.
 * No counterpart in the reference.
 */
int fa_b200_describe_plan_check(uint32_t tiles, const uint8_t* works, uint32_t key_tile, uint32_t out[1]);

/*
 * Which kernel had the last planned call on `cuda_stream`: out[0] = 1 if that is known (the stream's scratch
 * still holds the plan: no call with a divided last round came behind it), out[1] = 1 if it was the planned
 * kernel, 0 if the one behind it.  Synchronises the stream.  A diagnostic, for tests and harnesses: what the
 * mask holds is only known on the device, so fa_b200_describe_call cannot tell.  No counterpart in the
 * reference.
 */
int fa_b200_plan_taken(int device, void* cuda_stream, uint32_t out[2]);

/*
 * The family a call belongs to, as harnesses ask for it: 1 for the kernel with a query tile per CTA, for
 * every sequence that the kernel for short sequences takes, and for every call at head_dim 16 and 32
 * (whichever kernel serves those: FA_B200_FLAG_FORCE_PIPELINED is refused there), 2 for the
 * warp-specialised kernel, 3 for the warp-specialised kernel on pairs of CTAs (head_dim 128, whole work
 * items; a mask is taken to start on a 16-byte boundary, its rows then do so whenever L is a multiple of
 * 8, and not to be planned), negative status on invalid arguments.  fa_b200_describe_call says what a
 * call launches.  No counterpart in the reference.
 */
int fa_b200_select_kernel(uint32_t B, uint32_t L, uint32_t F, uint32_t head_dim,
                          int has_mask, uint32_t flags);

/*
 * How the warp-specialised kernel would spread a call's work over its CTAs on a device with
 * `sm_count` SMs, without a mask (head_dim 64 and 128; smaller ones are described as one CTA per query
 * tile, whichever kernel serves them, see fa_b200_select_kernel):
 * out[0] = kernel (1, 2 or 3, as fa_b200_select_kernel; for 3 a work item is 512 query
 * rows and out[1] CTAs form out[1]/2 pairs, nothing is divided), out[1] = CTAs launched,
 * out[2] = rounds of whole work items (a work item is 256 query rows of one (batch, head) against
 * all keys; CTA c takes items c, c + out[1], ...), out[3] = work items of the last, partial round
 * whose key steps are divided evenly among the first out[6] CTAs (0 = nothing is divided; a range
 * is at least half a work item, or exactly a third of each with out[6] = 3 * out[3]: a work item has
 * at most three parts), out[4] = key steps of
 * those items in all, out[5] = key steps (tiles of 128 keys) per work item.  Pure arithmetic, no
 * CUDA call; it is what the launcher itself uses (FA_B200_FLAG_NO_SPLIT in `flags` is honoured).
 * No counterpart in the reference, whose grid is one CTA per (batch, query chunk, head)
 * (include/fused_attn.cuh:883).
 */
int fa_b200_describe_schedule(uint32_t B, uint32_t L, uint32_t F, uint32_t head_dim,
                              uint32_t flags, uint32_t sm_count, uint32_t out[7]);

/*
 * ---- The paged 8-bit key/value cache: fa_b200_cache_append, fa_b200_cache_select, fa_b200_cache_attention.
 *
 * The keys and values of sequences, in pages of page_size tokens.  A page has for each of kv_heads heads e4m3 codes and one
 * fp32 scale for its keys and one for its values (a value is code * scale), and the bounds of its keys, the lowest and the
 * highest code by dimension.  The i-th block of page_size tokens of sequence b lies in page table[b][i].  The scales that
 * fa_b200_cache_append writes are powers of two from 2^-100 to 2^120; attention and selection take any others in this range, however
 * far apart (attention takes a value scale below 2^-100 for 2^-100).  A scale below zero counts as one that is not a number.
 *
 * What these functions are given is checked before anything is launched, as far as the host can see it.  What lies in device
 * memory (table, lengths, counts, selected pages) the kernels look at before they use it: tokens whose page is outside the
 * cache are left out, tokens behind the table or the rotation's last position are not appended, a length that the table has no
 * room for is cut, and the cache's status block receives the first such code and the number of reports: 1 a page outside the
 * cache or the table, 2 a position or length outside, 0x100 and above a bounded wait that expired.
 *
 * All three are asynchronous on `cuda_stream`, and repeat bit for bit.  None allocates: scratch comes from the caller, need not
 * be initialised, and may be used again by the next work on the same stream.
 */
enum { FA_B200_FP16 = 0u, FA_B200_BF16 = 1u };   /* dtype of 16-bit tensors */
enum {
    FA_B200_CACHE_NEIGHBOURS = 1u,   /* fa_b200_cache_append: the rotation's pairs are dimensions (2i, 2i + 1), not (i, i + H/2)   */
    FA_B200_CACHE_ALL_KEYS = 2u      /* fa_b200_cache_attention: every query sees every key of its sequence                       */
};

typedef struct fa_b200_cache {
    void* k;             /* e4m3 codes: page p, head h, token t at p * k_page_stride + h * k_head_stride + t * k_token_stride,   */
    void* v;             /* head_dim of them in a row.  Strides in bytes, multiples of 16; k, v and bounds on 16-byte boundaries */
    float* k_scale;      /* [n_pages, kv_heads] */
    float* v_scale;
    void* bounds;        /* [n_pages, kv_heads, 2, head_dim]: lowest and highest key code */
    uint32_t* status;    /* two words, zero until something is wrong */
    int64_t k_page_stride, k_head_stride, k_token_stride;
    int64_t v_page_stride, v_head_stride, v_token_stride;
    uint32_t n_pages, kv_heads, page_size, head_dim;
} fa_b200_cache;

typedef struct fa_b200_sequences {
    const int32_t* table;     /* [B, table_width], rows table_stride elements apart; entries that no token reaches may be anything */
    const int32_t* lengths;   /* [B]: tokens that the cache holds when the call begins */
    const int32_t* counts;    /* [B]: how many of the call's T tokens a sequence has, or NULL: all of them */
    int64_t table_stride;
    uint32_t table_width, B, T;
} fa_b200_sequences;

/*
 * Append T tokens to each sequence, at positions lengths[b], lengths[b] + 1, ...: keys and values [B, T, kv_heads * head_dim]
 * of 16-bit values with the last axis contiguous (strides in elements; rows on 16-byte boundaries).  With cos and sin (fp32
 * [positions, head_dim / 2]) keys are rotated by their position, x1 c - x2 s and x2 c + x1 s, and so are the queries, which are
 * written to `rotated` ([B, T, q_heads * head_dim] contiguous, rounded once; zeros where a sequence has no token; without cos
 * and sin they are copied).  Lengths are not changed.
 *
 * A page's scale is the smallest power of two, 2^-100 at least, with which the largest magnitude of its tokens is 448 or less;
 * a page that held tokens keeps a larger one, and where its scale grows its old codes are moved to the new one (exact but for
 * subnormal codes).  Codes are rounded to nearest even.  A value that is not finite makes the scale of its page and head NaN and
 * the codes zero.  Sequences of one call must not append to the same page.  Where tokens are taken back by lowering a length, their
 * page keeps the scale (a NaN too), the rounding of older tokens to it and the bounds until its first token is appended anew.
 */
int fa_b200_cache_append(const fa_b200_cache* cache, const fa_b200_sequences* sequences, const void* keys, int64_t keys_batch_stride,
                         int64_t keys_token_stride, const void* values, int64_t values_batch_stride, int64_t values_token_stride,
                         const void* queries_or_null, int64_t queries_batch_stride, int64_t queries_token_stride, uint32_t q_heads,
                         void* rotated, const float* cos_or_null, const float* sin_or_null, uint32_t positions, uint32_t dtype,
                         uint32_t flags, int device, void* cuda_stream);

/*
 * For each query and key/value head the `keep` pages with the highest scores among those up to the query's own, ascending, into
 * pages [B, T, kv_heads, keep] (block indices of the sequence, not page numbers; -1 behind the last).  Query t of a sequence
 * stands at position lengths[b] - counts[b] + t.  Score of a page: with q8 = rint(q * (1 / max |q| * 127)) of a query head and
 * lo8, hi8 = rint(bound / 4), sum over the dimensions of max(q8 lo8, q8 hi8), a whole number; times max |q| * (1 / 127); the largest
 * of the query heads of the key/value head; times the page's key scale (each product and quotient rounded to fp32).  Ties go to the lower page.  The first `first` blocks
 * and the last `last` up to the query's own (at least one) are taken before all others, behind them pages whose score is not a number.  Scratch: 4 * B * T * kv_heads *
 * table_width bytes.
 */
int fa_b200_cache_select(const fa_b200_cache* cache, const fa_b200_sequences* sequences, const void* queries, int64_t queries_batch_stride,
                         int64_t queries_token_stride, uint32_t q_heads, uint32_t dtype, uint32_t keep, uint32_t first, uint32_t last,
                         int32_t* pages, void* scratch, uint64_t scratch_bytes, int device, void* cuda_stream);

/*
 * y = softmax(q K^T / sqrt(head_dim)) V over the cache: queries [B, T, q_heads * head_dim] (q_heads a multiple of kv_heads:
 * query head h has key/value head h / (q_heads / kv_heads)), the last ones of their sequences: query t stands at position
 * lengths[b] - counts[b] + t and sees the keys up to its own, or all with FA_B200_CACHE_ALL_KEYS.  With `pages`
 * ([B, T, kv_heads, keep], as fa_b200_cache_select writes them, -1 for nothing) only those blocks.  y is contiguous, of the
 * queries' type; a query that sees no key, or that its sequence does not have, gets zeros.  Scores, weights and sums are held in
 * fp32; the weights are rounded to fp16 for the product with V.  In fp16 calls with `pages`, or with fewer than 64 rows (T * q_heads /
 * kv_heads), what that rounding takes away is multiplied as well, so that an error is little more than the rounding of y.
 * Among scores (times log2 e) of 2^22 and more, keys that tie on pages of different value scales are not weighed exactly.  Scratch: as fa_b200_cache_attention_scratch says, on a 16-byte
 * boundary.
 */
int fa_b200_cache_attention(const fa_b200_cache* cache, const fa_b200_sequences* sequences, const void* queries, int64_t queries_batch_stride,
                            int64_t queries_token_stride, uint32_t q_heads, uint32_t dtype, const int32_t* pages_or_null, uint32_t keep,
                            uint32_t flags, void* y, void* scratch, uint64_t scratch_bytes, int device, void* cuda_stream);

/* out[0] = bytes of scratch that such a call needs (keep = 0 without a list of pages).  Pure arithmetic on the device's facts. */
int fa_b200_cache_attention_scratch(uint32_t head_dim, uint32_t kv_heads, uint32_t q_heads, uint32_t page_size, uint32_t B, uint32_t T,
                                    uint32_t table_width, uint32_t keep, int device, uint64_t out[1]);

/*
 * ---- The pages of a cache: fa_b200_pages_fork, fa_b200_pages_reserve, fa_b200_pages_compact, fa_b200_cache_copy.
 *
 * refs[p] is how many entries of the table [B, table_width] hold page p; 0: it is free.  An entry is a page or -1, a row holds a page
 * once.  The functions keep refs and table in step; calls on one refs and table have to be ordered by streams.  All are asynchronous,
 * repeat bit for bit and allocate nothing.  `status` receives the first code and the number of reports: 1 an entry that is neither a page
 * nor -1 (taken for -1), 2 a length, count or parent outside, 3 no page was free, 4 refs and table are not in step.
 */
typedef struct fa_b200_pages {
    int32_t* refs;       /* [n_pages] */
    uint32_t* status;    /* four words, of which the first two are written; pools may share them */
    uint32_t n_pages;
} fa_b200_pages;

/*
 * Row b of the table becomes what row parents[b] was, and lengths[b] what its length was, all at once and in place; -1: an empty row
 * (its pages are let go of) and length 0.  A parent outside leaves a row as it is.  At most 57344 sequences.
 */
int fa_b200_pages_fork(const fa_b200_pages* pages, int32_t* table, int64_t table_stride, uint32_t table_width, uint32_t B, int32_t* lengths,
                       const int32_t* parents, int device, void* cuda_stream);

/*
 * Gives every sequence the blocks that lengths[b] + counts[b] tokens need (counts NULL: `count` each) and no more: blocks behind them are
 * let go of.  Blocks that the new tokens go to and that have no page get one, and so do those whose page others hold too, unless all that
 * hold it are about to write to it: then the sequence with the most tokens on it keeps it, the lowest of several.  New pages are the lowest
 * free ones, in the order of sequences and blocks; a block that finds none stays as it was, and nothing is written to it.  sources[b], targets[b]: the page that held the beginning of a block, and the one that has taken its place (-1: none);
 * fa_b200_cache_copy is to copy it before tokens are appended.  granted[b]: how many of the tokens have room, counts[b] unless pages ran out.
 * Scratch: 4 * n_pages bytes.
 */
int fa_b200_pages_reserve(const fa_b200_pages* pages, int32_t* table, int64_t table_stride, uint32_t table_width, uint32_t B, const int32_t* lengths,
                          const int32_t* counts_or_null, uint32_t count, uint32_t page_size, int32_t* granted, int32_t* sources, int32_t* targets,
                          void* scratch, uint64_t scratch_bytes, int device, void* cuda_stream);

/*
 * The move of all pages that are held to the front: with n_used of them, the k-th of those from n_used on goes to the k-th free one in front
 * of it.  Writes refs and table ([B, table_width] contiguous) as they are afterwards, and the moves: sources and targets [n_pages], -1 behind
 * the last.  The old ones are left as they are.  Beyond 100000 pages time grows with their square.  Scratch: 4 * n_pages + 8 bytes.
 */
int fa_b200_pages_compact(const fa_b200_pages* pages, const int32_t* table, int64_t table_stride, uint32_t table_width, uint32_t B, int32_t* new_refs,
                          int32_t* new_table, int32_t* sources, int32_t* targets, void* scratch, uint64_t scratch_bytes, int device, void* cuda_stream);

/* An array of pages: page p is n0 x n1 rows of row_bytes, row (i, j) at base + p * page_stride + i * stride0 + j * stride1 (bytes; all of
 * them multiples of 16 if row_bytes is, else of 4). */
typedef struct fa_b200_copy_area {
    void* base;
    int64_t page_stride, stride0, stride1;
    uint32_t n0, n1, row_bytes;
} fa_b200_copy_area;

/*
 * Copies page sources[i] to page targets[i] in each of the arrays, all of n_pages pages; pairs with -1 are passed over.  No page may be
 * a target twice, or a target and a source.  `areas` is read before the call returns.  status: two words, 1 a page outside.
 */
int fa_b200_cache_copy(const fa_b200_copy_area* areas, uint32_t n_areas, uint32_t n_pages, const int32_t* sources, const int32_t* targets, uint32_t pairs,
                       uint32_t* status, int device, void* cuda_stream);

/* How an array is copied: out[0], out[1], out[2] = its rows n0 x n1 and their bytes once rows that lie behind one another are one, out[3] = bytes
 * that a thread takes at a time, 16 or 4.  Pure arithmetic, no CUDA call; it is what fa_b200_cache_copy itself uses. */
int fa_b200_describe_copy(const fa_b200_copy_area* area, uint32_t out[4]);

/*
 * ---- The paged cache of latent vectors: fa_b200_latent_append, fa_b200_latent_attention, and fa_b200_latent_prompt.
 *
 * A token has one row for all heads: latent_dim 16-bit values (128, 256 or 512) that are key and value at once, and behind them rope_dim
 * (16, 32 or 64) that belong to the key and are rotated by the token's position.  Sequences, tables and what the status block receives are as
 * with the 8-bit cache above.  All functions are asynchronous, repeat bit for bit and allocate nothing.
 */
typedef struct fa_b200_latent_cache {
    void* data;          /* row t of page p at p * page_stride + t * token_stride (bytes, multiples of 16), on a 16-byte boundary */
    uint32_t* status;    /* two words, zero until something is wrong */
    int64_t page_stride, token_stride;
    uint32_t n_pages, page_size, latent_dim, rope_dim;
} fa_b200_latent_cache;

/*
 * Append T tokens to each sequence, at positions lengths[b], ...: latents [B, T, latent_dim] as they are, rope_keys [B, T, rope_dim] rotated
 * (strides in elements, last axis contiguous, rows on 16-byte boundaries).  Rotated keys [B, T, rope_dim] and, with queries
 * ([B, T, heads, rope_dim]), rotated queries are written out too, contiguous, rounded once; zeros where a sequence has no token or the
 * rotation no position.  cos and sin: fp32 [positions, rope_dim / 2]; without them nothing is rotated.  Lengths are not changed.
 */
int fa_b200_latent_append(const fa_b200_latent_cache* cache, const fa_b200_sequences* sequences, const void* latents, int64_t latents_batch_stride,
                          int64_t latents_token_stride, const void* rope_keys, int64_t keys_batch_stride, int64_t keys_token_stride, const void* queries_or_null,
                          int64_t queries_batch_stride, int64_t queries_token_stride, int64_t queries_head_stride, uint32_t heads, void* rotated_keys,
                          void* rotated_queries, const float* cos_or_null, const float* sin_or_null, uint32_t positions, uint32_t dtype, uint32_t flags, int device,
                          void* cuda_stream);

/*
 * y = sum of softmax(scale * (q_latent . c + q_rope . r)) c over the rows (c, r) that a query sees, for queries that have been multiplied into
 * the latent space: q_latent [B, T, heads, latent_dim], q_rope [B, T, heads, rope_dim] (rotated), y [B, T, heads, latent_dim] contiguous.  Queries
 * are the last tokens of their sequences, as with fa_b200_cache_attention, FA_B200_CACHE_ALL_KEYS too.  Cache and queries have one type.
 * Scores, sums and maxima are held in fp32, weights are rounded to the type for their product with c and summed as rounded.  A query that sees
 * nothing, or that its sequence does not have, gets zeros.  Rows that a query does not see do not reach it, whatever they hold.  scale: 2^-126 to 10^38.
 */
int fa_b200_latent_attention(const fa_b200_latent_cache* cache, const fa_b200_sequences* sequences, const void* q_latent, int64_t ql_batch_stride,
                             int64_t ql_token_stride, int64_t ql_head_stride, const void* q_rope, int64_t qr_batch_stride, int64_t qr_token_stride,
                             int64_t qr_head_stride, uint32_t heads, float scale, uint32_t dtype, uint32_t flags, void* y, void* scratch, uint64_t scratch_bytes,
                             int device, void* cuda_stream);

/* out[0] = bytes of scratch that such a call needs, on a 16-byte boundary.  Pure arithmetic on the device's facts. */
int fa_b200_latent_attention_scratch(uint32_t latent_dim, uint32_t heads, uint32_t page_size, uint32_t B, uint32_t T, uint32_t table_width, int device, uint64_t out[1]);

/*
 * The same attention with keys and values multiplied out of the latent vectors, for prompts: queries [B, T, heads, nope_dim] and
 * [B, T, heads, rope_dim] (rotated), expanded [B, S, heads, 2 * nope_dim], of each head its own part of the keys and behind it the values,
 * rope_keys [B, S, rope_dim] (rotated), the same for all heads; y [B, T, heads, nope_dim] contiguous.  nope_dim 64 or 128, rope_dim 16, 32 or 64.
 * y = softmax(scale * (q_nope . k + q_rope . r)) v, the queries the last counts[b] (NULL: T) of the lengths[b] (NULL: S) tokens of their
 * sequences; FA_B200_CACHE_ALL_KEYS as above.  Strides in elements, positive where an axis has more than one entry.  Scores, sums and maxima are
 * held in fp32, weights are rounded to the type for their product with v.  Keys that a query does not see do not reach it, whatever they hold.
 */
int fa_b200_latent_prompt(const void* q_nope, int64_t qn_batch_stride, int64_t qn_token_stride, int64_t qn_head_stride, const void* q_rope, int64_t qr_batch_stride,
                          int64_t qr_token_stride, int64_t qr_head_stride, const void* expanded, int64_t kv_batch_stride, int64_t kv_token_stride,
                          int64_t kv_head_stride, const void* rope_keys, int64_t rk_batch_stride, int64_t rk_token_stride, const int32_t* lengths_or_null,
                          const int32_t* counts_or_null, uint32_t B, uint32_t T, uint32_t S, uint32_t heads, uint32_t nope_dim, uint32_t rope_dim, float scale,
                          uint32_t dtype, uint32_t flags, void* y, int device, void* cuda_stream);

/* out[0], out[1] = first code and number of reports of fa_b200_latent_prompt's launches on the device (2: a length or count outside, cut;
 * 0x100 and above: a bounded wait expired); cleared when read.  Synchronises the device. */
int fa_b200_latent_status(int device, uint32_t out[2]);

#ifdef __cplusplus
}
#endif
#endif /* FA_B200_H_ */
