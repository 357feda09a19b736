// Torch extension module `fused_attn`: the operator surface of the reference binding
// (src/fused_attn_extention.cu:15-129) over the C ABI of include/fa_b200.h.
//
//   fused_attn.attention_forward(head_dim, chunk_size, queries, keys, values, mask=None) -> Tensor
//
// Same argument names, order and default; the same preconditions raise the same exception type
// (c10::Error -> RuntimeError).  Relaxed on purpose: sequence_len need not be a multiple of
// chunk_size.  Fixed on purpose: the output lives on queries.device() and the launch goes to the
// caller's current stream (the reference allocates on the current device and launches on stream 0,
// src/fused_attn_extention.cu:67-70, include/fused_attn.cuh:885).
#include <torch/extension.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "fa_b200.h"

namespace {

void check_input(const torch::Tensor& t, const char* name) {
    TORCH_CHECK(t.dtype() == torch::kFloat16 && t.device().type() == torch::kCUDA && t.is_contiguous() &&
                    t.dim() == 3,
                name, " must be a contiguous float16 CUDA tensor with 3 dimensions");
}

torch::Tensor attention_forward(int head_dim, int chunk_size, torch::Tensor queries, torch::Tensor keys,
                                torch::Tensor values, torch::optional<torch::Tensor> mask) {
    check_input(queries, "queries");
    check_input(keys, "keys");
    check_input(values, "values");
    if (mask.has_value()) check_input(*mask, "mask");

    TORCH_CHECK(head_dim > 0 && !(head_dim & (head_dim - 1)) && 16 <= head_dim && head_dim <= 128,
                "head_dim must be a power of two in [16, 128]");
    TORCH_CHECK(chunk_size > 0 && !(chunk_size & (chunk_size - 1)) && 16 <= chunk_size && chunk_size <= 128 &&
                    chunk_size <= 2 * head_dim,
                "chunk_size must be a power of two in [16, 128] and at most 2*head_dim");
    TORCH_CHECK(!(chunk_size == 16 && head_dim == 128), "chunk_size 16 with head_dim 128 is not supported");

    const int64_t B = queries.size(0), L = queries.size(1), F = queries.size(2);
    TORCH_CHECK(keys.size(0) == B && keys.size(1) == L && keys.size(2) == F, "keys must have the shape of queries");
    TORCH_CHECK(values.size(0) == B && values.size(1) == L && values.size(2) == F,
                "values must have the shape of queries");
    TORCH_CHECK(F % head_dim == 0, "the feature size must be divisible by head_dim");
    TORCH_CHECK(B > 0 && L > 0 && F > 0, "empty tensors are not supported");
    TORCH_CHECK(keys.device() == queries.device() && values.device() == queries.device(),
                "queries, keys and values must be on one device");
    if (mask.has_value()) {
        TORCH_CHECK(mask->size(0) == B && mask->size(1) == L && mask->size(2) == L, "mask must have shape [B, L, L]");
        TORCH_CHECK(mask->device() == queries.device(), "mask must be on the device of queries");
    }

    const c10::cuda::CUDAGuard guard(queries.device());
    auto output = torch::empty_like(queries);
    const auto stream = c10::cuda::getCurrentCUDAStream(queries.device().index());
    const int rc = fa_b200_attention_forward(
        queries.data_ptr(), keys.data_ptr(), values.data_ptr(), mask.has_value() ? mask->data_ptr() : nullptr,
        output.data_ptr(), static_cast<uint32_t>(B), static_cast<uint32_t>(L), static_cast<uint32_t>(F),
        static_cast<uint32_t>(head_dim), static_cast<uint32_t>(chunk_size), queries.device().index(),
        static_cast<void*>(stream.stream()), FA_B200_FLAG_DEFAULT);
    TORCH_CHECK(rc == FA_B200_OK, "fa_b200: ", fa_b200_strerror(rc), " (status ", rc, ")");
    return output;
}

// The call behind the package's Python function (fused_attention_b200.attention_forward), positional arguments (entry,
// head_dim, chunk_size, queries, keys, values, mask or None, flags): the output, the status of a launch that failed, or None
// for everything that is not a plain call with every precondition met, which Python then looks at with its own checks (and
// their messages).  `entry` is the address of fa_b200_attention_forward in the library that Python has loaded, which need not
// be the one that this module links (the checked and the clock-counting build).  Checks, allocation and call took 8.4 us in
// Python on B=1 R=4 L=256 H=64, more than the kernel.
bool plain_tensor(PyObject* o, at::Tensor& t) {
    if (!THPVariable_CheckExact(o)) return false;   // a subclass may have its own idea of every operation
    t = THPVariable_Unpack(o);
    using c10::DispatchKey;
    static const c10::DispatchKeySet wrapped({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                              DispatchKey::Functionalize, DispatchKey::Conjugate, DispatchKey::Negative});
    return t.defined() && !t.key_set().has_any(wrapped) && t.scalar_type() == at::kHalf && t.is_cuda() && t.dim() == 3 && t.is_contiguous();
}

PyObject* forward_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8 || !PyLong_CheckExact(args[0])) Py_RETURN_NONE;
    auto* const entry = reinterpret_cast<decltype(&fa_b200_attention_forward)>(PyLong_AsVoidPtr(args[0]));
    if (entry == nullptr) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    ++args;
    if (!PyLong_CheckExact(args[0]) || !PyLong_CheckExact(args[1]) || !PyLong_CheckExact(args[6]) ||
        at::impl::PythonTorchFunctionTLS::stack_len() > 0)
        Py_RETURN_NONE;
    int over = 0;
    const long H = PyLong_AsLongAndOverflow(args[0], &over), C = over ? 0 : PyLong_AsLongAndOverflow(args[1], &over);
    const long flags = over ? 0 : PyLong_AsLongAndOverflow(args[6], &over);
    auto is_pow2 = [](long x) { return x > 0 && (x & (x - 1)) == 0; };
    if (over || flags < 0 || flags > 0xFFFFFFFFL || !is_pow2(H) || !is_pow2(C) || H < 16 || H > 128 || C < 16 || C > 128 || C > 2 * H ||
        (C == 16 && H == 128))
        Py_RETURN_NONE;
    at::Tensor q, k, v, mask;
    const bool masked = args[5] != Py_None;
    if (!plain_tensor(args[2], q) || !plain_tensor(args[3], k) || !plain_tensor(args[4], v) || (masked && !plain_tensor(args[5], mask)))
        Py_RETURN_NONE;
    const int64_t B = q.size(0), L = q.size(1), F = q.size(2);
    if (k.sizes() != q.sizes() || v.sizes() != q.sizes() || B <= 0 || L <= 0 || F <= 0 || F % H != 0 || B > UINT32_MAX || L > UINT32_MAX ||
        F > UINT32_MAX || k.device() != q.device() || v.device() != q.device() ||
        (masked && (mask.size(0) != B || mask.size(1) != L || mask.size(2) != L || mask.device() != q.device())))
        Py_RETURN_NONE;
    const auto device = q.device().index();
    at::Tensor out = at::empty_like(q);
    const void *pq = q.data_ptr(), *pk = k.data_ptr(), *pv = v.data_ptr(), *pm = masked ? mask.data_ptr() : nullptr;
    void *py = out.data_ptr(), *stream = static_cast<void*>(c10::cuda::getCurrentCUDAStream(device).stream());
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS   // (a call that waits for the stream must not hold other threads up)
    rc = entry(pq, pk, pv, pm, py, static_cast<uint32_t>(B), static_cast<uint32_t>(L), static_cast<uint32_t>(F),
               static_cast<uint32_t>(H), static_cast<uint32_t>(C), device, stream, static_cast<uint32_t>(flags));
    Py_END_ALLOW_THREADS
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}
PyMethodDef forward_through_def = {"_forward_through", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward_through)),
                                   METH_FASTCALL, nullptr};

// ---- The calls of the key/value cache behind the package's Python functions, in the same manner: None for everything that is
// not a plain call with every precondition met.  `cache` is the address of the cache's fa_b200_cache, which was looked at when the
// handle was made.  (In Python the checks, the structure and some thirty converted arguments take 17 to 25 us a call.)
bool plain_cuda(PyObject* o, at::Tensor& t, int device, int64_t dims) {
    if (!THPVariable_CheckExact(o)) return false;
    t = THPVariable_Unpack(o);
    using c10::DispatchKey;
    static const c10::DispatchKeySet wrapped({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                              DispatchKey::Functionalize, DispatchKey::Conjugate, DispatchKey::Negative});
    return t.defined() && !t.key_set().has_any(wrapped) && t.is_cuda() && t.get_device() == device && t.dim() == dims;
}
// [B, T, F] of 16-bit values with rows on 16-byte boundaries
bool plain_rows(PyObject* o, at::Tensor& t, int device, int64_t width) {
    return plain_cuda(o, t, device, 3) && (t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16) && t.numel() > 0 && t.size(2) % width == 0 &&
           t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0 && t.size(0) <= UINT32_MAX &&
           t.size(1) <= UINT32_MAX && t.size(2) <= UINT32_MAX;
}
bool plain_ints(PyObject* o, at::Tensor& t, int device, int64_t dims, int64_t B) {
    return plain_cuda(o, t, device, dims) && t.scalar_type() == at::kInt && t.size(0) == B && (t.size(dims - 1) <= 1 || t.stride(dims - 1) == 1);
}
struct Sequences {
    at::Tensor table, lengths, counts;
    fa_b200_sequences s = {};
    bool take(PyObject* table_o, PyObject* lengths_o, PyObject* counts_o, int device, const at::Tensor& rows) {
        const int64_t B = rows.size(0);
        if (!plain_ints(table_o, table, device, 2, B) || !plain_ints(lengths_o, lengths, device, 1, B) ||
            (counts_o != Py_None && !plain_ints(counts_o, counts, device, 1, B)) || table.size(1) <= 0 || table.size(1) > UINT32_MAX)
            return false;
        s.table = table.data_ptr<int32_t>(), s.lengths = lengths.data_ptr<int32_t>();
        s.counts = counts_o != Py_None ? counts.data_ptr<int32_t>() : nullptr;
        s.table_stride = table.stride(0), s.table_width = static_cast<uint32_t>(table.size(1));
        s.B = static_cast<uint32_t>(B), s.T = static_cast<uint32_t>(rows.size(1));
        return true;
    }
};
// A whole number from a Python int; false for anything else.
bool whole(PyObject* o, int64_t& x) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    x = PyLong_AsLongLongAndOverflow(o, &over);
    return over == 0;
}
template <typename F>
F* address(PyObject* o) {
    if (!PyLong_CheckExact(o)) return nullptr;
    auto* const p = reinterpret_cast<F*>(PyLong_AsVoidPtr(o));
    if (p == nullptr) PyErr_Clear();
    return p;
}
uint32_t dtype_of(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? FA_B200_FP16 : FA_B200_BF16; }
void* stream_of(int device) { return static_cast<void*>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream()); }

// (entry, cache, device, keys, values, table, lengths, counts, queries, rotation, interleaved) -> queries' rotated form, True without any
PyObject* cache_append_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t device = 0;
    if (n != 11 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !whole(args[2], device)) Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_cache_append)>(args[0]);
    auto* const cache = address<const fa_b200_cache>(args[1]);
    if (!entry || !cache) Py_RETURN_NONE;
    const int dev = static_cast<int>(device);
    const int64_t H = cache->head_dim, F = H * cache->kv_heads;
    at::Tensor k, v, q, cos, sin, rotated;
    Sequences seqs;
    if (!plain_rows(args[3], k, dev, F) || k.size(2) != F || !plain_rows(args[4], v, dev, F) || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() ||
        !seqs.take(args[5], args[6], args[7], dev, k))
        Py_RETURN_NONE;
    const bool with_q = args[8] != Py_None, turned = args[9] != Py_None;
    if (with_q && (!plain_rows(args[8], q, dev, H) || q.size(0) != k.size(0) || q.size(1) != k.size(1) || q.scalar_type() != k.scalar_type())) Py_RETURN_NONE;
    if (turned) {
        if (!PyTuple_CheckExact(args[9]) || PyTuple_GET_SIZE(args[9]) != 2) Py_RETURN_NONE;
        for (int i = 0; i < 2; ++i) {
            at::Tensor& t = i ? sin : cos;
            if (!plain_cuda(PyTuple_GET_ITEM(args[9], i), t, dev, 2) || t.scalar_type() != at::kFloat || t.size(1) != H / 2 || t.size(0) <= 0 || !t.is_contiguous() ||
                (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) != 0 || t.sizes() != cos.sizes())
                Py_RETURN_NONE;
        }
    }
    const int neighbours = PyObject_IsTrue(args[10]);
    if (neighbours < 0) return nullptr;
    if (with_q) rotated = at::empty(q.sizes(), q.options());
    const int rc = entry(cache, &seqs.s, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), with_q ? q.data_ptr() : nullptr,
                         with_q ? q.stride(0) : 0, with_q ? q.stride(1) : 0, with_q ? static_cast<uint32_t>(q.size(2) / H) : 0, with_q ? rotated.data_ptr() : nullptr,
                         turned ? cos.data_ptr<float>() : nullptr, turned ? sin.data_ptr<float>() : nullptr,
                         turned ? static_cast<uint32_t>(std::min<int64_t>(cos.size(0), 0x7FFFFFFF)) : 0, dtype_of(k), neighbours ? FA_B200_CACHE_NEIGHBOURS : 0, dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    if (!with_q) Py_RETURN_TRUE;
    return THPVariable_Wrap(std::move(rotated));
    END_HANDLE_TH_ERRORS
}

// (entry, cache, device, queries, table, lengths, counts, keep, first, last) -> pages
PyObject* cache_select_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t device = 0, keep = 0, first = 0, last = 0;
    if (n != 10 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !whole(args[2], device) || !whole(args[7], keep) || !whole(args[8], first) ||
        !whole(args[9], last) || keep < 1 || keep > 0x7FFFFFFF || first < 0 || last < 1)
        Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_cache_select)>(args[0]);
    auto* const cache = address<const fa_b200_cache>(args[1]);
    if (!entry || !cache) Py_RETURN_NONE;
    const int dev = static_cast<int>(device);
    at::Tensor q;
    Sequences seqs;
    if (!plain_rows(args[3], q, dev, static_cast<int64_t>(cache->head_dim) * cache->kv_heads) || !seqs.take(args[4], args[5], args[6], dev, q)) Py_RETURN_NONE;
    const auto ints = q.options().dtype(at::kInt);
    const int64_t rows = q.size(0) * q.size(1) * cache->kv_heads;
    at::Tensor pages = at::empty({q.size(0), q.size(1), cache->kv_heads, keep}, ints);
    const at::Tensor scratch = at::empty({rows * seqs.s.table_width}, ints);
    const int rc = entry(cache, &seqs.s, q.data_ptr(), q.stride(0), q.stride(1), static_cast<uint32_t>(q.size(2) / cache->head_dim), dtype_of(q), static_cast<uint32_t>(keep),
                         static_cast<uint32_t>(std::min<int64_t>(first, 0x7FFFFFFF)), static_cast<uint32_t>(std::min<int64_t>(last, 0x7FFFFFFF)), pages.data_ptr<int32_t>(),
                         scratch.data_ptr(), 4 * static_cast<uint64_t>(scratch.numel()), dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(pages));
    END_HANDLE_TH_ERRORS
}

// (entry, entry for the scratch's size, cache, device, queries, table, lengths, counts, pages, causal, out) -> y
PyObject* cache_attention_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t device = 0;
    if (n != 11 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !whole(args[3], device)) Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_cache_attention)>(args[0]);
    auto* const size_of = address<decltype(fa_b200_cache_attention_scratch)>(args[1]);
    auto* const cache = address<const fa_b200_cache>(args[2]);
    if (!entry || !size_of || !cache) Py_RETURN_NONE;
    const int dev = static_cast<int>(device);
    at::Tensor q, pages, out;
    Sequences seqs;
    if (!plain_rows(args[4], q, dev, static_cast<int64_t>(cache->head_dim) * cache->kv_heads) || !seqs.take(args[5], args[6], args[7], dev, q)) Py_RETURN_NONE;
    const bool some = args[8] != Py_None, given = args[10] != Py_None;
    if (some && (!plain_cuda(args[8], pages, dev, 4) || pages.scalar_type() != at::kInt || pages.size(0) != q.size(0) || pages.size(1) != q.size(1) ||
                 pages.size(2) != cache->kv_heads || pages.size(3) <= 0 || pages.size(3) > 0x7FFFFFFF || !pages.is_contiguous()))
        Py_RETURN_NONE;
    if (given && (!plain_rows(args[10], out, dev, q.size(2)) || out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !out.is_contiguous())) Py_RETURN_NONE;
    const int causal = PyObject_IsTrue(args[9]);
    if (causal < 0) return nullptr;
    const uint32_t heads = static_cast<uint32_t>(q.size(2) / cache->head_dim), keep = some ? static_cast<uint32_t>(pages.size(3)) : 0;
    uint64_t bytes[1] = {0};
    int rc = size_of(cache->head_dim, cache->kv_heads, heads, cache->page_size, seqs.s.B, seqs.s.T, seqs.s.table_width, keep, dev, bytes);
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    if (!given) out = at::empty(q.sizes(), q.options());
    const at::Tensor scratch = at::empty({static_cast<int64_t>(bytes[0])}, q.options().dtype(at::kByte));
    rc = entry(cache, &seqs.s, q.data_ptr(), q.stride(0), q.stride(1), heads, dtype_of(q), some ? pages.data_ptr<int32_t>() : nullptr, keep,
               causal ? 0 : FA_B200_CACHE_ALL_KEYS, out.data_ptr(), scratch.data_ptr(), bytes[0], dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- The calls of the latent cache and of pages, in the same manner.
// 16-bit values of `type` on `device`, with every row on a 16-byte boundary; strides: of all axes but the last, 0 for one that is nowhere stepped along.
bool plain_16bit(PyObject* o, at::Tensor& t, int device, int64_t dims, at::ScalarType type, int64_t* strides) {
    if (!plain_cuda(o, t, device, dims) || t.scalar_type() != type || t.numel() == 0 || t.stride(dims - 1) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) != 0) return false;
    for (int64_t i = 0; i + 1 < dims; ++i) {
        strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
        if (strides[i] % 8 != 0 || t.size(i) > UINT32_MAX) return false;
    }
    return true;
}
bool dtype_code(PyObject* o, at::ScalarType& type) {
    int64_t code = 0;
    if (!whole(o, code) || code < 0 || code > 1) return false;
    type = code == FA_B200_FP16 ? at::kHalf : at::kBFloat16;
    return true;
}
// cos and sin, float32 [positions, half] each, from a tuple
bool plain_rotation(PyObject* o, at::Tensor& cos, at::Tensor& sin, int device, int64_t half) {
    if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 2) return false;
    for (int i = 0; i < 2; ++i) {
        at::Tensor& t = i ? sin : cos;
        if (!plain_cuda(PyTuple_GET_ITEM(o, i), t, device, 2) || t.scalar_type() != at::kFloat || t.size(1) != half || t.size(0) <= 0 || !t.is_contiguous() ||
            (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) != 0 || t.sizes() != cos.sizes())
            return false;
    }
    return true;
}
// A scale that the library takes, from a Python float.
bool positive(PyObject* o, float& x) {
    if (!PyFloat_CheckExact(o)) return false;
    x = static_cast<float>(PyFloat_AS_DOUBLE(o));
    return x >= 0x1p-126f && x <= 1e38f;
}

// (entry, cache, device, dtype, latents, rope_keys, table, lengths, counts, queries, rotation, interleaved) -> (keys, queries or None)
PyObject* latent_append_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t device = 0;
    at::ScalarType type;
    if (n != 12 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !whole(args[2], device) || !dtype_code(args[3], type)) Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_latent_append)>(args[0]);
    auto* const cache = address<const fa_b200_latent_cache>(args[1]);
    if (!entry || !cache) Py_RETURN_NONE;
    const int dev = static_cast<int>(device);
    at::Tensor c, k, q, cos, sin, rotated;
    int64_t cs[2], ks[2], qs[3] = {0, 0, 0};
    Sequences seqs;
    if (!plain_16bit(args[4], c, dev, 3, type, cs) || c.size(2) != cache->latent_dim || !plain_16bit(args[5], k, dev, 3, type, ks) || k.size(0) != c.size(0) ||
        k.size(1) != c.size(1) || k.size(2) != cache->rope_dim || !seqs.take(args[6], args[7], args[8], dev, c))
        Py_RETURN_NONE;
    const bool with_q = args[9] != Py_None, turned = args[10] != Py_None;
    if (with_q && (!plain_16bit(args[9], q, dev, 4, type, qs) || q.size(0) != c.size(0) || q.size(1) != c.size(1) || q.size(3) != cache->rope_dim)) Py_RETURN_NONE;
    if (turned && !plain_rotation(args[10], cos, sin, dev, cache->rope_dim / 2)) Py_RETURN_NONE;
    const int neighbours = PyObject_IsTrue(args[11]);
    if (neighbours < 0) return nullptr;
    at::Tensor keys = at::empty(k.sizes(), k.options());
    if (with_q) rotated = at::empty(q.sizes(), q.options());
    const int rc = entry(cache, &seqs.s, c.data_ptr(), cs[0], cs[1], k.data_ptr(), ks[0], ks[1], with_q ? q.data_ptr() : nullptr, qs[0], qs[1], qs[2],
                         with_q ? static_cast<uint32_t>(q.size(2)) : 0, keys.data_ptr(), with_q ? rotated.data_ptr() : nullptr, turned ? cos.data_ptr<float>() : nullptr,
                         turned ? sin.data_ptr<float>() : nullptr, turned ? static_cast<uint32_t>(std::min<int64_t>(cos.size(0), 0x7FFFFFFF)) : 0, dtype_of(c),
                         neighbours ? FA_B200_CACHE_NEIGHBOURS : 0, dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    THPObjectPtr first(THPVariable_Wrap(std::move(keys))), second(with_q ? THPVariable_Wrap(std::move(rotated)) : Py_NewRef(Py_None));
    if (!first || !second) return nullptr;
    return PyTuple_Pack(2, first.get(), second.get());
    END_HANDLE_TH_ERRORS
}

// (entry, entry for the scratch's size, cache, device, dtype, q_latent, q_rope, table, lengths, scale, counts, causal, out) -> y
PyObject* latent_attention_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t device = 0;
    at::ScalarType type;
    float scale = 0;
    if (n != 13 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !whole(args[3], device) || !dtype_code(args[4], type) || !positive(args[9], scale)) Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_latent_attention)>(args[0]);
    auto* const size_of = address<decltype(fa_b200_latent_attention_scratch)>(args[1]);
    auto* const cache = address<const fa_b200_latent_cache>(args[2]);
    if (!entry || !size_of || !cache) Py_RETURN_NONE;
    const int dev = static_cast<int>(device);
    at::Tensor ql, qr, out;
    int64_t ls[3], rs[3], os[3];
    Sequences seqs;
    if (!plain_16bit(args[5], ql, dev, 4, type, ls) || ql.size(3) != cache->latent_dim || !plain_16bit(args[6], qr, dev, 4, type, rs) || qr.size(0) != ql.size(0) ||
        qr.size(1) != ql.size(1) || qr.size(2) != ql.size(2) || qr.size(3) != cache->rope_dim || !seqs.take(args[7], args[8], args[10], dev, ql))
        Py_RETURN_NONE;
    const bool given = args[12] != Py_None;
    if (given && (!plain_16bit(args[12], out, dev, 4, type, os) || out.sizes() != ql.sizes() || !out.is_contiguous())) Py_RETURN_NONE;
    const int causal = PyObject_IsTrue(args[11]);
    if (causal < 0) return nullptr;
    const uint32_t heads = static_cast<uint32_t>(ql.size(2));
    uint64_t bytes[1] = {0};
    int rc = size_of(cache->latent_dim, heads, cache->page_size, seqs.s.B, seqs.s.T, seqs.s.table_width, dev, bytes);
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    if (!given) out = at::empty(ql.sizes(), ql.options());
    const at::Tensor scratch = at::empty({static_cast<int64_t>(bytes[0])}, ql.options().dtype(at::kByte));
    rc = entry(cache, &seqs.s, ql.data_ptr(), ls[0], ls[1], ls[2], qr.data_ptr(), rs[0], rs[1], rs[2], heads, scale, dtype_of(ql), causal ? 0 : FA_B200_CACHE_ALL_KEYS,
               out.data_ptr(), scratch.data_ptr(), bytes[0], dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// (entry, q_nope, q_rope, expanded, rope_keys, scale or None, lengths, counts, causal, out) -> y
PyObject* latent_prompt_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !THPVariable_CheckExact(args[1])) Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_latent_prompt)>(args[0]);
    if (!entry) Py_RETURN_NONE;
    const at::Tensor& first = THPVariable_Unpack(args[1]);
    if (!first.defined() || !first.is_cuda() || (first.scalar_type() != at::kHalf && first.scalar_type() != at::kBFloat16)) Py_RETURN_NONE;
    const int dev = first.get_device();
    const at::ScalarType type = first.scalar_type();
    at::Tensor qn, qr, kv, rk, lengths, counts, out;
    int64_t ns[3], rs[3], vs[3], ks[2], os[3];
    if (!plain_16bit(args[1], qn, dev, 4, type, ns) || !plain_16bit(args[2], qr, dev, 4, type, rs) || !plain_16bit(args[3], kv, dev, 4, type, vs) ||
        !plain_16bit(args[4], rk, dev, 3, type, ks))
        Py_RETURN_NONE;
    const int64_t B = qn.size(0), T = qn.size(1), heads = qn.size(2), nope = qn.size(3), rope = qr.size(3), S = kv.size(1);
    if ((nope != 64 && nope != 128) || (rope != 16 && rope != 32 && rope != 64) || qr.size(0) != B || qr.size(1) != T || qr.size(2) != heads || kv.size(0) != B ||
        kv.size(2) != heads || kv.size(3) != 2 * nope || rk.size(0) != B || rk.size(1) != S || rk.size(2) != rope)
        Py_RETURN_NONE;
    float scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(nope + rope)));
    if (args[5] != Py_None && !positive(args[5], scale)) Py_RETURN_NONE;
    if ((args[6] != Py_None && !plain_ints(args[6], lengths, dev, 1, B)) || (args[7] != Py_None && !plain_ints(args[7], counts, dev, 1, B))) Py_RETURN_NONE;
    const int causal = PyObject_IsTrue(args[8]);
    if (causal < 0) return nullptr;
    const bool given = args[9] != Py_None;
    if (given && (!plain_16bit(args[9], out, dev, 4, type, os) || out.size(0) != B || out.size(1) != T || out.size(2) != heads || out.size(3) != nope || !out.is_contiguous())) Py_RETURN_NONE;
    for (const int64_t stride : {B > 1 ? ns[0] : 1, T > 1 ? ns[1] : 1, heads > 1 ? ns[2] : 1, B > 1 ? rs[0] : 1, T > 1 ? rs[1] : 1, heads > 1 ? rs[2] : 1, B > 1 ? vs[0] : 1,
                                 S > 1 ? vs[1] : 1, heads > 1 ? vs[2] : 1, B > 1 ? ks[0] : 1, S > 1 ? ks[1] : 1})
        if (stride <= 0) Py_RETURN_NONE;
    if (!given) out = at::empty({B, T, heads, nope}, qn.options());
    const int rc = entry(qn.data_ptr(), ns[0], ns[1], ns[2], qr.data_ptr(), rs[0], rs[1], rs[2], kv.data_ptr(), vs[0], vs[1], vs[2], rk.data_ptr(), ks[0], ks[1],
                         lengths.defined() ? lengths.data_ptr<int32_t>() : nullptr, counts.defined() ? counts.data_ptr<int32_t>() : nullptr, static_cast<uint32_t>(B),
                         static_cast<uint32_t>(T), static_cast<uint32_t>(S), static_cast<uint32_t>(heads), static_cast<uint32_t>(nope), static_cast<uint32_t>(rope), scale,
                         dtype_of(qn), causal ? 0 : FA_B200_CACHE_ALL_KEYS, out.data_ptr(), dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// A table [B, W] of whole numbers whose rows do not overlap.
bool plain_table(PyObject* o, at::Tensor& t, int device) {
    return plain_cuda(o, t, device, 2) && t.scalar_type() == at::kInt && t.size(0) > 0 && t.size(1) > 0 && t.size(0) <= UINT32_MAX && t.size(1) <= 0x7FFFFFFF &&
           (t.size(1) == 1 || t.stride(1) == 1) && (t.size(0) == 1 || t.stride(0) >= t.size(1));
}

// (entry, pool, device, table, lengths, parents) -> True
PyObject* pages_fork_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t device = 0;
    if (n != 6 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !whole(args[2], device)) Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_pages_fork)>(args[0]);
    auto* const pool = address<const fa_b200_pages>(args[1]);
    if (!entry || !pool) Py_RETURN_NONE;
    const int dev = static_cast<int>(device);
    at::Tensor table, lengths, parents;
    if (!plain_table(args[3], table, dev) || !plain_ints(args[4], lengths, dev, 1, table.size(0)) || !plain_ints(args[5], parents, dev, 1, table.size(0)) || table.size(0) > 57344)
        Py_RETURN_NONE;
    const int rc = entry(pool, table.data_ptr<int32_t>(), table.stride(0), static_cast<uint32_t>(table.size(1)), static_cast<uint32_t>(table.size(0)),
                         lengths.data_ptr<int32_t>(), parents.data_ptr<int32_t>(), dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// (entry, pool, device, table, lengths, counts, page_size) -> (granted, sources, targets)
PyObject* pages_reserve_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t device = 0, page = 0, count = 0;
    if (n != 7 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !whole(args[2], device) || !whole(args[6], page) || (page != 16 && page != 32 && page != 64 && page != 128))
        Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_pages_reserve)>(args[0]);
    auto* const pool = address<const fa_b200_pages>(args[1]);
    if (!entry || !pool) Py_RETURN_NONE;
    const int dev = static_cast<int>(device);
    at::Tensor table, lengths, counts;
    if (!plain_table(args[3], table, dev) || !plain_ints(args[4], lengths, dev, 1, table.size(0))) Py_RETURN_NONE;
    if (PyLong_CheckExact(args[5])) {
        if (!whole(args[5], count) || count < 0 || count > 0x7FFFFFFF) Py_RETURN_NONE;
    } else if (!plain_ints(args[5], counts, dev, 1, table.size(0))) {
        Py_RETURN_NONE;
    }
    const int64_t B = table.size(0);
    const at::Tensor all = at::empty({3, B}, table.options()), scratch = at::empty({static_cast<int64_t>(pool->n_pages)}, table.options());
    int32_t* const to = all.data_ptr<int32_t>();
    const int rc = entry(pool, table.data_ptr<int32_t>(), table.stride(0), static_cast<uint32_t>(table.size(1)), static_cast<uint32_t>(B), lengths.data_ptr<int32_t>(),
                         counts.defined() ? counts.data_ptr<int32_t>() : nullptr, static_cast<uint32_t>(count), static_cast<uint32_t>(page), to, to + B, to + 2 * B,
                         scratch.data_ptr(), 4 * static_cast<uint64_t>(pool->n_pages), dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    THPObjectPtr a(THPVariable_Wrap(all.select(0, 0))), b(THPVariable_Wrap(all.select(0, 1))), c(THPVariable_Wrap(all.select(0, 2)));
    if (!a || !b || !c) return nullptr;
    return PyTuple_Pack(3, a.get(), b.get(), c.get());
    END_HANDLE_TH_ERRORS
}

// (entry, pool, device, table) -> (refs, table, sources, targets)
PyObject* pages_compact_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t device = 0;
    if (n != 4 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !whole(args[2], device)) Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_pages_compact)>(args[0]);
    auto* const pool = address<const fa_b200_pages>(args[1]);
    if (!entry || !pool) Py_RETURN_NONE;
    const int dev = static_cast<int>(device);
    at::Tensor table;
    if (!plain_table(args[3], table, dev)) Py_RETURN_NONE;
    const int64_t pages = pool->n_pages;
    at::Tensor refs = at::empty({pages}, table.options()), renumbered = at::empty({table.size(0), table.size(1)}, table.options());
    const at::Tensor moves = at::empty({2, pages}, table.options()), scratch = at::empty({pages + 2}, table.options());
    int32_t* const to = moves.data_ptr<int32_t>();
    const int rc = entry(pool, table.data_ptr<int32_t>(), table.stride(0), static_cast<uint32_t>(table.size(1)), static_cast<uint32_t>(table.size(0)), refs.data_ptr<int32_t>(),
                         renumbered.data_ptr<int32_t>(), to, to + pages, scratch.data_ptr(), 4 * static_cast<uint64_t>(pages) + 8, dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    THPObjectPtr a(THPVariable_Wrap(std::move(refs))), b(THPVariable_Wrap(std::move(renumbered))), c(THPVariable_Wrap(moves.select(0, 0))), d(THPVariable_Wrap(moves.select(0, 1)));
    if (!a || !b || !c || !d) return nullptr;
    return PyTuple_Pack(4, a.get(), b.get(), c.get(), d.get());
    END_HANDLE_TH_ERRORS
}

// (entry, ((address of areas, how many), ...) by cache, pages of a cache, address of the status, device, sources, targets) -> True
PyObject* cache_copy_through(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t pages = 0, device = 0;
    if (n != 7 || at::impl::PythonTorchFunctionTLS::stack_len() > 0 || !PyTuple_CheckExact(args[1]) || !whole(args[2], pages) || !whole(args[4], device)) Py_RETURN_NONE;
    auto* const entry = address<decltype(fa_b200_cache_copy)>(args[0]);
    auto* const status = address<uint32_t>(args[3]);
    if (!entry || !status) Py_RETURN_NONE;
    const int dev = static_cast<int>(device);
    at::Tensor sources, targets;
    if (!plain_cuda(args[5], sources, dev, 1) || sources.scalar_type() != at::kInt || sources.numel() == 0 || sources.numel() > 0x7FFFFFFF ||
        (sources.numel() > 1 && sources.stride(0) != 1) || !plain_ints(args[6], targets, dev, 1, sources.size(0)))
        Py_RETURN_NONE;
    std::vector<fa_b200_copy_area> areas;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[1]); ++i) {
        PyObject* const cache = PyTuple_GET_ITEM(args[1], i);
        int64_t count = 0;
        if (!PyTuple_CheckExact(cache) || PyTuple_GET_SIZE(cache) < 2 || !whole(PyTuple_GET_ITEM(cache, 1), count)) Py_RETURN_NONE;
        auto* const from = address<const fa_b200_copy_area>(PyTuple_GET_ITEM(cache, 0));
        if (!from) Py_RETURN_NONE;
        areas.insert(areas.end(), from, from + count);
    }
    const int rc = entry(areas.data(), static_cast<uint32_t>(areas.size()), static_cast<uint32_t>(pages), sources.data_ptr<int32_t>(), targets.data_ptr<int32_t>(),
                         static_cast<uint32_t>(sources.numel()), status, dev, stream_of(dev));
    if (rc != FA_B200_OK) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*kFunction)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* native_function(const char* name) {
    static PyMethodDef def = {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kFunction)), METH_FASTCALL, nullptr};
    return PyCFunction_New(&def, nullptr);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("attention_forward", &attention_forward, py::arg("head_dim"), py::arg("chunk_size"), py::arg("queries"),
          py::arg("keys"), py::arg("values"), py::arg("mask") = torch::optional<torch::Tensor>(),
          "Fused multihead attention");
    m.add_object("_forward_through", PyCFunction_New(&forward_through_def, nullptr));
    m.add_object("_cache_append_through", native_function<&cache_append_through>("_cache_append_through"));
    m.add_object("_cache_select_through", native_function<&cache_select_through>("_cache_select_through"));
    m.add_object("_cache_attention_through", native_function<&cache_attention_through>("_cache_attention_through"));
    m.add_object("_latent_append_through", native_function<&latent_append_through>("_latent_append_through"));
    m.add_object("_latent_attention_through", native_function<&latent_attention_through>("_latent_attention_through"));
    m.add_object("_latent_prompt_through", native_function<&latent_prompt_through>("_latent_prompt_through"));
    m.add_object("_pages_fork_through", native_function<&pages_fork_through>("_pages_fork_through"));
    m.add_object("_pages_reserve_through", native_function<&pages_reserve_through>("_pages_reserve_through"));
    m.add_object("_pages_compact_through", native_function<&pages_compact_through>("_pages_compact_through"));
    m.add_object("_cache_copy_through", native_function<&cache_copy_through>("_cache_copy_through"));
}
