"""The C ABI of the latent cache and of pages without a GPU: structures as the header declares them, and what is rejected before any CUDA call."""
import ctypes
import os
import re

import pytest
import torch

import fused_attention_b200 as fa
from fused_attention_b200 import _lib

BUF = ctypes.create_string_buffer(256)
A = (ctypes.addressof(BUF) + 63) & ~63


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cache(**kw):
    return _lib.LatentCache(**{**dict(data=A, status=A, page_stride=16 * 1152, token_stride=1152, n_pages=4, page_size=16, latent_dim=512, rope_dim=64), **kw})


def seqs(**kw):
    return _lib.Sequences(**{**dict(table=A, lengths=A, counts=None, table_stride=4, table_width=4, B=2, T=1), **kw})


def append(lib, c=None, s=None, latents=A, lt=576, keys=A, q=None, qh=64, heads=0, out=A, q_out=None, cos=None, sin=None, dtype=0, flags=0):
    return lib.fa_b200_latent_append(ctypes.byref(c or cache()), ctypes.byref(s or seqs()), latents, 576, lt, keys, 576, 576, q, 64, 64, qh, heads, out, q_out, cos, sin, 8,
                                     dtype, flags, 0, None)


def attention(lib, c=None, s=None, ql=A, qlh=512, qr=A, heads=4, scale=0.1, dtype=0, flags=0, y=A, scratch=A, size=0):
    return lib.fa_b200_latent_attention(ctypes.byref(c or cache()), ctypes.byref(s or seqs()), ql, 2048, 2048, qlh, qr, 256, 256, 64, heads, scale, dtype, flags, y, scratch,
                                        size, 0, None)


def prompt(lib, qn=A, kv=A, vh=256, rk=A, lengths=None, B=1, T=4, S=4, heads=2, nope=128, rope=64, scale=0.1, dtype=0, flags=0, y=A):
    return lib.fa_b200_latent_prompt(qn, 1024, 256, 128, A, 512, 128, 64, kv, 2048, 512, vh, rk, 256, 64, lengths, None, B, T, S, heads, nope, rope, scale, dtype, flags, y, 0, None)


def test_structures_are_those_of_the_header(repo_root):
    with open(os.path.join(repo_root, "include", "fa_b200.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    for name, struct in (("fa_b200_latent_cache", _lib.LatentCache), ("fa_b200_pages", _lib.Pages), ("fa_b200_copy_area", _lib.CopyArea)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        fields = []
        for line in body.split(";"):
            m = re.match(r"\s*(const )?(void|float|uint32_t|int32_t|int64_t)\s*(.*)", line.strip(), flags=re.S)
            if m:
                for field in m.group(3).split(","):
                    kind = ctypes.c_void_p if "*" in field else {"uint32_t": ctypes.c_uint32, "int64_t": ctypes.c_int64}[m.group(2)]
                    fields.append((field.replace("*", "").strip(), kind))
        assert fields == struct._fields_, name


@pytest.mark.parametrize("call", [append, attention])
def test_what_both_cache_calls_look_at(lib, call):
    for field in ("data", "status"):
        assert call(lib, c=cache(**{field: None})) == _lib.ERR_NULL_POINTER
    for bad in (dict(latent_dim=64), dict(latent_dim=576), dict(rope_dim=0), dict(rope_dim=48), dict(rope_dim=128)):
        assert call(lib, c=cache(**bad)) == _lib.ERR_HEAD_DIM
    for page in (0, 8, 48, 256):
        assert call(lib, c=cache(page_size=page)) == _lib.ERR_PAGE
    for bad in (dict(data=A + 8), dict(page_stride=1160), dict(token_stride=1160), dict(status=A + 2)):
        assert call(lib, c=cache(**bad)) == _lib.ERR_ALIGNMENT
    for bad in (dict(n_pages=0), dict(n_pages=0x7FFFFFFF), dict(page_stride=-16), dict(token_stride=1 << 25)):
        assert call(lib, c=cache(**bad)) == _lib.ERR_SHAPE
    for bad in (dict(B=0), dict(T=0), dict(table_width=0), dict(table_width=1 << 30)):
        assert call(lib, s=seqs(**bad)) == _lib.ERR_SHAPE
    for bad in (dict(table=None), dict(lengths=None)):
        assert call(lib, s=seqs(**bad)) == _lib.ERR_NULL_POINTER
    assert call(lib, s=seqs(counts=A + 2)) == _lib.ERR_ALIGNMENT
    assert call(lib, dtype=2) == _lib.ERR_DTYPE


def test_append_rejections(lib):
    assert append(lib, latents=None) == _lib.ERR_NULL_POINTER
    assert append(lib, keys=A + 2) == _lib.ERR_ALIGNMENT
    assert append(lib, lt=580) == _lib.ERR_ALIGNMENT
    assert append(lib, out=None) == _lib.ERR_NULL_POINTER
    assert append(lib, q=A, heads=2) == _lib.ERR_NULL_POINTER             # nowhere to put them
    assert append(lib, q=A, heads=0, q_out=A) == _lib.ERR_SHAPE
    assert append(lib, q=A, heads=2, qh=68, q_out=A) == _lib.ERR_ALIGNMENT
    assert append(lib, cos=A) == _lib.ERR_NULL_POINTER
    assert append(lib, cos=A, sin=A + 4) == _lib.ERR_ALIGNMENT
    assert append(lib, flags=2) == _lib.ERR_FLAGS


def test_attention_rejections(lib):
    for bad in (dict(ql=None), dict(qr=None), dict(y=None), dict(scratch=None)):
        assert attention(lib, **bad) == _lib.ERR_NULL_POINTER
    assert attention(lib, qlh=516) == _lib.ERR_ALIGNMENT
    assert attention(lib, flags=1) == _lib.ERR_FLAGS
    for bad in (dict(heads=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(scale=1e-39), dict(scale=2e38), dict(heads=1 << 31)):
        assert attention(lib, **bad) == _lib.ERR_SHAPE


def test_prompt_rejections(lib):
    for bad in (dict(qn=None), dict(kv=None), dict(rk=None), dict(y=None)):
        assert prompt(lib, **bad) == _lib.ERR_NULL_POINTER
    for bad in (dict(qn=A + 2), dict(vh=260), dict(lengths=A + 2)):
        assert prompt(lib, **bad) == _lib.ERR_ALIGNMENT
    for bad in (dict(nope=96), dict(nope=256), dict(rope=8), dict(rope=128)):
        assert prompt(lib, **bad) == _lib.ERR_HEAD_DIM
    for bad in (dict(B=0), dict(T=0), dict(S=0), dict(heads=0), dict(scale=0.0), dict(scale=float("nan"))):
        assert prompt(lib, **bad) == _lib.ERR_SHAPE
    assert prompt(lib, dtype=2) == _lib.ERR_DTYPE
    assert prompt(lib, flags=1) == _lib.ERR_FLAGS


def test_pages_rejections(lib):
    def pages(**kw):
        return ctypes.byref(_lib.Pages(**{**dict(refs=A, status=A, n_pages=8), **kw}))

    def fork(p=None, table=A, W=4, B=2, lengths=A, parents=A):
        return lib.fa_b200_pages_fork(p or pages(), table, 4, W, B, lengths, parents, 0, None)

    def reserve(p=None, table=A, W=4, B=2, lengths=A, counts=A, count=0, page=16, out=A, scratch=A, size=32):
        return lib.fa_b200_pages_reserve(p or pages(), table, 4, W, B, lengths, counts, count, page, out, out, out, scratch, size, 0, None)

    def compact(p=None, table=A, W=4, B=2, out=A, scratch=A, size=40):
        return lib.fa_b200_pages_compact(p or pages(), table, 4, W, B, out, out, out, out, scratch, size, 0, None)
    for call in (fork, reserve, compact):
        for bad in (dict(refs=None), dict(status=None)):
            assert call(p=pages(**bad)) == _lib.ERR_NULL_POINTER
        assert call(p=pages(refs=A + 2)) == _lib.ERR_ALIGNMENT
        for n in (0, 1 << 30):
            assert call(p=pages(n_pages=n)) == _lib.ERR_SHAPE
        assert call(table=None) == _lib.ERR_NULL_POINTER
        assert call(table=A + 1) == _lib.ERR_ALIGNMENT
        assert call(W=0) == _lib.ERR_SHAPE and call(B=0) == _lib.ERR_SHAPE
    assert fork(B=57345) == _lib.ERR_TOO_LARGE
    assert fork(parents=None) == _lib.ERR_NULL_POINTER
    assert reserve(page=8) == _lib.ERR_PAGE
    assert reserve(count=1 << 31) == _lib.ERR_SHAPE
    assert reserve(size=31) == _lib.ERR_TOO_LARGE and compact(size=39) == _lib.ERR_TOO_LARGE
    assert reserve(out=None) == _lib.ERR_NULL_POINTER and compact(out=None) == _lib.ERR_NULL_POINTER

    def copy(n=1, n_pages=8, pairs=1, status=A, sources=A, **kw):
        area = _lib.CopyArea(**{**dict(base=A, page_stride=64, stride0=32, stride1=16, n0=2, n1=2, row_bytes=16), **kw})
        return lib.fa_b200_cache_copy(ctypes.byref(area), n, n_pages, sources, A, pairs, status, 0, None)
    for bad in (dict(base=None), dict(status=None), dict(sources=None)):
        assert copy(**bad) == _lib.ERR_NULL_POINTER
    for bad in (dict(base=A + 8), dict(page_stride=72), dict(stride1=8), dict(row_bytes=6), dict(sources=A + 2)):
        assert copy(**bad) == _lib.ERR_ALIGNMENT
    for bad in (dict(n=0), dict(n_pages=0), dict(pairs=0), dict(n0=0), dict(row_bytes=0)):
        assert copy(**bad) == _lib.ERR_SHAPE


def test_python_refuses_what_is_not_on_a_gpu():
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.LatentCache(torch.zeros(2, 16, 576, dtype=torch.bfloat16), 512)
    with pytest.raises(RuntimeError, match="float16"):
        fa.LatentCache(torch.zeros(2, 16, 576), 512)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.PagePool(torch.zeros(4, dtype=torch.int32))
    for bad in (dict(latent_dim=64), dict(rope_dim=8), dict(n_pages=0), dict(page_size=8), dict(dtype=torch.float32)):
        with pytest.raises(RuntimeError, match="must be"):
            fa.latent_cache_create(**{**dict(latent_dim=512, rope_dim=64, n_pages=8), **bad})
    with pytest.raises(RuntimeError, match="n_pages"):
        fa.page_pool_create(0)
    for f in (lambda: fa.latent_append(None, None, None, None, None), lambda: fa.latent_attention(None, None, None, None, None, scale=1.0)):
        with pytest.raises(RuntimeError, match="LatentCache"):
            f()
    for f in (lambda: fa.pages_fork(None, None, None, None), lambda: fa.pages_reserve(None, None, None, 1, 64), lambda: fa.pages_compact(None, None)):
        with pytest.raises(RuntimeError, match="PagePool"):
            f()
    with pytest.raises(RuntimeError, match="KVCache, a LatentCache"):
        fa.cache_copy([], None, None)
    q = torch.zeros(1, 2, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.latent_prompt(q, q, q, q)
