"""The C ABI of the key/value cache without a GPU: structures as the header declares them, and what is rejected before any CUDA call."""
import ctypes
import os
import re

import pytest

from fused_attention_b200 import _lib

BUF = ctypes.create_string_buffer(256)
A = (ctypes.addressof(BUF) + 63) & ~63


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cache(**kw):
    d = dict(k=A, v=A, k_scale=A, v_scale=A, bounds=A, status=A, k_page_stride=4096, k_head_stride=1024, k_token_stride=64, v_page_stride=4096,
             v_head_stride=1024, v_token_stride=64, n_pages=4, kv_heads=2, page_size=16, head_dim=64)
    return _lib.Cache(**{**d, **kw})


def seqs(**kw):
    return _lib.Sequences(**{**dict(table=A, lengths=A, counts=None, table_stride=4, table_width=4, B=2, T=1), **kw})


def append(lib, c=None, s=None, keys=A, kb=128, kt=128, values=A, q=None, heads=0, rotated=None, cos=None, sin=None, dtype=0, flags=0):
    return lib.fa_b200_cache_append(ctypes.byref(c or cache()), ctypes.byref(s or seqs()), keys, kb, kt, values, 128, 128, q, 256, 256, heads, rotated, cos, sin, 8, dtype,
                                    flags, 0, None)


def select(lib, c=None, s=None, q=A, heads=4, dtype=0, keep=2, last=1, pages=A, scratch=A, size=1 << 20):
    return lib.fa_b200_cache_select(ctypes.byref(c or cache()), ctypes.byref(s or seqs()), q, 256, 256, heads, dtype, keep, 1, last, pages, scratch, size, 0, None)


def attention(lib, c=None, s=None, q=A, qt=256, heads=4, dtype=0, pages=None, keep=0, flags=0, y=A, scratch=A, size=0):
    return lib.fa_b200_cache_attention(ctypes.byref(c or cache()), ctypes.byref(s or seqs()), q, 256, qt, heads, dtype, pages, keep, flags, y, scratch, size, 0, None)


def test_structures_are_those_of_the_header(repo_root):
    with open(os.path.join(repo_root, "include", "fa_b200.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    for name, struct in (("fa_b200_cache", _lib.Cache), ("fa_b200_sequences", _lib.Sequences)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        fields = []
        for line in body.split(";"):
            m = re.match(r"\s*(const )?(void|float|uint32_t|int32_t|int64_t)\s*(.*)", line.strip(), flags=re.S)
            if m:
                for field in m.group(3).split(","):
                    pointer = "*" in field
                    kind = ctypes.c_void_p if pointer else {"uint32_t": ctypes.c_uint32, "int64_t": ctypes.c_int64}[m.group(2)]
                    fields.append((field.replace("*", "").strip(), kind))
        assert fields == struct._fields_
    for name, value in re.findall(r"FA_B200_(FP16|BF16|CACHE_\w+) = (\d+)u", text):
        assert getattr(_lib, name) == int(value)


@pytest.mark.parametrize("call", [append, select, attention])
def test_what_every_call_looks_at(lib, call):
    for field in ("k", "v", "k_scale", "v_scale", "bounds", "status"):
        assert call(lib, c=cache(**{field: None})) == _lib.ERR_NULL_POINTER
    for H in (0, 8, 48, 256):
        assert call(lib, c=cache(head_dim=H)) == _lib.ERR_HEAD_DIM
    for page in (0, 8, 48, 256):
        assert call(lib, c=cache(page_size=page)) == _lib.ERR_PAGE
    for field in ("k", "v", "bounds"):
        assert call(lib, c=cache(**{field: A + 8})) == _lib.ERR_ALIGNMENT
    for field in ("k_page_stride", "k_head_stride", "k_token_stride", "v_page_stride", "v_head_stride", "v_token_stride"):
        assert call(lib, c=cache(**{field: 72})) == _lib.ERR_ALIGNMENT
    for bad in (dict(n_pages=0), dict(n_pages=1 << 31), dict(kv_heads=0)):
        assert call(lib, c=cache(**bad)) == _lib.ERR_SHAPE
    for bad in (dict(B=0), dict(T=0), dict(table_width=0), dict(table_width=1 << 30)):
        assert call(lib, s=seqs(**bad)) == _lib.ERR_SHAPE
    for bad in (dict(table=None), dict(lengths=None)):
        assert call(lib, s=seqs(**bad)) == _lib.ERR_NULL_POINTER
    assert call(lib, s=seqs(counts=A + 2)) == _lib.ERR_ALIGNMENT
    assert call(lib, dtype=2) == _lib.ERR_DTYPE


def test_append_rejections(lib):
    assert append(lib, keys=None) == _lib.ERR_NULL_POINTER
    assert append(lib, values=A + 2) == _lib.ERR_ALIGNMENT
    assert append(lib, kt=132) == _lib.ERR_ALIGNMENT
    assert append(lib, q=A, heads=2) == _lib.ERR_NULL_POINTER            # nowhere to put them
    assert append(lib, q=A, heads=0, rotated=A) == _lib.ERR_SHAPE
    assert append(lib, cos=A) == _lib.ERR_NULL_POINTER
    assert append(lib, cos=A, sin=A + 4) == _lib.ERR_ALIGNMENT
    assert append(lib, flags=2) == _lib.ERR_FLAGS


def test_select_rejections(lib):
    assert select(lib, pages=None) == _lib.ERR_NULL_POINTER
    assert select(lib, scratch=None) == _lib.ERR_NULL_POINTER
    for bad in (dict(heads=3), dict(heads=0), dict(keep=0), dict(last=0)):
        assert select(lib, **bad) == _lib.ERR_SHAPE
    assert select(lib, size=4 * 2 * 2 * 4 - 1) == _lib.ERR_TOO_LARGE


def test_attention_rejections(lib):
    assert attention(lib, y=None) == _lib.ERR_NULL_POINTER
    assert attention(lib, scratch=None) == _lib.ERR_NULL_POINTER
    assert attention(lib, qt=260) == _lib.ERR_ALIGNMENT
    assert attention(lib, flags=1) == _lib.ERR_FLAGS
    for bad in (dict(heads=3), dict(heads=0), dict(pages=A), dict(keep=3), dict(pages=A, keep=1 << 28)):
        assert attention(lib, **bad) == _lib.ERR_SHAPE


def test_python_refuses_what_is_not_on_a_gpu():
    import torch

    import fused_attention_b200 as fa
    codes = torch.zeros(2, 1, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.KVCache(codes, codes, torch.ones(2, 1), torch.ones(2, 1), torch.zeros(2, 1, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn))
    for bad in (dict(head_dim=48), dict(page_size=8), dict(n_pages=0), dict(kv_heads=0)):
        with pytest.raises(RuntimeError, match="must be"):
            fa.cache_create(**{**dict(head_dim=64, kv_heads=2, n_pages=8, page_size=16), **bad})
    for f in (lambda: fa.cache_attention(None, None, None, None), lambda: fa.cache_select(None, None, None, None, 1), lambda: fa.cache_append(None, None, None, None, None)):
        with pytest.raises(RuntimeError, match="KVCache"):
            f()
