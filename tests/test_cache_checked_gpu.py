"""The key/value cache's kernels under the checked build (-DFA_DEBUG): indexes are looked at where addresses are formed, tensor-memory
accesses against the CTA's allocation, tiles, results and scratch are filled with NaN beforehand.  No check may fire, no NaN may
survive, and the bits are the normal build's."""
import ctypes
import os

import pytest
import torch

import fused_attention_b200 as fa
from fused_attention_b200 import _lib, build, cache as module
from test_cache_gpu import angles, queries_of, random_cache, table_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def checked(monkeypatch):
    """Calling it makes the checked library the one that all calls go to."""
    if not os.path.exists(build.DEBUG_LIB):
        pytest.skip("checked library not built (python -m fused_attention_b200.build --debug)")

    def change():
        monkeypatch.setattr(_lib, "_lib", None)
        monkeypatch.setattr(_lib, "LIB_PATH", build.DEBUG_LIB)
        monkeypatch.setattr(module, "_native", None)
    yield change


def twice(checked, call):
    """What `call(cache-making number)` returns under the normal library and under the checked one, and the latter's caches."""
    want = call()
    checked()
    got = call()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("H,G,group,page,T,lengths,counts,causal", [
    (128, 2, 4, 64, 1, [300, 64, 1, 0], None, True), (64, 2, 8, 16, 1, [6000, 17], None, True), (32, 1, 5, 32, 5, [900, 5], [5, 3], True),
    (16, 2, 20, 128, 1, [3000], None, False), (128, 1, 3, 16, 9, [700], None, True),
    (128, 2, 2, 64, 130, [900, 130], [130, 70], True), (64, 4, 1, 32, 300, [300, 800, 500], None, True), (64, 1, 1, 16, 257, [5000], None, False),
    (32, 2, 3, 128, 70, [70, 1000], None, True), (16, 8, 4, 16, 600, [700] * 5, None, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention(checked, H, G, group, page, T, lengths, counts, causal, dtype):
    n = len(lengths) * (max(lengths) // page + 2)
    cache = random_cache(H, G, n, page, T)
    table, held = table_of(lengths, page, n, H)
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    q = queries_of(len(lengths), T, G * group * H, dtype, 2)
    few = [fa.cache_select(cache, q, table, held, 5, counts=counts, last=2)] if T <= 9 else []

    def call():
        return [fa.cache_attention(cache, q, table, held, counts=counts, causal=causal, pages=pages) for pages in [None] + few]
    twice(checked, call)
    assert cache.read_status() == (0, 0)
    assert all(torch.isfinite(y).all() for y in call())


@pytest.mark.parametrize("T", [1, 90])
def test_attention_of_value_scales_far_apart_and_of_missing_pages(checked, T):
    H, G, page = 64, 2, 16
    cache = random_cache(H, G, 60, page, T)
    cache.v_scale.copy_(torch.where(torch.rand_like(cache.v_scale) < 0.5, 2.0 ** -100, 2.0 ** 60))
    table, held = table_of([600], page, 60, 1)
    q = queries_of(1, T, G * 2 * H, torch.bfloat16, 2)
    twice(checked, lambda: [fa.cache_attention(cache, q, table, held)])
    assert cache.read_status() == (0, 0)
    table[0, 7], table[0, 20] = 60, -2
    assert torch.isfinite(fa.cache_attention(cache, q, table, held)).all() and cache.read_status()[0] == 1


@pytest.mark.parametrize("H,G,group,page,T,lengths,keep", [
    (128, 2, 4, 64, 1, [5000, 64], 7), (64, 1, 70, 16, 2, [900, 33], 5), (32, 3, 5, 32, 40, [2000], 9), (16, 1, 1, 16, 3, [140000], 40)])
def test_select(checked, H, G, group, page, T, lengths, keep):
    n = len(lengths) * (max(lengths) // page + 2)
    cache = random_cache(H, G, n, page, T)
    table, held = table_of(lengths, page, n, H)
    q = queries_of(len(lengths), T, G * group * H, torch.float16, 2)
    twice(checked, lambda: [fa.cache_select(cache, q, table, held, keep, last=2)])
    assert cache.read_status() == (0, 0)


@pytest.mark.parametrize("H,G,page,T,held,counts", [
    (128, 2, 64, 1, [0, 1, 63, 130], None), (64, 3, 16, 4, [0, 15, 16], [4, 0, 3]), (32, 1, 32, 70, [30, 31], None), (16, 2, 128, 300, [100], None)])
def test_append(checked, H, G, page, T, held, counts):
    B = len(held)
    n = B * ((max(held) + T) // page + 2)
    caches = [random_cache(H, G, n, page, T) for _ in range(2)]
    table, _ = table_of([h + T for h in held], page, n, T)
    lengths = torch.tensor(held, dtype=torch.int32, device="cuda")
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    keys, values, q = (queries_of(B, T, h * H, torch.bfloat16, h) for h in (G, G, 5 * G))
    left = list(caches)

    def call():
        c = left.pop()
        rotated = fa.cache_append(c, keys, values, table, lengths, counts=counts, queries=q, rotation=angles(max(held) + T, H))
        return [rotated] + [t.view(torch.uint8).clone() for t in (c.k, c.v, c.bounds)] + [c.k_scale.clone(), c.v_scale.clone()]
    twice(checked, call)
    assert all(c.read_status() == (0, 0) for c in caches)


def test_the_checked_library_is_the_one_that_checks(checked):
    """It fills a call's scratch beforehand (here one that an undivided problem does not use to the end), the normal one does not."""
    cache = random_cache(64, 1, 4, 64, 1)
    table, held = table_of([100], 64, 4, 1)
    q = queries_of(1, 1, 64, torch.float16, 1)

    def untouched():
        scratch = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
        y = torch.empty_like(q)
        seqs = _lib.Sequences(table.data_ptr(), held.data_ptr(), None, table.stride(0), table.shape[1], 1, 1)
        assert _lib.load().fa_b200_cache_attention(ctypes.byref(cache._handle), ctypes.byref(seqs), q.data_ptr(), 64, 64, 1, _lib.FP16, None, 0, 0, y.data_ptr(),
                                                   scratch.data_ptr(), scratch.numel(), 0, None) == 0
        torch.cuda.synchronize()
        return not scratch.any()
    torch.cuda.synchronize()
    assert untouched()
    checked()
    assert not untouched()
