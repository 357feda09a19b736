"""The latent cache's kernels under the checked build (-DFA_DEBUG): copies, indexes and tensor-memory accesses are looked at first, tiles, results
and scratch are filled with NaN beforehand.  No check may fire, no NaN may survive, and the bits are the normal build's."""
import os

import pytest
import torch

import fused_attention_b200 as fa
from fused_attention_b200 import _lib, build, latent as module
from test_latent_gpu import cache_of, ints, normal, table_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def twice(monkeypatch):
    """What a call returns under the normal library and under the checked one."""
    if not os.path.exists(build.DEBUG_LIB):
        pytest.skip("checked library not built (python -m fused_attention_b200.build --debug)")

    def both(call):
        want = call()
        monkeypatch.setattr(_lib, "_lib", None)
        monkeypatch.setattr(_lib, "LIB_PATH", build.DEBUG_LIB)
        monkeypatch.setattr(module, "_native", None)
        module._scratch_bytes.cache_clear()
        got = call()
        torch.cuda.synchronize()
        assert torch.equal(want, got) and torch.isfinite(got).all() and fa.latent_status(0) == (0, 0)
    yield both
    module._scratch_bytes.cache_clear()


@pytest.mark.parametrize("latent,rope,heads,page,T,lengths,counts,causal", [
    (512, 64, 16, 64, 1, [300, 64, 1, 0], None, True), (512, 64, 128, 16, 1, [6000, 17], None, True), (256, 32, 5, 32, 5, [900, 5], [5, 3], True),
    (128, 16, 40, 128, 1, [3000], None, False), (512, 16, 3, 16, 90, [700, 90], None, True), (256, 64, 16, 64, 1, [500] * 70, None, True),
    (128, 64, 64, 32, 1, [12000], None, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention(twice, latent, rope, heads, page, T, lengths, counts, causal, dtype):
    n = len(lengths) * (max(lengths) // page + 2)
    cache = cache_of(latent, rope, n, page, dtype, T)
    table, held = table_of(lengths, page, n, heads)
    counts = None if counts is None else ints(counts)
    ql, qr = normal(1, dtype, len(lengths), T, heads, latent), normal(2, dtype, len(lengths), T, heads, rope)
    twice(lambda: fa.latent_attention(cache, ql, qr, table, held, scale=0.07, counts=counts, causal=causal))
    assert cache.read_status() == (0, 0)


@pytest.mark.parametrize("nope,rope,T,S,lengths,counts", [(64, 16, 130, 130, None, None), (128, 64, 300, 700, [700, 301], [300, 77]), (128, 32, 1, 900, [900, 5], None)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt(twice, nope, rope, T, S, lengths, counts, dtype):
    q, qr, kv, r = (normal(i, dtype, 2, *n) for i, n in enumerate(((T, 3, nope), (T, 3, rope), (S, 3, 2 * nope), (S, rope))))
    lengths, counts = (None if x is None else ints(x) for x in (lengths, counts))
    for causal in (True, False):
        twice(lambda: fa.latent_prompt(q, qr, kv, r, lengths=lengths, counts=counts, causal=causal))
