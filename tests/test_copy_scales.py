"""cache_copy takes every cache that the other calls take: scales need only be contiguous, whatever boundary they start on and however many heads there are."""
import ctypes
import random

import pytest
import torch

import fused_attention_b200 as fa
from fused_attention_b200 import _lib, pages


def codes(n, heads, rows, H, device):
    return torch.randint(0, 120, (n, heads, rows, H), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)


def scales(n, heads, offset, device):
    """A slice of a larger buffer, `offset` values into it."""
    return torch.rand(offset + n * heads, device=device)[offset:].view(n, heads)


@pytest.mark.parametrize("heads", [1, 3, 4, 8, 20])
@pytest.mark.parametrize("offset", [0, 1, 2, 4])
def test_the_areas_of_a_cache(heads, offset):
    """Without a GPU: a stand-in for a cache with the tensors of one."""
    n, page, H = 5, 16, 32
    cache = object.__new__(fa.KVCache)
    cache._copy_areas = None
    cache.k, cache.v, cache.bounds = codes(n, heads, page, H, "cpu"), codes(n, heads, page, H, "cpu"), codes(n, heads, 2, H, "cpu")
    cache.k_scale, cache.v_scale = scales(n, heads, offset, "cpu"), scales(n, heads, offset, "cpu")
    _, count, areas = pages._areas(cache)
    moved = 0
    for area in areas:
        out = (ctypes.c_uint32 * 4)()
        assert _lib.load().fa_b200_describe_copy(ctypes.byref(area), out) == _lib.OK
        moved += out[0] * out[1] * out[2]
    assert count == len(areas) and moved == heads * (2 * page * H + 2 * H + 8)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,offset", [(4, 1), (8, 2), (8, 0), (3, 1), (1, 3)])
def test_copied_on_the_gpu(heads, offset):
    n, page, H = 9, 16, 32
    cache = fa.KVCache(codes(n, heads, page, H, "cuda"), codes(n, heads, page, H, "cuda"), scales(n, heads, offset, "cuda"), scales(n, heads, offset, "cuda"),
                       codes(n, heads, 2, H, "cuda"))
    tensors = (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.bounds)
    before = [t.clone() for t in tensors]
    both = random.Random(heads).sample(range(n), 6)
    fa.cache_copy(cache, *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (both[:3], both[3:])))
    for now, was in zip(tensors, before):
        want = was.view(torch.uint8).clone()
        want[both[3:]] = was.view(torch.uint8)[both[:3]]
        assert torch.equal(now.view(torch.uint8), want)
    assert cache.read_status() == (0, 0)
