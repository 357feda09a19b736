"""Attention and selection over a cache that has a scale below zero, which no append writes."""
import pytest
import torch

import fused_attention_b200 as fa
from test_cache_gpu import queries_of, random_cache, table_of

pytestmark = pytest.mark.gpu
FP16 = torch.float16


@pytest.mark.parametrize("T", [1, 4, 90])
def test_scales_below_zero_are_not_numbers(T):
    """A key's or value's scale below zero makes the queries that see its page NaN, and no others."""
    H, G, page = 64, 2, 16
    cache = random_cache(H, G, 40, page, T)
    table, lengths = table_of([T + 200], page, 40, 4)
    q = queries_of(1, T, G * 2 * H, FP16, T)
    want = fa.cache_attention(cache, q, table, lengths)
    last = int(table[0, (T + 199) // page])
    first_in_last = (T + 199) // page * page - 200            # queries from this one on see the last page
    for scale in (cache.k_scale, cache.v_scale):
        was = float(scale[last, 1])
        scale[last, 1] = -was
        y = fa.cache_attention(cache, q, table, lengths)
        half = G * H
        assert torch.equal(y[..., :half], want[..., :half])
        at = max(0, first_in_last)
        assert torch.isnan(y[:, at:, half:]).all() and torch.equal(y[:, :at, half:], want[:, :at, half:])
        scale[last, 1] = was
    assert cache.read_status() == (0, 0)


@pytest.mark.parametrize("W", [20, 300, 9000])
def test_selection_takes_them_for_scores_that_are_not_numbers(W):
    """-1 among them, alone and beside a table entry that is none: these pages come behind the first and last ones, before all others."""
    H, G, page = 32, 2, 16
    cache = random_cache(H, G, W, page, W)
    cache.k_scale[2:12, 1] = -1.0
    table = torch.arange(W, dtype=torch.int32, device="cuda")[None].contiguous()
    lengths = torch.tensor([W * page - 3], dtype=torch.int32, device="cuda")
    q = queries_of(1, 2, 4 * H, FP16, 1)
    got = fa.cache_select(cache, q, table, lengths, 15, first=2, last=3)
    assert got[0, :, 1].tolist() == [list(range(12)) + [W - 3, W - 2, W - 1]] * 2 and cache.read_status() == (0, 0)
    table[0, 5] = -1
    got = fa.cache_select(cache, q, table, lengths, 14, first=2, last=3)
    assert got[0, :, 1].tolist() == [[0, 1, 2, 3, 4, 6, 7, 8, 9, 10, 11, W - 3, W - 2, W - 1]] * 2 and cache.read_status()[0] == 1
