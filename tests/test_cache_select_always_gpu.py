"""The pages that are selected in any case come before all others, also before those whose score is infinite or not a number."""
import math

import pytest
import torch

import fused_attention_b200 as fa
from test_cache_gpu import queries_of, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("W", [20, 300, 1500, 9000])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_first_and_last_come_before_scores_that_are_not_finite(W, bad):
    H, G, page = 32, 2, 16
    cache = random_cache(H, G, W, page, W)
    cache.k_scale[2:12, 1] = bad
    table = torch.arange(W, dtype=torch.int32, device="cuda")[None].contiguous()
    lengths = torch.tensor([W * page - 3], dtype=torch.int32, device="cuda")
    q = queries_of(1, 2, 4 * H, torch.float16, 1)
    plain = fa.cache_select(cache, q, table, lengths, 6, first=2, last=3)
    assert plain[0, :, 1].tolist() == [[0, 1, 2, W - 3, W - 2, W - 1]] * 2                     # one place is left: for the lowest of them
    few = fa.cache_select(cache, q, table, lengths, 4, first=2, last=3)
    assert few[0].reshape(-1, 4).tolist() == [[0, 1, W - 3, W - 2]] * 4                         # more than there are places for: the lower ones
    exact = fa.cache_select(cache, q, table, lengths, 5, first=2, last=3)
    assert exact[0].reshape(-1, 5).tolist() == [[0, 1, W - 3, W - 2, W - 1]] * 4
    more = fa.cache_select(cache, q, table, lengths, 15, first=2, last=3)
    assert more[0, :, 1].tolist() == [list(range(12)) + [W - 3, W - 2, W - 1]] * 2
    assert cache.read_status() == (0, 0)


def test_scores_that_overflow_do_not_displace_them():
    H, G, page, W = 64, 1, 16, 200
    cache = random_cache(H, G, W, page, 2)
    cache.k_scale.fill_(2.0 ** 100)
    table = torch.arange(W, dtype=torch.int32, device="cuda")[None].contiguous()
    lengths = torch.tensor([W * page], dtype=torch.int32, device="cuda")
    q = (queries_of(1, 1, 2 * H, torch.float32, 1) * 1e30).to(torch.bfloat16)
    got = fa.cache_select(cache, q, table, lengths, 8, first=1, last=4)
    assert got[0, 0, 0].tolist() == [0, 1, 2, 3, W - 4, W - 3, W - 2, W - 1]
