"""How exact fp16 results of few query rows are does not depend on what else is in the call, nor on the table's width."""
import pytest
import torch

import fused_attention_b200 as fa
from oracle import kv_cache as oracle
from test_cache_gpu import queries_of, random_cache, table_of

pytestmark = pytest.mark.gpu


def tight(cache, q, table, lengths, **kw):
    """(y, bound) with the weights' 2^-11 out of the oracle's bound: what is left is the result's own rounding, fp32 sums and
    2^-21 for weights of two fp16 numbers."""
    want, bound = oracle.attention(cache, q, table, lengths, **kw)
    codes = cache.v.view(torch.uint8)
    was = codes.clone()
    codes.bitwise_and_(0x7F)
    size, _ = oracle.attention(cache, q, table, lengths, **kw)
    codes.copy_(was)
    return want, bound - (2.0 ** -11 - 2.0 ** -21) * size


@pytest.mark.parametrize("H,G,group,T,B,tokens,keep", [(128, 8, 4, 1, 64, 1100, 0), (64, 4, 2, 2, 130, 1200, 0), (32, 2, 8, 3, 100, 2300, 0), (128, 4, 4, 1, 64, 3000, 30),
                                                       (64, 4, 8, 1, 100, 1100, 0), (128, 4, 3, 3, 100, 1100, 0), (16, 4, 16, 1, 100, 1100, 0), (64, 2, 17, 1, 5, 1100, 0), (64, 2, 12, 2, 40, 900, 9)])
def test_many_sequences_are_as_exact_as_one(H, G, group, T, B, tokens, keep):
    page = 64
    width = -(-tokens // page)
    cache = random_cache(H, G, B * width, page, H)
    table, lengths = table_of([tokens - b for b in range(B)], page, B * width, T)
    q = queries_of(B, T, G * group * H, torch.float16, T, sigma=8.0)      # a few keys have most of the weight
    pages = fa.cache_select(cache, q, table, lengths, keep) if keep else None
    y = fa.cache_attention(cache, q, table, lengths, pages=pages)
    some = slice(0, B, 8)
    want, bound = tight(cache, q[some], table[some], lengths[some], pages=None if pages is None else pages[some].contiguous())
    assert ((y[some].double() - want).abs() <= bound).all()


def test_a_wide_table_changes_nothing():
    H, G, group, page = 128, 8, 4, 64
    cache = random_cache(H, G, 64, page, 3)
    table, lengths = table_of([700, 300, 64, 1], page, 64, 1)
    q = queries_of(4, 1, G * group * H, torch.float16, 1, sigma=8.0)
    want, bound = tight(cache, q, table, lengths)
    for width in (table.shape[1], 100, 2048, 16384):
        wide = torch.full((4, width), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        assert ((fa.cache_attention(cache, q, wide, lengths).double() - want).abs() <= bound).all()
