"""A latent cache whose tokens lie further apart than its pages, [page_size, n_pages, width] seen as [n_pages, page_size, width]: rows do not lie on one another,
so that all calls take it."""
import pytest
import torch

import fused_attention_b200 as fa
from test_latent_gpu import BF16, ints, normal, table_of

pytestmark = pytest.mark.gpu


def test_tokens_outside_their_pages():
    latent, rope, page, n, B, heads = 256, 32, 32, 11, 2, 5
    data = normal(1, BF16, page, n, latent + rope).transpose(0, 1)
    plain, cache = fa.LatentCache(data.contiguous(), latent), fa.LatentCache(data, latent)
    table, lengths = table_of([90, 50], page, 9, 1)
    c, r = normal(2, BF16, B, 6, latent), normal(3, BF16, B, 6, rope)
    sources, targets = ints([0, 3]), ints([9, 10])
    ql, qr = normal(4, BF16, B, 6, heads, latent), normal(5, BF16, B, 6, heads, rope)
    for x in (plain, cache):
        fa.latent_append(x, c, r, table, lengths)
        fa.cache_copy(x, sources, targets)
    assert torch.equal(plain.data, cache.data) and torch.equal(cache.data[9], cache.data[0])
    want = fa.latent_attention(plain, ql, qr, table, lengths + 6, scale=0.1)
    assert torch.equal(want, fa.latent_attention(cache, ql, qr, table, lengths + 6, scale=0.1))
    assert cache.read_status() == plain.read_status() == (0, 0)


@pytest.mark.parametrize("shape,strides", [((4, 32), (288, 288)), ((4, 32), (296, 288)), ((4, 32), (288, 296)), ((4, 32), (32 * 288 - 8, 288)), ((4, 32), (280, 4 * 288)), ((2, 32), (256, 296))])
def test_rows_on_one_another_are_still_refused(shape, strides):
    cache = fa.LatentCache(torch.zeros(60000, dtype=BF16, device="cuda").as_strided((*shape, 288), (*strides, 1)), 256)
    with pytest.raises(RuntimeError, match="on top of one another"):
        fa.latent_append(cache, normal(1, BF16, 1, 1, 256), normal(2, BF16, 1, 1, 32), ints([[0]]), ints([0]))
    with pytest.raises(RuntimeError, match="on top of one another"):
        fa.cache_copy(cache, ints([0]), ints([1]))
