"""Attention over pages whose value scales lie as far apart as appending can bring them: 2^-100 (pages of zeros) to 2^110.

Bounds are the oracle's, in which nothing depends on the scales: weights of 2^-25 of the largest and less may be lost where they are
multiplied by values, none where they are summed.  Of the sum a kernel may lose 2^-17 and less of itself at these scales.
"""
import pytest
import torch

import fused_attention_b200 as fa
from test_cache_gpu import check_attention, gen_of, queries_of, random_cache, table_of

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def fill(cache, table, exponents):
    """Value scales 2^exponents[i] for the i-th blocks of all sequences, in turn; codes of zero where that is -100."""
    for b in range(table.shape[0]):
        for i, p in enumerate(table[b].tolist()):
            if p >= 0:
                e = exponents[i % len(exponents)]
                cache.v_scale[p] = 2.0 ** e
                if e == -100:
                    cache.v.view(torch.uint8)[p] = 0


@pytest.mark.parametrize("top", [27, 60, 110])
@pytest.mark.parametrize("pattern", ["zeros first", "zeros last", "in turn", "far behind"])
@pytest.mark.parametrize("H,page,T,group,lengths", [
    (64, 64, 1, 4, [300, 65]), (128, 16, 1, 2, [6000]), (32, 32, 5, 5, [700, 40]),          # rows: undivided, divided, two tiles
    (64, 16, 80, 1, [3000, 300]), (128, 64, 130, 2, [500]), (32, 128, 70, 3, [1000])])      # prompts: in parts, on one key head
def test_pages_of_zeros_count_beside_large_values(H, page, T, group, lengths, pattern, top):
    """Equal scores: every result is the mean of the values, zeros among them."""
    G, width = 2, -(-max(lengths) // page)
    n = len(lengths) * width
    cache = random_cache(H, G, n, page, T)
    table, held = table_of(lengths, page, n, H)
    half = max(1, width // 2)
    fill(cache, table, {"zeros first": [-100] * half + [top] * (width - half), "zeros last": [top] * half + [-100] * (width - half),
                        "in turn": [-100, top], "far behind": [top] + [-100] * max(1, width - 1)}[pattern])
    q = torch.zeros(len(lengths), T, G * group * H, dtype=BF16, device="cuda")
    check_attention(cache, q, table, held)


@pytest.mark.parametrize("low,high,dtype", [(-100, 110, BF16), (-60, 60, BF16), (-100, 4, FP16)])
@pytest.mark.parametrize("H,page,T,group,lengths", [
    (64, 64, 1, 4, [300, 65]), (128, 16, 1, 2, [6000]), (16, 32, 5, 5, [700, 40]), (128, 128, 9, 3, [900]),
    (64, 16, 80, 1, [3000, 300]), (128, 64, 130, 2, [500]), (128, 16, 70, 2, [1200, 70]), (16, 32, 300, 1, [700])])
def test_scales_and_scores_of_any_order(H, page, T, group, lengths, low, high, dtype):
    """Weights and values far apart in either direction: the largest product is not the largest weight's."""
    G, width = 2, -(-max(lengths) // page)
    n = len(lengths) * width
    cache = random_cache(H, G, n, page, T + high)
    cache.v_scale.copy_(torch.exp2(torch.randint(low, high + 1, cache.v_scale.shape, generator=gen_of(high), device="cuda").float()))
    table, held = table_of(lengths, page, n, H)
    q = queries_of(len(lengths), T, G * group * H, dtype, 3, sigma=30.0)
    y = check_attention(cache, q, table, held)
    assert y.any()
    if T <= 9:
        pages = fa.cache_select(cache, q, table, held, 7)
        check_attention(cache, q, table, held, pages=pages)
