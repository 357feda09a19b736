"""latent_attention on chunks of prompts with many heads, against the 64-bit form: so many groups of rows that CTAs come in several rounds, and so many that
each goes over all sequences by itself; sequences divided and undivided, empty ones, queries in front of the first key, counts.  Within the bounds that
oracle/latent.py derives from the roundings."""
import pytest
import torch

from test_latent_gpu import BF16, F16, cache_of, check, ints, normal, table_of

pytestmark = pytest.mark.gpu


# groups of 64 rows: 100, 200, 592, 600 and 38
@pytest.mark.parametrize("T,heads", [(50, 128), (100, 128), (296, 128), (300, 128), (149, 16)])
@pytest.mark.parametrize("width", [1216, 512])   # tokens that the table has room for: with the first sequences are divided where CTAs suffice
def test_chunks(T, heads, width):
    latent, rope, page, dtype = 128, 16, 64, BF16 if T % 100 else F16
    held = [width - 30, 200, 0, 70, width // 2]
    n = len(held) * (width // page) + 1
    cache = cache_of(latent, rope, n, page, dtype, T)
    table, lengths = table_of(held, page, n, heads, width=width // page)
    B = len(held)
    ql, qr = normal(1, dtype, B, T, heads, latent), normal(2, dtype, B, T, heads, rope)
    for causal, counts in ((True, None), (True, ints([T, T // 2, T, T, 0])), (False, ints([T, 1, 3, T - 1, T]))):
        y = check(cache, ql, qr, table, lengths, counts=counts, causal=causal)
        assert not y[2].any()


@pytest.mark.parametrize("width", [1088, 960])
def test_chunks_of_the_widest_vectors(width):
    latent, rope, page, T, heads = 512, 64, 32, 301, 128
    held = [width - 3, 310]
    n = 2 * (width // page) + 1
    cache = cache_of(latent, rope, n, page, BF16, 1)
    table, lengths = table_of(held, page, n, 2, width=width // page)
    check(cache, normal(1, BF16, 2, T, heads, latent), normal(2, BF16, 2, T, heads, rope), table, lengths, counts=ints([T, 299]))
