"""Appending across the rotation's last position: the tokens in front of it are appended as if they were all, those behind it are not."""
import pytest
import torch

import fused_attention_b200 as fa
from test_cache_gpu import angles, queries_of, random_cache, state_of, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,page,T,positions,held", [
    (64, 16, 4, 8, [6, 0, 4, 8, 7]), (128, 64, 3, 65, [63, 64, 65, 62]), (16, 32, 2, 32, [31, 30, 40]),      # a warp a task
    (64, 16, 40, 50, [0, 10, 11, 30, 49, 50, 90]), (32, 128, 200, 256, [100, 56, 57, 255]), (128, 32, 9, 33, [30, 24, 25])])   # a CTA a task
def test_tokens_up_to_the_last_position_are_appended(H, page, T, positions, held, interleaved):
    G, B = 2, len(held)
    width = -(-(max(held) + T) // page)
    n = B * width
    held_t = torch.tensor(held, dtype=torch.int32, device="cuda")
    table, _ = table_of([h + T for h in held], page, n, T, width=width)
    rotation = angles(positions, H)
    keys, values, q = (queries_of(B, T, h * H, torch.float16, h) for h in (G, G, 3 * G))
    there = (positions - held_t).clamp(0, T)
    for counts in (None, torch.tensor([T - (b % 3 == 1) for b in range(B)], dtype=torch.int32, device="cuda")):
        one, other = random_cache(H, G, n, page, 1), random_cache(H, G, n, page, 1)
        fits = there if counts is None else torch.minimum(there, counts)
        got = fa.cache_append(one, keys, values, table, held_t, counts=counts, queries=q, rotation=rotation, interleaved=interleaved)
        assert one.read_status()[0] == 2
        want = fa.cache_append(other, keys, values, table, held_t, counts=fits.to(torch.int32), queries=q, rotation=rotation, interleaved=interleaved)
        assert other.read_status() == (0, 0)
        assert torch.equal(got, want)
        for a, b in zip(state_of(one)[:2], state_of(other)[:2]):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(state_of(one)[2], state_of(other)[2])
