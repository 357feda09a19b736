"""What sequences hold stays what it was through reserving, copying and appending, whoever shares pages with whom and however few pages are free.

Sequences whose tokens were taken back after a fork share a page of which they hold different numbers of tokens.  If all of them write to it, one
may keep it; the others get pages of their own or, where none is free, no token and stay on it.  So whoever keeps it must hold as many of
its tokens as any other.
"""
import random

import pytest
import torch

from oracle import pages as oracle


def state(rng, B, W, page, spare, most):
    """Sequences that go on as beginnings of others, with tokens taken back; counts; `spare` pages free."""
    table, lengths, n = [], [], 0
    for b in range(B):
        row = [-1] * W
        if b and rng.random() < 0.8:
            other = rng.randrange(b)
            held = lengths[other] - rng.choice((0, 0, 1, 3, rng.randint(0, page), rng.randint(0, lengths[other])))
            held = max(0, held)
            row = list(table[other])   # with the blocks behind `held`: it has not given them back yet
        else:
            held = rng.randint(0, (W - 1) * page)
            for i in range(-(-held // page)):
                row[i], n = n, n + 1
        table.append(row)
        lengths.append(held)
    n += spare
    names, order = rng.sample(range(n), n), rng.sample(range(B), B)
    table, lengths = [[names[p] if p >= 0 else -1 for p in table[b]] for b in order], [lengths[b] for b in order]
    counts = [rng.choice((0, 1, 1, 1, rng.randint(1, most))) for _ in range(B)]
    return table, lengths, counts, n


def held_by(table, lengths, page, contents):
    return [[contents[row[i // page]][i % page] for i in range(held)] for row, held in zip(table, lengths)]


def test_the_definition():
    """The lists that the kernels are held to (oracle/pages.py), with the contents of pages as lists too."""
    short = 0
    for seed in range(400):
        rng = random.Random(seed)
        page = 4
        table, lengths, counts, n = state(rng, rng.randint(2, 6), 4, page, rng.choice((0, 0, 1, 3)), 7)
        contents = [[(p, t) for t in range(page)] for p in range(n)]
        before = held_by(table, lengths, page, contents)
        new, granted, sources, targets = oracle.reserve(table, lengths, counts, n, page)
        for s, t in zip(sources, targets):
            if s >= 0:
                contents[t] = list(contents[s])
        for b, g in enumerate(granted):
            for i in range(lengths[b], lengths[b] + g):
                contents[new[b][i // page]][i % page] = ("new", b, i)
        after = held_by(new, [x + g for x, g in zip(lengths, granted)], page, contents)
        for b, (was, now) in enumerate(zip(before, after)):
            assert now[:len(was)] == was, (seed, b)
            assert now[len(was):] == [("new", b, i) for i in range(len(was), len(now))], (seed, b)
        short += any(g < min(c, 4 * page - x) for g, c, x in zip(granted, counts, lengths))
    assert short > 100


def test_who_keeps_a_page_by_hand():
    """The longest of those that hold it; of two as long, the first."""
    assert oracle.reserve([[0], [0]], [5, 8], [1, 1], 1, 16) == ([[0], [0]], [0, 1], [-1, -1], [-1, -1])
    assert oracle.reserve([[0], [0]], [5, 8], [1, 1], 2, 16) == ([[1], [0]], [1, 1], [0, -1], [1, -1])
    assert oracle.reserve([[0], [0]], [8, 5], [1, 1], 1, 16) == ([[0], [0]], [1, 0], [-1, -1], [-1, -1])
    assert oracle.reserve([[0], [0], [0]], [5, 8, 8], [1, 1, 1], 2, 16) == ([[1], [0], [0]], [1, 1, 0], [0, -1, -1], [1, -1, -1])
    # the second holds tokens of the page that the first has only got back to: 16 of the first's 20 new tokens have room
    assert oracle.reserve([[0, 1], [2, 1]], [0, 18], [20, 1], 3, 16) == ([[0, 1], [2, 1]], [16, 1], [-1, -1], [-1, -1])


# (sequences, blocks, page, free pages, most tokens): entries kept in registers, several blocks a thread, more sequences than threads, and tables
# that several CTAs go over
CASES = [(2, 3, 16, 0, 1), (12, 4, 16, 1, 20), (200, 5, 32, 20, 3), (40, 60, 16, 30, 900), (1500, 4, 16, 200, 1), (2100, 3, 16, 100, 2), (300, 150, 16, 60, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,W,page,spare,most", CASES)
def test_on_the_gpu(B, W, page, spare, most):
    import fused_attention_b200 as fa

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    refused = 0
    for trial in range(4):
        rng = random.Random(B * W + trial)
        table, lengths, counts, n = state(rng, B, W, page, spare, most)
        want, granted, sources, targets = oracle.reserve(table, lengths, counts, n, page)
        refused += granted != counts
        cache = fa.LatentCache(torch.randn(n, page, 144, device="cuda").half(), 128)
        pool, t, held = fa.PagePool(ints(oracle.counted(table, n))), ints(table), ints(lengths)
        positions = torch.arange(W * page, device="cuda")

        def rows():
            return cache.data[t.long().clamp(min=0)].flatten(1, 2)
        mine = positions < held[:, None]
        before = rows()
        got = fa.pages_reserve(pool, t, held, ints(counts), page)
        assert [x.tolist() for x in got] == [granted, sources, targets]
        assert t.tolist() == want and pool.refs.tolist() == oracle.counted(want, n)
        fa.cache_copy(cache, got[1], got[2])
        T = max(max(counts), 1)
        c, r = torch.randn(B, T, 128, device="cuda").half(), torch.randn(B, T, 16, device="cuda").half()
        fa.latent_append(cache, c, r, t, held, counts=got[0])
        after = rows()
        assert torch.equal(after[mine], before[mine])
        at = positions - held[:, None]
        new = (at >= 0) & (at < got[0][:, None])
        assert torch.equal(after[new], torch.cat((c, r), -1)[new.nonzero()[:, 0], at[new]])
        assert cache.read_status() == (0, 0) and pool.read_status()[0] in (0, 2, 3)
    assert refused
