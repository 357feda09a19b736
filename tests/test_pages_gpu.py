"""The pages of a cache against lists and loops (oracle/pages.py): all whole numbers, all equal."""
import random

import pytest
import torch

import fused_attention_b200 as fa
from oracle import pages as oracle

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def state(rng, B, W, page, n, shared=0.5):
    """A table in which sequences share beginnings, its lengths and counts; pages in no order."""
    order = list(range(n))
    rng.shuffle(order)
    table, lengths = [], []
    for b in range(B):
        held = rng.randint(0, (W - 1) * page)
        blocks = -(-held // page)
        row = [-1] * W
        k = 0
        if b and rng.random() < shared:
            other = rng.randrange(b)
            k = rng.randint(0, min(blocks, -(-lengths[other] // page)))
            if rng.random() < 0.5 and lengths[other]:   # the whole of the other, its last block in part
                held = lengths[other]
                blocks = k = -(-held // page)
            row[:k] = table[other][:k]
        if blocks - k > len(order):
            held, blocks = k * page, k
        for i in range(k, blocks):
            row[i] = order.pop()
        table.append(row)
        lengths.append(held)
    return table, lengths


def pool_of(table, n):
    return fa.PagePool(ints(oracle.counted(table, n)))


@pytest.mark.parametrize("B,W,page,n,T", [(1, 3, 16, 5, 1), (5, 6, 32, 40, 1), (33, 9, 16, 400, 1), (40, 20, 64, 900, 300), (300, 7, 128, 2500, 1), (7, 300, 16, 3000, 2000),
                                          (2100, 4, 16, 9000, 1), (600, 70, 16, 30000, 40), (300, 150, 16, 50000, 1)])
def test_reserve(B, W, page, n, T):
    """Any counts, shared blocks of every kind, blocks behind the need; tables one CTA goes over and larger ones."""
    rng = random.Random(B * W)
    for trial in range(3):
        table, lengths = state(rng, B, W, page, n - (B if trial else 0))
        counts = [rng.choice((0, 1, rng.randint(0, T))) if trial else T for _ in range(B)]
        if trial == 2:   # tokens taken back: blocks behind them are let go of
            lengths = [rng.randint(0, x) for x in lengths]
        want, granted, sources, targets = oracle.reserve(table, lengths, counts, n, page)
        pool, t, held = pool_of(table, n), ints(table), ints(lengths)
        got = fa.pages_reserve(pool, t, held, T if trial == 0 else ints(counts), page)
        assert [x.tolist() for x in got] == [granted, sources, targets]
        assert t.tolist() == want and pool.refs.tolist() == oracle.counted(want, n) and held.tolist() == lengths
        code, reports = pool.read_status()
        outside = any(x + c > W * page for x, c in zip(lengths, counts))
        short = any(g < min(c, W * page - x) for g, x, c in zip(granted, lengths, counts))
        assert (code == 0) == (not outside and not short) and (code in (0, 2, 3))


def test_reserve_without_pages_left():
    """Two sequences share a block that both are about to write to, and no page is free: the lowest keeps it, the other writes nothing."""
    page = 16
    for B in (2, 1030):
        table = [[0, -1], [0, -1]] + [[-1, -1]] * (B - 2)
        lengths, counts = [5, 5] + [0] * (B - 2), [3, 3] + [0] * (B - 2)
        pool, t = pool_of(table, 1), ints(table)
        granted, sources, targets = fa.pages_reserve(pool, t, ints(lengths), ints(counts), page)
        assert granted.tolist() == [3, 0] + [0] * (B - 2) and t.tolist() == table and pool.refs.tolist() == [2]
        assert pool.read_status() == (3, 1)
        # one page for what three want: in order of sequences and blocks
        table = [[0, -1], [0, -1]] + [[-1, -1]] * (B - 2)
        pool, t = fa.PagePool(ints([2, 0])), ints(table)
        granted, sources, targets = fa.pages_reserve(pool, t, ints(lengths), ints([20, 20] + [0] * (B - 2)), page)
        assert granted.tolist()[:2] == [20, 0] and t.tolist()[:2] == [[0, 1], [0, -1]] and pool.refs.tolist() == [2, 1]
        assert pool.read_status()[0] == 3


def test_reserve_reports():
    pool, t = fa.PagePool(ints([1, 1, 0, 0])), ints([[0, 9, -1], [1, -7, -1]])
    granted, sources, targets = fa.pages_reserve(pool, t, ints([16, 3]), ints([1, 100]), 16)
    # 45 of the 100 tokens have room in the table, 29 in pages: two are free, and the first sequence takes one
    assert granted.tolist() == [1, 29] and pool.read_status()[0] in (1, 2, 3)
    assert t.tolist()[0] == [0, 2, -1] and t.tolist()[1][:2] == [1, 3] and pool.read_status() == (0, 0)
    # counts that are not in step with the table
    pool, t = fa.PagePool(ints([0, 0])), ints([[0, 1]])
    fa.pages_reserve(pool, t, ints([3]), 0, 16)
    assert pool.read_status()[0] == 4


@pytest.mark.parametrize("B,W", [(1, 1), (8, 5), (100, 33), (3000, 3), (15000, 2)])
def test_fork(B, W):
    rng = random.Random(B)
    n = B * W + 3
    table, lengths = state(rng, B, W, 16, n)
    parents = [rng.choice((b, rng.randrange(B), -1)) for b in range(B)]
    want, held = oracle.fork(table, lengths, parents)
    pool, t, at = pool_of(table, n), ints(table), ints(lengths)
    fa.pages_fork(pool, t, at, ints(parents))
    assert t.tolist() == want and at.tolist() == held and pool.refs.tolist() == oracle.counted(want, n) and pool.read_status() == (0, 0)
    fa.pages_fork(pool, t, at, ints([-1] * B))   # all let go
    assert not pool.refs.any() and (t == -1).all() and not at.any()


def test_fork_reports_and_views():
    """A parent outside leaves a row as it is; an entry outside becomes -1; tables that are slices of wider ones."""
    wide = torch.full((3, 9), 77, dtype=torch.int32, device="cuda")
    t = wide[:, 2:6]
    t.copy_(ints([[0, 1, -1, -1], [2, 50, -1, -1], [-1, -1, -1, -1]]))
    pool, lengths = fa.PagePool(ints([1, 1, 1, 0])), ints([20, 20, 0])
    fa.pages_fork(pool, t, lengths, ints([5, 0, 1]))
    assert t.tolist() == [[0, 1, -1, -1], [0, 1, -1, -1], [2, -1, -1, -1]] and lengths.tolist() == [20, 20, 20]
    assert pool.refs.tolist() == [2, 2, 1, 0] and pool.read_status()[0] in (1, 2)
    assert (wide[:, :2] == 77).all() and (wide[:, 6:] == 77).all()


@pytest.mark.parametrize("B,W,n", [(1, 1, 1), (3, 5, 40), (20, 30, 4096), (20, 30, 4097), (50, 40, 20011)])
def test_compact(B, W, n):
    rng = random.Random(n)
    table, lengths = state(rng, B, W, 16, n)
    pool, t = pool_of(table, n), ints(table)
    before = pool.refs.tolist()
    want, refs, moved, holes = oracle.compact(table, before)
    new, renumbered, sources, targets = fa.pages_compact(pool, t)
    assert renumbered.tolist() == want and new.refs.tolist() == refs
    k = len(moved)
    assert sources.tolist() == moved + [-1] * (n - k) and targets.tolist() == holes + [-1] * (n - k)
    assert t.tolist() == table and pool.refs.tolist() == before and pool.read_status() == (0, 0)   # left as they are


def test_compact_reports_entries_that_are_not_counted():
    pool, t = fa.PagePool(ints([0, 0, 1, 0])), ints([[2, 3, 8]])
    new, renumbered, sources, targets = fa.pages_compact(pool, t)
    assert renumbered.tolist() == [[0, -1, -1]] and new.refs.tolist() == [1, 0, 0, 0] and pool.read_status()[0] in (1, 4)


def kv_cache(n, page=16, H=32, G=3, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    cache = fa.cache_create(H, G, n, page)
    for t in (cache.k, cache.v, cache.bounds):
        t.view(torch.uint8).copy_(torch.randint(0, 120, t.shape, generator=g, device="cuda"))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.rand(t.shape, generator=g, device="cuda"))
    return cache


def contents(cache):
    ts = (cache.k, cache.v, cache.bounds, cache.k_scale, cache.v_scale) if isinstance(cache, fa.KVCache) else (cache.data,)
    return [t.view(torch.uint8).clone() for t in ts]


def test_copy():
    """Both kinds of cache, one and several, strided ones, many pairs and few; what is not a target stays."""
    n = 50
    latent = fa.LatentCache(torch.randn(n, 32, 288, device="cuda").half(), 256)
    padded = fa.LatentCache(torch.randn(n, 33, 304, device="cuda").bfloat16()[:, :32, 8:296], 256)
    kv = kv_cache(n)
    whole = kv_cache(n, seed=2)
    swapped = fa.KVCache(whole.k.transpose(1, 2).contiguous().transpose(1, 2), whole.v, whole.k_scale, whole.v_scale, whole.bounds)   # tokens before heads
    for caches in (latent, padded, kv, swapped, [kv, swapped], [latent, padded, latent], [kv, latent], [kv] * 9):
        for k in (1, 7, 25):
            rng = random.Random(k)
            both = rng.sample(range(n), 2 * k)
            sources, targets = both[:k], both[k:]
            several = caches if isinstance(caches, list) else [caches]
            before = [contents(c) for c in several]
            gaps_s, gaps_t = [-1, *sources, -1, 3], [4, *targets, -1, -1]
            fa.cache_copy(caches, ints(gaps_s), ints(gaps_t))
            for c, old in zip(several, before):
                for now, was in zip(contents(c), old):
                    want = was.clone()
                    want[targets] = was[sources]
                    assert torch.equal(now, want)
                assert c.read_status() == (0, 0)


def test_copy_reports_and_refusals():
    a, b, other = kv_cache(6), fa.latent_cache_create(128, 16, 6, 16), fa.latent_cache_create(128, 16, 7, 16)
    before = contents(a) + contents(b)
    fa.cache_copy([a, b], ints([6, 1, -3]), ints([0, 1 << 20, 2]))
    assert a.read_status() == (1, 3) and all(torch.equal(x, y) for x, y in zip(before, contents(a) + contents(b)))
    for match, args in (("as many pages", ([a, other], ints([1]), ints([2]))), ("int32", (a, ints([1]).long(), ints([2]))), ("shape of sources", (a, ints([1]), ints([2, 3]))),
                        ("KVCache", ("cache", ints([1]), ints([2]))), ("contiguous", (a, ints([[1]]), ints([[2]])))):
        with pytest.raises(RuntimeError, match=match):
            fa.cache_copy(*args)
    one = torch.zeros(1, 3, 16, 32, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).expand(6, 3, 16, 32)
    with pytest.raises(RuntimeError, match="on top of one another"):
        fa.cache_copy(fa.KVCache(one, one, a.k_scale, a.v_scale, a.bounds), ints([1]), ints([2]))


def test_refusals():
    pool, t, lengths = fa.page_pool_create(8), torch.full((2, 3), -1, dtype=torch.int32, device="cuda"), ints([0, 0])
    for match, f in (("int32", lambda: fa.pages_fork(pool, t.long(), lengths, ints([0, 1]))), ("shape", lambda: fa.pages_fork(pool, t, lengths, ints([0]))),
                     ("shape", lambda: fa.pages_reserve(pool, t, ints([0]), 1, 16)), ("page_size", lambda: fa.pages_reserve(pool, t, lengths, 1, 48)),
                     ("counts", lambda: fa.pages_reserve(pool, t, lengths, -1, 16)), ("counts", lambda: fa.pages_reserve(pool, t, lengths, ints([1]), 16)),
                     ("on top of one another", lambda: fa.pages_fork(pool, t[:1].expand(2, 3), lengths, ints([0, 1]))), ("contiguous", lambda: fa.pages_compact(pool, t.t())),
                     ("int32", lambda: fa.pages_compact(pool, None)), ("contiguous", lambda: fa.PagePool(torch.zeros(8, dtype=torch.int32, device="cuda")[::2]))):
        with pytest.raises(RuntimeError, match=match):
            f()
    assert t.shape == (2, 3) and not pool.refs.any()


def test_captured_and_replayed():
    """Reserving, forking and copying in a graph: a decoder's step, replayed until the pages run out, against lists."""
    rng = random.Random(3)
    B, W, page, n = 6, 5, 16, 22
    cache = fa.LatentCache(torch.randn(n, page, 144, device="cuda").half(), 128)
    pool, t, lengths = fa.page_pool_create(n), torch.full((B, W), -1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    parents, counts = torch.arange(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    fa.pages_fork(pool, t, lengths, parents)
    granted, sources, targets = fa.pages_reserve(pool, t, lengths, counts, page)
    fa.cache_copy(cache, sources, targets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fa.pages_fork(pool, t, lengths, parents)
        granted, sources, targets = fa.pages_reserve(pool, t, lengths, counts, page)
        fa.cache_copy(cache, sources, targets)
        lengths += granted
    table, held = t.tolist(), lengths.tolist()
    for step in range(40):
        now_parents = [rng.choice((b, b, b, rng.randrange(B))) for b in range(B)]
        now_counts = [rng.randint(0, 9) for _ in range(B)]
        parents.copy_(ints(now_parents))
        counts.copy_(ints(now_counts))
        graph.replay()
        table, held = oracle.fork(table, held, now_parents)
        table, g, s, d = oracle.reserve(table, held, now_counts, n, page)
        held = [x + y for x, y in zip(held, g)]
        assert [granted.tolist(), sources.tolist(), targets.tolist()] == [g, s, d]
        assert t.tolist() == table and lengths.tolist() == held and pool.refs.tolist() == oracle.counted(table, n)
        for a, b in zip(s, d):
            assert a < 0 or torch.equal(cache.data[a], cache.data[b])
