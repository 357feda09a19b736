"""A pool and the one that compacting makes of it report in the same place; calls on the two, with tables of their own, have nothing else in common: they
may run side by side."""
import random

import pytest
import torch

import fused_attention_b200 as fa
from oracle import pages as oracle
from test_pages_gpu import ints, pool_of, state

pytestmark = pytest.mark.gpu
B, W, PAGE, N = 400, 120, 16, 60000   # a table that several CTAs go over


def problem(seed):
    rng = random.Random(seed)
    table, lengths = state(rng, B, W, PAGE, N - 2 * B, shared=0.3)
    counts = [rng.choice((0, 1, rng.randint(0, 40))) for _ in range(B)]
    lengths = [rng.randint(0, x) if rng.random() < 0.3 else x for x in lengths]
    counts = [min(c, W * PAGE - x) for c, x in zip(counts, lengths)]
    return table, lengths, counts


def test_whatever_the_rest_of_the_status_holds():
    """Only the first code and the number of reports are anyone's: what else is in the block decides nothing."""
    table, lengths, counts = problem(1)
    want, *result = oracle.reserve(table, lengths, counts, N, PAGE)
    for left in (0, 1, 5, -1):
        pool, t = pool_of(table, N), ints(table)
        pool._status[2:] = left
        got = fa.pages_reserve(pool, t, ints(lengths), ints(counts), PAGE)
        assert [x.tolist() for x in got] == result and t.tolist() == want and pool.refs.tolist() == oracle.counted(want, N)
        assert pool.read_status() == (0, 0) and (pool._status[2:] == left).all()


def test_old_and_new_pool_on_two_streams():
    table, lengths, counts = problem(2)
    old_want, *old_result = oracle.reserve(table, lengths, counts, N, PAGE)
    new_table, *_ = oracle.compact(table, oracle.counted(table, N))
    new_want, *new_result = oracle.reserve(new_table, lengths, counts, N, PAGE)
    streams = [torch.cuda.Stream() for _ in range(2)]
    held, more = ints(lengths), ints(counts)
    runs = []
    for _ in range(12):
        old, t = pool_of(table, N), ints(table)
        new, u, _, _ = fa.pages_compact(old, t)
        runs.append(((old, t), (new, u)))
    torch.cuda.synchronize()
    got = []
    for run in runs:
        for stream, (pool, at) in zip(streams, run):
            with torch.cuda.stream(stream):
                got.append(fa.pages_reserve(pool, at, held, more, PAGE))
    torch.cuda.synchronize()
    for i, ((old, t), (new, u)) in enumerate(runs):
        for (pool, at), g, want, result in (((old, t), got[2 * i], old_want, old_result), ((new, u), got[2 * i + 1], new_want, new_result)):
            assert [x.tolist() for x in g] == result
            assert at.tolist() == want and pool.refs.tolist() == oracle.counted(want, N)
        assert old.read_status() == (0, 0) and new._status.data_ptr() == old._status.data_ptr()
