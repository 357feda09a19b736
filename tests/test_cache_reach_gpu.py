"""The key/value cache where addresses, tables and calls reach far: codes beyond 2^32 bytes, caches that the kernel for many rows does not
reach, missing pages under many rows, tables wider than their sequences, scratch that is too small, two streams at a time."""
import ctypes

import pytest
import torch

import fused_attention_b200 as fa
from fused_attention_b200 import _lib
from oracle import kv_cache as oracle
from test_cache_gpu import UNIT, check_attention, queries_of, random_cache, table_of

pytestmark = pytest.mark.gpu


def stretched(small, apart):
    """The cache's pages `apart` bytes from one another, in memory of their own (the gaps are never touched)."""
    n, G, page, H = small.k.shape
    parts = []
    for codes in (small.k, small.v):
        memory = torch.empty((n - 1) * apart + codes[0].numel(), dtype=torch.uint8, device="cuda")
        view = memory.as_strided((n, G, page, H), (apart, page * H, H, 1))
        view.copy_(codes.view(torch.uint8))
        parts.append(view.view(torch.float8_e4m3fn))
    return fa.KVCache(*parts, small.k_scale, small.v_scale, small.bounds)


@pytest.mark.parametrize("H,page,dtype", [(64, 16, torch.float16), (128, 32, torch.bfloat16), (32, 64, torch.float16), (16, 128, torch.bfloat16)])
def test_codes_beyond_32_bits_under_many_rows(H, page, dtype):
    """Pages of 6 GB in all: the last of them begin behind 2^32 bytes, and behind 2^31."""
    G, n = 2, 25
    small = random_cache(H, G, n, page, H)
    far = stretched(small, 1 << 28)
    table, lengths = table_of([n * page - 3], page, n, 5)
    for T, group in ((1, 3), (70, 2), (150, 1)):
        q = queries_of(1, min(T, n * page - 3), G * group * H, dtype, T)
        assert torch.equal(fa.cache_attention(far, q, table, lengths), check_attention(small, q, table, lengths))
    assert far.read_status() == (0, 0)


def raw_attention(cache, handle, q, table, lengths, bytes_short=0):
    """The C entry with a handle of one's own: (status, y)."""
    B, T, F = q.shape
    heads, need = F // cache.head_dim, ctypes.c_uint64()
    lib = _lib.load()
    assert lib.fa_b200_cache_attention_scratch(cache.head_dim, cache.kv_heads, heads, cache.page_size, B, T, table.shape[1], 0, 0, ctypes.byref(need)) == 0
    scratch, y = torch.empty(need.value, dtype=torch.uint8, device="cuda"), torch.empty_like(q)
    seqs = _lib.Sequences(table.data_ptr(), lengths.data_ptr(), None, table.stride(0), table.shape[1], B, T)
    rc = lib.fa_b200_cache_attention(ctypes.byref(handle), ctypes.byref(seqs), q.data_ptr(), q.stride(0), q.stride(1), heads,
                                     _lib.FP16 if q.dtype == torch.float16 else _lib.BF16, None, 0, 0, y.data_ptr(), scratch.data_ptr(), need.value - bytes_short, 0,
                                     torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return rc, y


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,page,T,group", [(64, 16, 100, 1), (128, 64, 40, 5), (16, 32, 300, 2)])
def test_many_rows_over_a_cache_of_more_than_64_gigabytes(H, page, T, group, dtype):
    """As its handle says: pages up to 2^31 - 1, of which the table names the few that there are.  The kernel for few rows takes the call."""
    G = 2
    cache = random_cache(H, G, 60, page, T)
    table, lengths = table_of([T + 500], page, 60, 1)
    q = queries_of(1, T, G * group * H, dtype, 1)
    handle = _lib.Cache.from_buffer_copy(cache._handle)
    handle.n_pages = 0x7FFFFFFF
    rc, y = raw_attention(cache, handle, q, table, lengths)
    want, bound = oracle.attention(cache, q, table, lengths, unit=UNIT[dtype])
    assert rc == 0 and cache.read_status() == (0, 0) and ((y.double() - want).abs() <= bound).all()
    rc, y = raw_attention(cache, cache._handle, q, table, lengths)
    assert rc == 0 and torch.equal(y, check_attention(cache, q, table, lengths))


@pytest.mark.parametrize("H,T,group,lengths", [(64, 1, 4, [300]), (128, 1, 4, [40000]), (64, 130, 1, [700]), (128, 300, 2, [5000, 300])])
def test_scratch_a_byte_short_is_refused(H, T, group, lengths):
    """Of what the form of the call needs: an undivided problem, a divided one, prompts, prompts in parts."""
    G, page = 2, 64
    n = len(lengths) * (max(lengths) // page + 1)
    cache = random_cache(H, G, n, page, 1)
    table, held = table_of(lengths, page, n, 1)
    q = queries_of(len(lengths), T, G * group * H, torch.float16, 1)
    assert raw_attention(cache, cache._handle, q, table, held)[0] == 0
    lib, need = _lib.load(), ctypes.c_uint64()
    # the size covers both kernels that may take the call: what is refused is less than the smaller of their needs
    assert lib.fa_b200_cache_attention_scratch(H, G, G * group, page, len(lengths), T, table.shape[1], 0, 0, ctypes.byref(need)) == 0
    assert raw_attention(cache, cache._handle, q, table, held, bytes_short=need.value - 15)[0] == _lib.ERR_TOO_LARGE
    if T * group < 64:
        assert raw_attention(cache, cache._handle, q, table, held, bytes_short=1)[0] == _lib.ERR_TOO_LARGE


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("H,T,group,dtype", [(64, 3, 2, torch.float16), (64, 80, 1, torch.bfloat16), (128, 70, 3, torch.float16), (16, 200, 2, torch.bfloat16)])
def test_missing_pages_are_left_out_and_reported(H, T, group, dtype, page):
    """Entries outside the cache in the middle of a sequence and at its ends, under any number of rows."""
    G, lens = 2, [T + 900, T + 260]
    n = 2 * (max(lens) // page + 1)
    cache = random_cache(H, G, n, page, T)
    table, lengths = table_of(lens, page, n, 4)
    W = table.shape[1]
    blocks = [-(-x // page) for x in lens]
    gone = [{0, blocks[0] // 2, blocks[0] - 1}, {1}]
    bad = table.clone()
    for b, which in enumerate(gone):
        for i, block in enumerate(sorted(which)):
            bad[b, block] = (n, -3, 2 ** 31 - 1)[i]
    q = queries_of(2, T, G * group * H, dtype, 1)
    y = fa.cache_attention(cache, q, bad, lengths)
    code, reports = cache.read_status()
    assert code == 1 and reports >= 4
    left = torch.full((2, W), -1, dtype=torch.int32, device="cuda")
    for b, which in enumerate(gone):
        kept = [i for i in range(blocks[b]) if i not in which]
        left[b, :len(kept)] = torch.tensor(kept, dtype=torch.int32, device="cuda")
    want, bound = oracle.attention(cache, q, table, lengths, pages=left[:, None, None].expand(2, T, G, W), unit=UNIT[dtype])
    assert not torch.isnan(y).any() and ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("T,group", [(1, 4), (90, 2)])
def test_lengths_out_of_range_are_cut_and_reported(T, group):
    H, G, page = 64, 2, 32
    cache = random_cache(H, G, 20, page, T)
    table, lengths = table_of([page * 8, page * 8, page * 8], page, 24, 4)
    table = table % 20
    q = queries_of(3, T, G * group * H, torch.float16, 1)
    want = check_attention(cache, q, table, lengths)
    y = fa.cache_attention(cache, q, table, torch.tensor([page * 8 + 1, -5, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    assert cache.read_status()[0] == 2
    assert torch.equal(y[0], want[0]) and not y[1].any() and torch.equal(y[2], want[2])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,group,lengths", [(1, 4, [300, 3000]), (6, 4, [700, 64]), (500, 4, [500]), (100, 1, [900, 100, 2000])])
def test_a_table_for_131072_tokens(T, group, lengths, dtype):
    """Calls are planned by the table's width: whatever the plan, the results are the same within their bound, the pages the same."""
    H, G, page = 64, 2, 16
    n = sum(-(-x // page) for x in lengths) + 2 * len(lengths) * (max(lengths) // page)
    cache = random_cache(H, G, n, page, T)
    narrow, held = table_of(lengths, page, n, 1)
    wide = torch.full((len(lengths), 131072 // page), -1, dtype=torch.int32, device="cuda")
    wide[:, :narrow.shape[1]] = narrow
    q = queries_of(len(lengths), T, G * group * H, dtype, 1)
    check_attention(cache, q, wide, held)
    pages = fa.cache_select(cache, q, wide, held, 9, last=2)
    assert torch.equal(pages, fa.cache_select(cache, q, narrow, held, 9, last=2))
    check_attention(cache, q, wide, held, pages=pages)


def test_two_streams_on_one_cache():
    """Calls of every form on two streams at a time, over pages that neither writes."""
    H, G, page = 64, 2, 32
    cache = random_cache(H, G, 200, page, 1)
    table, lengths = table_of([2000, 900], page, 200, 1)
    calls = [(queries_of(2, T, G * group * H, dtype, T), dtype) for T, group, dtype in ((1, 4, torch.float16), (5, 4, torch.bfloat16), (200, 2, torch.float16))]
    want = [(fa.cache_attention(cache, q, table, lengths), fa.cache_select(cache, q[:, -1:], table, lengths, 5)) for q, _ in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for s, mine in zip(streams, got):
            with torch.cuda.stream(s):
                for q, _ in calls if s is streams[0] else calls[::-1]:
                    mine.append((fa.cache_attention(cache, q, table, lengths), fa.cache_select(cache, q[:, -1:], table, lengths, 5)))
    torch.cuda.synchronize()
    for mine, order in zip(got, (want, want[::-1])):
        for i, (y, pages) in enumerate(mine):
            assert torch.equal(y, order[i % 3][0]) and torch.equal(pages, order[i % 3][1])
    assert cache.read_status() == (0, 0)
