"""The paged 8-bit key/value cache against the same in 64 bits (oracle/kv_cache.py).

Attention: every value within the bound that the oracle derives from the roundings (weights to fp16, scores and sums in fp32,
the result once to its type).  Selection: equal.  Appending: scales equal; a value no further from its code than half the
code's grain and the fp32 error of the rotation, two roundings of each product and one of the sum: 2^-22 of the products' magnitudes.
"""
import math

import pytest
import torch

import fused_attention_b200 as fa
from oracle import kv_cache as oracle

pytestmark = pytest.mark.gpu
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen_of(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def random_cache(H, G, n_pages, page, seed, spread=3):
    """A cache of random codes and bounds that are theirs; what no token reaches of it is random too."""
    g = gen_of(seed)
    cache = fa.cache_create(H, G, n_pages, page)
    for t in (cache.k, cache.v):
        t.copy_((torch.randn(t.shape, generator=g, device="cuda") * 80).clamp_(-448, 448))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.exp2(torch.randint(-8, -8 + spread, t.shape, generator=g, device="cuda").float()))
    k = cache.k.float()
    cache.bounds.copy_(torch.stack((k.amin(2), k.amax(2)), dim=2))
    return cache


def table_of(lengths, page, n_pages, seed, width=None):
    """Pages in no order, -1 behind what a sequence reaches."""
    lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    B, W = len(lengths), width or max(1, -(-int(lengths.max()) // page))
    order = torch.randperm(n_pages, generator=gen_of(seed), device="cuda")[:B * W].to(torch.int32).view(B, W)
    return torch.where(torch.arange(W, device="cuda") * page < lengths[:, None], order, -1), lengths


def queries_of(B, T, F, dtype, seed, sigma=1.0):
    return (torch.randn(B, T, F, generator=gen_of(seed), device="cuda") * sigma).to(dtype)


def check_attention(cache, q, table, lengths, **kw):
    y = fa.cache_attention(cache, q, table, lengths, **kw)
    want, bound = oracle.attention(cache, q, table, lengths, unit=UNIT[q.dtype], **kw)
    off = (y.double() - want).abs() - bound
    assert not torch.isnan(y).any() and float(off.max()) <= 0, (float(off.max()), float((y.double() - want).abs().max()))
    assert y.dtype == q.dtype and cache.read_status() == (0, 0)
    assert torch.equal(y, fa.cache_attention(cache, q, table, lengths, **kw))   # the same bits again
    return y


# ----------------------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H", [16, 32, 64, 128])
@pytest.mark.parametrize("G,group,page,lengths", [
    (1, 1, 16, [1]), (2, 4, 64, [1, 15, 16, 17]), (3, 5, 32, [31, 32, 33, 300]), (8, 4, 64, [127, 128, 129, 1000]),
    (1, 8, 128, [5000]), (2, 16, 16, [700, 2, 0]), (1, 20, 32, [300, 65]), (1, 40, 64, [257]), (4, 7, 128, [2049, 1, 640, 64, 4097])])
def test_single_tokens(H, dtype, G, group, page, lengths):
    n = sum(-(-x // page) for x in lengths) + len(lengths) * (max(lengths) // page + 2)
    cache = random_cache(H, G, n, page, H + page)
    table, lengths = table_of(lengths, page, n, H)
    check_attention(cache, queries_of(len(lengths), 1, G * group * H, dtype, 5), table, lengths)


@pytest.mark.parametrize("H,dtype", [(16, torch.float16), (32, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("G,group,page,T,lengths,counts", [
    (2, 4, 16, 2, [2, 3, 50], None), (2, 5, 16, 5, [333, 5, 129], None), (1, 8, 64, 9, [1000, 400], [9, 1]), (2, 1, 32, 33, [33, 100, 64], [33, 0, 17]),
    (1, 3, 128, 130, [130, 2000], [130, 77]), (2, 2, 64, 300, [300, 513], None), (1, 1, 64, 257, [800], None)])
def test_several_tokens(H, dtype, G, group, page, T, lengths, counts):
    n = 2 * sum(-(-x // page) for x in lengths) + 40 * len(lengths)
    cache = random_cache(H, G, n, page, T + H)
    table, lengths = table_of(lengths, page, n, T)
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    q = queries_of(len(lengths), T, G * group * H, dtype, T)
    for causal in (True, False):
        y = check_attention(cache, q, table, lengths, counts=counts, causal=causal)
        if counts is not None:
            for b, c in enumerate(counts.tolist()):
                assert not y[b, c:].any()


@pytest.mark.parametrize("H,G,group,page,T,keep,dtype", [(128, 2, 4, 64, 1, 5, torch.float16), (64, 1, 8, 16, 3, 9, torch.bfloat16), (32, 2, 1, 128, 2, 1, torch.float16),
                                                         (16, 1, 40, 32, 2, 30, torch.bfloat16), (128, 1, 20, 16, 1, 70, torch.float16), (128, 4, 2, 32, 70, 6, torch.bfloat16)])
def test_selected_pages(H, G, group, page, T, keep, dtype):
    lengths = [T, T + 3, 40 * page + 5, 7 * page]
    n = 4 * 42 + 5
    cache = random_cache(H, G, n, page, keep)
    table, lengths = table_of(lengths, page, n, keep)
    q = queries_of(4, T, G * group * H, dtype, 9)
    pages = fa.cache_select(cache, q, table, lengths, keep, last=2)
    check_attention(cache, q, table, lengths, pages=pages)
    # any order and gaps; pages behind the query's own (nothing of them is seen); none at all
    mixed = pages.flip(-1).contiguous()
    mixed[:, :, 0, ::3] = -1
    check_attention(cache, q, table, lengths, pages=mixed)
    behind = torch.full_like(pages, table.shape[1] - 1)
    behind[..., 1:] = -1
    check_attention(cache, q, table, lengths, pages=behind)
    assert not fa.cache_attention(cache, q, table, lengths, pages=torch.full_like(pages, -1)).any()


@pytest.mark.parametrize("T", [1, 3, 150])
def test_scales_that_differ_by_much(T):
    """Value scales 2^40 apart in one row, zero among them, and scales that are no powers of two."""
    H, G, page = 64, 2, 16
    cache = random_cache(H, G, 80, page, T)
    g = gen_of(3)
    cache.v_scale.copy_(torch.exp2(torch.randint(-20, 21, cache.v_scale.shape, generator=g, device="cuda").float()))
    cache.k_scale.copy_(torch.rand(cache.k_scale.shape, generator=g, device="cuda") * 0.02 + 1e-4)
    table, lengths = table_of([page * 30 + 7, T], page, 80, 1)
    q = queries_of(2, T, G * 2 * H, torch.bfloat16, T)
    check_attention(cache, q, table, lengths)
    cache.v_scale.copy_(torch.rand(cache.v_scale.shape, generator=g, device="cuda") + 0.3)
    cache.v_scale[table[0, 3].long()] = 0.0
    check_attention(cache, q, table, lengths)


@pytest.mark.parametrize("T", [1, 200])
def test_large_and_small_queries(T):
    """bf16 queries beyond fp16's range, and tiny ones; scores that single out one key."""
    H, G, page = 128, 1, 32
    cache = random_cache(H, G, 30, page, 8)
    table, lengths = table_of([700], page, 30, 1)
    q = queries_of(1, T, 3 * H, torch.bfloat16, 2)
    q[..., :H] *= 1e30
    q[..., H:2 * H] *= 1e-30
    cache.k_scale.mul_(2.0 ** -8)
    y = fa.cache_attention(cache, q, table, lengths)
    k, ks = oracle.values_of(cache.k, cache.k_scale, table[0].long(), 0)
    v, vs = oracle.values_of(cache.v, cache.v_scale, table[0].long(), 0)
    at = 700 - T + torch.arange(T, device="cuda")
    s = q[0, :, :H].double() @ (k * ks[:, None]).T
    s = torch.where(torch.arange(len(k), device="cuda") <= at[:, None], s, -math.inf)
    winner = s.argmax(-1)                                               # differences of scores are beyond any exponent
    torch.testing.assert_close(y[0, :, :H].double(), (v * vs[:, None])[winner], rtol=2.0 ** -8, atol=0)
    mean = torch.stack([(v * vs[:, None])[:i + 1].mean(0) for i in at.tolist()])       # all weights are the same
    torch.testing.assert_close(y[0, :, H:2 * H].double(), mean, rtol=2.0 ** -8, atol=2e-4)


def test_nothing_of_what_no_query_sees_is_used():
    """Codes behind a sequence's length are NaN, scales of later pages too; table entries behind it are anything."""
    H, G, page = 128, 2, 64
    for T in (1, 4, 100):
        cache = random_cache(H, G, 12, page, T)
        table, lengths = table_of([page * 3 + 20, page * 2], page, 12, 4, width=5)
        q = queries_of(2, T, G * 4 * H, torch.float16, T)
        want = fa.cache_attention(cache, q, table, lengths)
        used = set(table[0, :4].tolist() + table[1, :2].tolist())
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[int(table[0, 3]), :, 20:] = 0x7F
        for p in range(12):
            if p not in used:
                for t in (cache.k, cache.v):
                    t.view(torch.uint8)[p] = 0x7F
                cache.k_scale[p], cache.v_scale[p] = math.nan, math.nan
        table[0, 4], table[1, 2:] = 123456789, torch.tensor([-7, 2 ** 31 - 1, 11], dtype=torch.int32, device="cuda")
        assert torch.equal(want, fa.cache_attention(cache, q, table, lengths)) and cache.read_status() == (0, 0)
        # a page whose scale is NaN, seen by the first sequence's last query alone: NaN for it, nothing for the others
        cache.v_scale[int(table[0, 3]), 1] = math.nan
        y = fa.cache_attention(cache, q, table, lengths)
        half = G * 4 * H // 2
        assert torch.equal(y[:, :, :half], want[:, :, :half]) and torch.equal(y[1], want[1])
        assert torch.isnan(y[0, -min(T, 20):, half:]).all()
        if T > 20:
            assert torch.equal(y[0, :-20], want[0, :-20])


def test_pages_and_lengths_out_of_range_are_left_out_and_reported():
    H, G, page = 64, 2, 16
    cache = random_cache(H, G, 20, page, 1)
    table, lengths = table_of([page * 4, page * 4], page, 20, 4)
    q = queries_of(2, 1, 4 * H, torch.float16, 1)
    bad = table.clone()
    bad[0, 1], bad[0, 2] = 20, -3
    y = fa.cache_attention(cache, q, bad, lengths)
    code, reports = cache.read_status()
    assert code == 1 and reports >= 2 and cache.read_status() == (0, 0)
    pages = torch.tensor([0, 3], dtype=torch.int32, device="cuda").expand(2, 1, G, 2).contiguous()
    want, bound = oracle.attention(cache, q[:1], table[:1], lengths[:1], pages=pages[:1])
    assert ((y[:1].double() - want).abs() <= bound).all()
    # a length beyond the table is cut to it, a negative one is none
    y = fa.cache_attention(cache, q, table, torch.tensor([page * 4 + 1, -5], dtype=torch.int32, device="cuda"))
    assert cache.read_status()[0] == 2 and not y[1].any() and not torch.isnan(y).any()
    pages[0, 0, 0, 1] = 4
    fa.cache_attention(cache, q, table, lengths, pages=pages)
    assert cache.read_status()[0] == 1


def test_strides_streams_and_graphs():
    """Queries that are slices of a wider tensor, pages that hold tokens before heads, keys and values interleaved; on a stream
    of its own; captured and replayed with other lengths."""
    H, G, page, n = 64, 2, 32, 40
    base = random_cache(H, G, n, page, 6)
    both = torch.empty(n, page, 2, G, H, dtype=torch.float8_e4m3fn, device="cuda")
    k, v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    k.copy_(base.k), v.copy_(base.v)
    cache = fa.KVCache(k, v, base.k_scale, base.v_scale, base.bounds)
    wide = queries_of(3, 4, 10 * H, torch.float16, 1)
    q = wide[:, 1:3, 2 * H:6 * H]
    whole = table_of([300, 33, 64], page, n, 4)[0]
    table, lengths = torch.cat((whole, whole), dim=1)[:, :whole.shape[1]], torch.tensor([300, 33, 64], dtype=torch.int32, device="cuda")
    want = fa.cache_attention(base, q.contiguous(), whole, lengths)
    assert torch.equal(want, fa.cache_attention(cache, q, table, lengths))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(want, fa.cache_attention(cache, q, table, lengths))
        chosen = fa.cache_select(cache, q, table, lengths, 3)
    side.synchronize()
    assert torch.equal(chosen, fa.cache_select(base, q.contiguous(), whole, lengths, 3))
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fa.cache_attention(cache, q, table, lengths, out=out)
    for lens in ([300, 33, 64], [2, 3, 4], [299, 30, 10]):
        lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, fa.cache_attention(base, q.contiguous(), whole, lengths))


def test_many_sequences_of_all_lengths():
    """More sequences than a CTA has threads; empty ones, and some of a single token, among them."""
    H, G, page, B = 32, 2, 32, 200
    lens = torch.randint(0, 900, (B,), generator=gen_of(7), device="cuda").tolist()
    lens[0], lens[1], lens[130], lens[199] = 0, 1, 0, 899
    cache = random_cache(H, G, B * 29 + 3, page, 2)
    table, lengths = table_of(lens, page, B * 29 + 3, 3)
    q = queries_of(B, 1, G * 3 * H, torch.float16, 4)
    y = check_attention(cache, q, table, lengths)
    assert not y[0].any() and not y[130].any()
    got = fa.cache_select(cache, q, table, lengths, 6)
    assert torch.equal(got.cpu(), oracle.select(cache, q, table, lengths, 6))
    check_attention(cache, q, table, lengths, pages=got)


@pytest.mark.parametrize("H,dtype,causal", [(64, torch.float16, True), (128, torch.bfloat16, False), (32, torch.bfloat16, True)])
def test_more_items_than_multiprocessors(H, dtype, causal):
    """192 items of 256 query rows, the last 44 of them cut by keys; sequences without a token for the call between them."""
    G, group, page, T = 8, 2, 64, 300
    lens, counts = [300, 700, 512, 301, 900, 640, 300, 333], torch.tensor([300, 300, 0, 1, 129, 300, 257, 300], dtype=torch.int32, device="cuda")
    cache = random_cache(H, G, 8 * 16, page, H)
    table, lengths = table_of(lens, page, 8 * 16, 5)
    q = queries_of(8, T, G * group * H, dtype, 6)
    check_attention(cache, q, table, lengths, causal=causal)
    y = check_attention(cache, q, table, lengths, counts=counts, causal=causal)
    assert not y[2].any() and not y[3, 1:].any()


def test_one_pair_of_query_tiles_and_a_row_more():
    """Rows that end on a tile's edge, one in front of it and one behind it, and a tile that has hardly any."""
    H, G, page = 64, 1, 16
    cache = random_cache(H, G, 80, page, 9)
    for T in (127, 128, 129, 255, 256, 257, 385):
        table, lengths = table_of([T, 600], page, 80, T)
        check_attention(cache, queries_of(2, T, H, torch.float16, T), table, lengths)


def test_offsets_beyond_32_bits():
    """A page whose codes lie more than 2^32 bytes from the first, and one more than 2^31 tokens... of strides, not of memory read."""
    H, G, page = 128, 1, 128
    n = (1 << 32) // (H * page) + 4
    cache = KV = fa.KVCache(*(torch.zeros(n, G, page, H, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)),
                            *(torch.ones(n, G, device="cuda") for _ in range(2)), torch.zeros(n, G, 2, H, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn))
    small = random_cache(H, G, 3, page, 4)
    ids = [n - 1, n - 2, n - 3]
    for i, p in enumerate(ids):
        for name in ("k", "v", "k_scale", "v_scale", "bounds"):
            (getattr(KV, name).view(torch.uint8) if "scale" not in name else getattr(KV, name))[p] = (
                getattr(small, name).view(torch.uint8) if "scale" not in name else getattr(small, name))[i]
    lengths = torch.tensor([3 * page - 5], dtype=torch.int32, device="cuda")
    q = queries_of(1, 2, 4 * H, torch.float16, 1)
    far, near = (torch.tensor([t], dtype=torch.int32, device="cuda") for t in (ids, [0, 1, 2]))
    assert torch.equal(fa.cache_attention(cache, q, far, lengths), fa.cache_attention(small, q, near, lengths))
    assert torch.equal(fa.cache_select(cache, q, far, lengths, 2), fa.cache_select(small, q, near, lengths, 2))
    more = queries_of(1, 3, H, torch.float16, 2)
    before = lengths - 2
    for c, table in ((cache, far), (small, near)):
        fa.cache_append(c, more, more, table, before)
    assert torch.equal(cache.k.view(torch.uint8)[n - 3], small.k.view(torch.uint8)[2])
    assert torch.equal(cache.v.view(torch.uint8)[n - 3], small.v.view(torch.uint8)[2])


# ----------------------------------------------------------------------------- selection

@pytest.mark.parametrize("H,G,group,page,T,lengths,keep,first,last,dtype", [
    (128, 2, 4, 64, 1, [1, 64, 65, 5000], 4, 1, 1, torch.float16), (64, 3, 5, 16, 4, [4, 200, 1000], 9, 0, 2, torch.bfloat16),
    (32, 1, 17, 32, 2, [2, 900], 5, 2, 1, torch.float16), (16, 2, 1, 128, 3, [1500], 3, 1, 1, torch.bfloat16),
    (128, 1, 40, 16, 1, [9000], 33, 1, 2, torch.bfloat16), (128, 1, 1, 16, 2, [40000], 64, 1, 3, torch.float16), (64, 1, 2, 16, 50, [50, 400], 7, 3, 9, torch.float16),
    (64, 1, 70, 16, 2, [900, 33], 5, 1, 1, torch.bfloat16), (128, 2, 3, 32, 40, [2000], 9, 1, 2, torch.bfloat16)])
def test_select(H, G, group, page, T, lengths, keep, first, last, dtype):
    n = sum(-(-x // page) for x in lengths) + len(lengths) * (max(lengths) // page + 1)
    cache = random_cache(H, G, n, page, keep)
    table, lengths = table_of(lengths, page, n, keep)
    q = queries_of(len(lengths), T, G * group * H, dtype, keep)
    got = fa.cache_select(cache, q, table, lengths, keep, first=first, last=last)
    assert torch.equal(got.cpu(), oracle.select(cache, q, table, lengths, keep, first=first, last=last))
    counts = torch.randint(0, T + 1, (len(lengths),), generator=gen_of(1), device="cuda", dtype=torch.int32)
    got = fa.cache_select(cache, q, table, lengths, keep, counts=counts, first=first, last=last)
    assert torch.equal(got.cpu(), oracle.select(cache, q, table, lengths, keep, counts=counts, first=first, last=last))
    assert cache.read_status() == (0, 0)


@pytest.mark.parametrize("W", [40, 600, 3000, 9000])
def test_select_ties_go_to_the_lower_page(W):
    """Pages with few different bounds, so that most scores are shared by many, zero queries among them."""
    H, G, page, keep = 16, 2, 16, 21
    cache = random_cache(H, G, W, page, W)
    pattern = torch.randint(0, 3, (W, 1, 1, 1), generator=gen_of(W), device="cuda")
    cache.bounds.copy_((pattern * 16 * torch.tensor([-1.0, 1.0], device="cuda").view(1, 1, 2, 1)).expand(W, G, 2, H))
    cache.k_scale.fill_(0.5)
    table = torch.arange(W, dtype=torch.int32, device="cuda")[None].contiguous()
    lengths = torch.tensor([W * page - 3], dtype=torch.int32, device="cuda")
    q = queries_of(1, 2, 4 * H, torch.float16, 1)
    q[0, 1] = 0
    got = fa.cache_select(cache, q, table, lengths, keep)
    assert torch.equal(got.cpu(), oracle.select(cache, q, table, lengths, keep))
    assert got[0, 1, 0, :-1].tolist() == list(range(keep - 1))


# ----------------------------------------------------------------------------- appending

def angles(positions, H):
    a = torch.arange(positions, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, H, 2, device="cuda") / H)
    return a.cos(), a.sin()


def check_append(cache, before, keys, values, table, held, counts, rotation, interleaved, queries, rotated):
    """`before`: codes (as bytes) and scales of the cache before the call, and the bounds."""
    B, T, F = keys.shape
    H, G, page = cache.head_dim, cache.kv_heads, cache.page_size
    untouched = {name: torch.ones(cache.n_pages, G, page if name in "kv" else 1, dtype=torch.bool, device="cuda") for name in ("k", "v", "ks", "vs")}
    for b in range(B):
        n = T if counts is None else int(counts[b])
        start = int(held[b])
        at = start + torch.arange(n, device="cuda")
        if queries is not None:
            want, size = oracle.rotate(queries[b, :n].double().view(n, queries.shape[2] // H, H), at, rotation, interleaved)
            got = rotated[b, :n].double().view(n, queries.shape[2] // H, H)
            unit = UNIT[queries.dtype]
            assert ((got - want).abs() <= unit * want.abs() + 2.0 ** -22 * size + 2.0 ** -25).all() and not rotated[b, n:].any()
        new_k, size = oracle.rotate(keys[b, :n].double().view(n, G, H), at, rotation, interleaved)
        new_v = values[b, :n].double().view(n, G, H)
        for block in range(start // page, -(-(start + n) // page) if n else start // page):
            p = int(table[b, block])
            kept = max(0, start - block * page)
            rows = slice(max(0, block * page - start), min(n, (block + 1) * page - start))
            end = kept + rows.stop - rows.start
            for codes, scales, was, name, new, slack in ((cache.k, cache.k_scale, before[0], "k", new_k, size), (cache.v, cache.v_scale, before[1], "v", new_v, 0 * size)):
                untouched[name][p, :, :end] = False
                untouched[name + "s"][p] = False
                for g in range(G):
                    x = new[rows, g]
                    # the kernel's largest magnitude is the fp32 one
                    most = x.float().abs().max().item()
                    scale = oracle.scale_of(most)
                    old_scale = float(was[1][p, g])
                    if kept:
                        scale = max(scale, old_scale)
                    near = abs(most / (448 * scale) - 1) < 1e-6 or abs(most / (224 * scale) - 1) < 1e-6   # (of a power of two)
                    got_scale = float(scales[p, g])
                    assert got_scale == scale or (near and got_scale in (2 * scale, scale / 2)), (got_scale, scale, most)
                    got = codes.view(torch.uint8)[p, g].view(torch.float8_e4m3fn).double()
                    if kept:
                        old = was[0][p, g].view(torch.float8_e4m3fn).double()[:kept]
                        assert torch.equal(got[:kept], oracle.codes_of(old * (old_scale / got_scale)))
                    x = x / got_scale
                    grain = torch.exp2(((torch.frexp(x).exponent - 1).clamp(min=-6) - 3).double())
                    assert ((got[kept:end] - x).abs() <= grain / 2 + 2.0 ** -22 * slack[rows, g] / got_scale).all()
                    if name == "k":
                        bounds = cache.bounds.view(torch.uint8)[p, g].view(torch.float8_e4m3fn).double()
                        low, high = got[kept:end].amin(0), got[kept:end].amax(0)
                        if kept:   # (tokens that the page held and that were taken back since may still be in them)
                            old = oracle.codes_of(before[2][p, g].view(torch.float8_e4m3fn).double() * (old_scale / got_scale))
                            low, high = torch.minimum(low, old[0]), torch.maximum(high, old[1])
                        assert torch.equal(bounds, torch.stack((low, high)))
    for name, now, was in (("k", cache.k.view(torch.uint8), before[0][0]), ("v", cache.v.view(torch.uint8), before[1][0])):
        assert torch.equal(now[untouched[name]], was[untouched[name]])
    for name, now, was in (("ks", cache.k_scale, before[0][1]), ("vs", cache.v_scale, before[1][1])):
        assert torch.equal(now[untouched[name][..., 0]], was[untouched[name][..., 0]])


def state_of(cache):
    return tuple((c.view(torch.uint8).clone(), s.clone()) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))) + (cache.bounds.view(torch.uint8).clone(),)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,page,T,held,counts", [
    (128, 2, 64, 1, [0, 1, 63, 64, 130], None), (64, 3, 16, 1, [0, 15, 16], None), (32, 1, 32, 3, [30, 31, 0], None), (16, 2, 16, 4, [13, 5], [4, 0]),
    (128, 1, 64, 65, [0, 63, 64], None), (64, 2, 128, 300, [100, 0], [300, 29]), (16, 1, 32, 70, [31], None), (32, 2, 16, 17, [1, 15, 16], [17, 1, 16])])
def test_append(H, G, page, T, held, counts, dtype, interleaved):
    n = 60 + 2 * len(held) * (T // page + 3)
    held_t = torch.tensor(held, dtype=torch.int32, device="cuda")
    table, _ = table_of([h + T for h in held], page, n, T)
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    cache = random_cache(H, G, n, page, T + page)
    # bounds of what a page holds: its first tokens
    for b, h in enumerate(held):
        if h % page:
            p = int(table[b, h // page])
            k = cache.k.float()[p, :, :h % page]
            cache.bounds[p] = torch.stack((k.amin(1), k.amax(1)), dim=1).to(torch.float8_e4m3fn)
    B = len(held)
    rotation = angles(max(held) + T, H)
    for sigma, rot, heads in ((1.0, rotation, 3), (0.01, None, 0), (30.0, rotation, 1)):   # scales that grow and that stay
        before = state_of(cache)
        keys, values = queries_of(B, T, G * H, dtype, 1, sigma), queries_of(B, T, G * H, dtype, 2, sigma)
        q = queries_of(B, T, heads * H, dtype, 3) if heads else None
        rotated = fa.cache_append(cache, keys, values, table, held_t, counts=counts, queries=q, rotation=rot, interleaved=interleaved)
        assert (rotated is None) == (q is None) and cache.read_status() == (0, 0)
        check_append(cache, before, keys, values, table, held_t, counts, rot, interleaved, q, rotated)


def test_append_token_by_token_is_append_at_once():
    """Powers of two as scales: but for codes that became subnormal on the way the pages end the same."""
    H, G, page, n = 64, 2, 16, 8
    one, many = fa.cache_create(H, G, n, page), fa.cache_create(H, G, n, page)
    keys, values = queries_of(2, 40, G * H, torch.float16, 1), queries_of(2, 40, G * H, torch.float16, 2)
    table = torch.randperm(n, device="cuda").to(torch.int32).view(2, 4)
    lengths = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    fa.cache_append(many, keys, values, table, lengths)
    at = lengths.clone()
    for t in range(40):
        fa.cache_append(one, keys[:, t:t + 1], values[:, t:t + 1], table, at)
        at += 1
    pages = [int(table[0, i]) for i in range(1, 2)] + [int(table[1, i]) for i in range(3)]
    for a, b, s, r in ((one.k, many.k, one.k_scale, many.k_scale), (one.v, many.v, one.v_scale, many.v_scale)):
        assert torch.equal(s[pages], r[pages])
        x, y = a.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float(), b.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()
        assert ((x - y).abs() <= 2.0 ** -9).all() and (x == y)[y.abs() >= 2.0 ** -5].all()


def test_append_zeros_tiny_values_and_values_that_are_not_finite():
    H, G, page = 32, 2, 16
    cache = fa.cache_create(H, G, 4, page)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    zero = torch.zeros(1, 4, G * H, dtype=torch.bfloat16, device="cuda")
    tiny = torch.full_like(zero, 2.0 ** -120)
    lengths = torch.tensor([0], dtype=torch.int32, device="cuda")
    fa.cache_append(cache, zero, tiny, table, lengths)
    assert (cache.k_scale[2] == 2.0 ** -100).all() and (cache.v_scale[2] == 2.0 ** -100).all()
    assert not cache.k.float()[2].any() and not cache.v.float()[2].any()
    lengths += 4
    values = queries_of(1, 4, G * H, torch.bfloat16, 1)
    keys = values.clone()
    keys[0, 2, H + 3] = math.inf
    fa.cache_append(cache, keys, values, table, lengths)
    assert torch.isnan(cache.k_scale[2, 1]) and not cache.k.float()[2, 1].any() and not cache.k.float()[2, 0, :4].any()
    assert torch.isfinite(cache.k_scale[2, 0]) and torch.isfinite(cache.v_scale[2]).all()
    keys[0, 2, H + 3] = math.nan
    lengths += 4
    fa.cache_append(cache, values, keys, table, lengths)
    assert torch.isnan(cache.k_scale[2, 1]) and torch.isnan(cache.v_scale[2, 1]) and torch.isfinite(cache.v_scale[2, 0])
    assert cache.read_status() == (0, 0)


def test_append_out_of_range_writes_nothing_and_is_reported():
    H, G, page = 64, 1, 16
    cache = random_cache(H, G, 4, page, 3)
    before = state_of(cache)
    keys = queries_of(1, 1, H, torch.float16, 1)
    rotation = angles(8, H)
    for table, held, rot, code in (([[4]], 0, None, 1), ([[-1]], 3, None, 1), ([[2]], 16, None, 2), ([[2]], -1, None, 2), ([[2]], 8, rotation, 2)):
        fa.cache_append(cache, keys, keys, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([held], dtype=torch.int32, device="cuda"), rotation=rot)
        assert cache.read_status()[0] == code
    now = state_of(cache)
    assert torch.equal(before[2], now[2])
    for (a, s), (c, r) in zip(before[:2], now[:2]):
        assert torch.equal(a, c) and torch.equal(s, r)


# ----------------------------------------------------------------------------- refusals

def test_refusals():
    H, G, page = 64, 2, 16
    cache = fa.cache_create(H, G, 8, page)
    table, lengths = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    q, kv = queries_of(2, 1, 4 * H, torch.float16, 1), queries_of(2, 1, G * H, torch.float16, 1)
    fa.cache_attention(cache, q, table, lengths)

    def refuses(what, f, *args, **kw):
        with pytest.raises(RuntimeError, match=what):
            f(*args, **kw)

    for f, extra in ((fa.cache_attention, ()), (fa.cache_select, (3,))):
        refuses("KVCache", f, None, q, table, lengths, *extra)
        refuses("float16 or bfloat16", f, cache, q.float(), table, lengths, *extra)
        refuses("device", f, cache, q.cpu(), table, lengths, *extra)
        refuses("3 dimensions", f, cache, q[0], table, lengths, *extra)
        refuses("whole heads", f, cache, q[..., :H], table, lengths, *extra)
        refuses("whole heads", f, cache, q[:, :0], table, lengths, *extra)
        refuses("16-byte", f, cache, queries_of(2, 1, 4 * H + 4, torch.float16, 1)[..., 4:], table, lengths, *extra)
        refuses("contiguous", f, cache, q.transpose(1, 2).contiguous().transpose(1, 2).expand(2, 3, 4 * H)[:, :, ::2], table, lengths, *extra)
        refuses("int32", f, cache, q, table.long(), lengths, *extra)
        refuses("first of them B", f, cache, q, table[:1], lengths, *extra)
        refuses("int32", f, cache, q, table, lengths.float(), *extra)
        refuses("device", f, cache, q, table, lengths.cpu(), *extra)
        refuses("first of them B", f, cache, q, table, lengths, *extra, counts=lengths[:1])
        refuses("no pages", f, cache, q, table[:, :0], lengths, *extra)
    refuses("keep", fa.cache_select, cache, q, table, lengths, 0)
    refuses("last", fa.cache_select, cache, q, table, lengths, 3, last=0)
    pages = torch.zeros(2, 1, G, 3, dtype=torch.int32, device="cuda")
    refuses("pages", fa.cache_attention, cache, q, table, lengths, pages=pages.long())
    refuses("pages", fa.cache_attention, cache, q, table, lengths, pages=pages[:, :, :1])
    refuses("pages", fa.cache_attention, cache, q, table, lengths, pages=pages[..., :2])
    refuses("out", fa.cache_attention, cache, q, table, lengths, out=q.bfloat16())
    refuses("kv_heads", fa.cache_append, cache, q, q, table, lengths)
    refuses("type of the others", fa.cache_append, cache, kv, kv.bfloat16(), table, lengths)
    refuses("shape", fa.cache_append, cache, kv, kv[:1], table, lengths)
    refuses("rotation", fa.cache_append, cache, kv, kv, table, lengths, rotation=angles(4, H)[0])
    refuses("head_dim / 2", fa.cache_append, cache, kv, kv, table, lengths, rotation=angles(4, 2 * H))
    refuses("float32", fa.cache_append, cache, kv, kv, table, lengths, rotation=tuple(t.half() for t in angles(4, H)))
    for bad in (dict(head_dim=48), dict(page_size=8), dict(n_pages=0), dict(kv_heads=0)):
        refuses("must be", fa.cache_create, **{**dict(head_dim=64, kv_heads=2, n_pages=8, page_size=16), **bad})
    parts = [cache.k, cache.v, cache.k_scale, cache.v_scale, cache.bounds]
    for i, bad, what in ((0, cache.k.view(torch.uint8), "k must be"), (1, cache.v[:4], "shape of k"), (2, cache.k_scale[:, :1], "scales"), (3, cache.v_scale.double(), "v_scale"),
                         (4, cache.bounds[:, :, :1], "bounds"), (0, cache.k.cpu(), "CUDA"), (2, cache.k_scale.t().contiguous().t(), "contiguous")):
        refuses(what, fa.KVCache, *parts[:i], bad, *parts[i + 1:])
    stacked = fa.KVCache(cache.k[:1].expand(8, G, page, H), cache.v, *parts[2:])
    refuses("on top of one another", fa.cache_append, stacked, kv, kv, table, lengths)


def test_native_calls_take_plain_calls_and_agree_with_ctypes(monkeypatch):
    """The extension module answers every plain call itself, with the bits of the call through ctypes; a slice, a graph or a
    keyword more do not change that."""
    import os

    from fused_attention_b200 import build, cache as module
    assert os.path.exists(build.ext_path()), "the extension module has not been built"
    H, G, page = 64, 2, 32
    a, b = random_cache(H, G, 20, page, 1), random_cache(H, G, 20, page, 1)
    table, lengths = table_of([70, 5], page, 20, 2, width=4)
    table[table < 0] = 19
    keys, q, counts = queries_of(2, 3, G * H, torch.bfloat16, 1), queries_of(2, 3, 6 * H, torch.bfloat16, 2), torch.tensor([3, 2], dtype=torch.int32, device="cuda")

    def everything(cache):
        out = [fa.cache_append(cache, keys, keys, table, lengths, counts=counts, queries=q, rotation=angles(80, H), interleaved=True), cache.k.view(torch.uint8).clone()]
        assert fa.cache_append(cache, keys, keys, table, lengths) is None
        pages = fa.cache_select(cache, q, table, lengths, 2, counts=counts, first=0, last=2)
        given = torch.empty_like(q)
        y = fa.cache_attention(cache, q, table, lengths, counts=counts, pages=pages, out=given)
        assert y.data_ptr() == given.data_ptr()
        return out + [pages, y, fa.cache_attention(cache, q[:, 1:], table, lengths, causal=False)]

    calls = module._calls()
    answers = []

    def noting(f):
        def call(*args):
            answers.append(f(*args))
            return answers[-1]
        return call

    monkeypatch.setattr(module, "_native", tuple(noting(f) for f in calls[:3]) + (calls[3],))
    got = everything(a)
    assert len(answers) == 5 and not [x for x in answers if x is None or x.__class__ is int]
    monkeypatch.setattr(module, "_native", (lambda *args: None,) * 3 + (calls[3],))
    for x, y in zip(got, everything(b)):
        assert torch.equal(x, y)


# ----------------------------------------------------------------------------- where one kernel takes over from another

@pytest.mark.parametrize("H,dtype", [(16, torch.bfloat16), (32, torch.float16), (64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("group,T", [(3, 21), (4, 16), (5, 13), (1, 127), (16, 4), (64, 1)])
def test_attention_with_about_64_rows(H, dtype, page, group, T):
    G, lens = 2, [T, 300, 1111, T + 1]
    n = sum(-(-x // page) for x in lens) + 4 * (1111 // page + 1)
    cache = random_cache(H, G, n, page, T)
    table, lengths = table_of(lens, page, n, T)
    counts = torch.tensor([T, 0, T - T // 2, 1], dtype=torch.int32, device="cuda")
    q = queries_of(4, T, G * group * H, dtype, T)
    check_attention(cache, q, table, lengths)
    check_attention(cache, q, table, lengths, counts=counts, causal=False)


@pytest.mark.parametrize("longest", [512, 513, 1024, 1025])
def test_attention_of_many_short_sequences(longest):
    H, G, page, B = 32, 3, 32, 150
    lens = torch.randint(0, longest, (B,), generator=gen_of(longest), device="cuda").tolist()
    lens[3], lens[4], lens[149] = longest, 0, longest - 1
    width = -(-longest // page)
    cache = random_cache(H, G, B * width, page, 2)
    table, lengths = table_of(lens, page, B * width, 3)
    check_attention(cache, queries_of(B, 1, G * 2 * H, torch.float16, 4), table, lengths)


@pytest.mark.parametrize("T,page,pairs", [(5, 64, False), (9, 16, True), (16, 128, False), (40, 32, True), (64, 16, False)])
def test_appending_many_sequences_is_appending_a_few_at_a_time(T, page, pairs):
    """Bit for bit, whichever form each call takes."""
    H, G, B = 64, 4, 200
    held = torch.randint(0, 3 * page, (B,), generator=gen_of(T), device="cuda", dtype=torch.int32)
    counts = torch.randint(0, T + 1, (B,), generator=gen_of(T + 1), device="cuda", dtype=torch.int32)
    width = -(-(3 * page + T) // page)
    one = random_cache(H, G, B * width, page, T)
    few = fa.cache_create(H, G, B * width, page)
    for a, b in ((one.k, few.k), (one.v, few.v), (one.bounds, few.bounds)):
        b.view(torch.uint8).copy_(a.view(torch.uint8))
    few.k_scale.copy_(one.k_scale), few.v_scale.copy_(one.v_scale)
    table = torch.randperm(B * width, generator=gen_of(1), device="cuda").to(torch.int32).view(B, width)
    keys, values, q = (queries_of(B, T, h * H, torch.bfloat16, h) for h in (G, G, 2 * G))
    values = values.flip(0).contiguous()
    args = dict(rotation=angles(3 * page + T, H), interleaved=pairs)
    rotated = fa.cache_append(one, keys, values, table, held, counts=counts, queries=q, **args)
    for b in range(0, B, 4):
        s = slice(b, b + 4)
        part = fa.cache_append(few, keys[s], values[s], table[s], held[s], counts=counts[s], queries=q[s], **args)
        assert torch.equal(part, rotated[s])
    for a, b in ((one.k, few.k), (one.v, few.v), (one.bounds, few.bounds)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(one.k_scale, few.k_scale) and torch.equal(one.v_scale, few.v_scale) and one.read_status() == few.read_status() == (0, 0)


@pytest.mark.parametrize("W", [70, 700, 2500, 8200])
@pytest.mark.parametrize("keep,first,last", [(1, 0, 1), (40, 1, 2), (64, 40, 40), (69, 0, 1)])
def test_select_of_scores_far_apart(W, keep, first, last):
    """Scores from 2^-60 to 2^60 of either sign, most of them close together: the counting has to go on in a narrow range."""
    H, G, page = 16, 2, 16
    cache = random_cache(H, G, W, page, W + keep)
    g = gen_of(W)
    cache.k_scale.copy_(torch.where(torch.rand(W, G, generator=g, device="cuda") < 0.05, torch.exp2(torch.randint(-60, 61, (W, G), generator=g, device="cuda").float()), 0.25))
    table = torch.randperm(W, generator=g, device="cuda").to(torch.int32)[None].contiguous()
    lengths = torch.tensor([W * page], dtype=torch.int32, device="cuda")
    q = queries_of(1, 2, 4 * H, torch.float16, 1)
    got = fa.cache_select(cache, q, table, lengths, keep, first=first, last=last)
    assert torch.equal(got.cpu(), oracle.select(cache, q, table, lengths, keep, first=first, last=last))
