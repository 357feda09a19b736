"""The cache of latent vectors against the same in 64 bits (oracle/latent.py): appending to it, the absorbed form of attention over it, the
expanded form for prompts.  Every value lies within the bound that the oracle derives from the roundings; what is copied is equal.

Appending: latent vectors equal; a rotary part off by its rounding (half of eps, relative) and by two fp32 roundings of each product and one of
the sum, 2^-22 of the products' magnitudes.
"""
import pytest
import torch

import fused_attention_b200 as fa
from oracle import latent as oracle

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def gen_of(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(seed, dtype, *shape):
    return torch.randn(shape, generator=gen_of(seed), device="cuda").to(dtype)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def table_of(lengths, page, n, seed, width=None):
    lengths = ints(lengths)
    W = width or max(1, -(-int(lengths.max()) // page))
    order = torch.randperm(n, generator=gen_of(seed), device="cuda")[:len(lengths) * W].to(torch.int32).view(len(lengths), W)
    return torch.where(torch.arange(W, device="cuda") * page < lengths[:, None], order, -1), lengths


def cache_of(latent, rope, n, page, dtype, seed):
    return fa.LatentCache(normal(seed, dtype, n, page, latent + rope), latent)


def within(y, want, bound):
    off = (y.double() - want).abs() - bound
    assert not torch.isnan(y).any() and float(off.max()) <= 0, (float(off.max()), float((y.double() - want).abs().max()), off.flatten().argmax().item())


def check(cache, ql, qr, table, lengths, scale=0.07, **kw):
    y = fa.latent_attention(cache, ql, qr, table, lengths, scale=scale, **kw)
    within(y, *oracle.attention(cache.data, cache.latent_dim, ql, qr, table, lengths, scale, **kw))
    assert y.dtype == ql.dtype and cache.read_status() == (0, 0)
    assert torch.equal(y, fa.latent_attention(cache, ql, qr, table, lengths, scale=scale, **kw))   # the same bits again
    return y


# ----------------------------------------------------------------------------- absorbed

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("latent,rope", [(128, 16), (256, 32), (512, 64)])
@pytest.mark.parametrize("heads,page,lengths", [
    (1, 16, [1]), (16, 64, [1, 63, 64, 65]), (5, 32, [31, 300, 0]), (17, 128, [127, 129, 1000]), (40, 16, [700, 2]), (64, 64, [257, 64]), (128, 64, [513, 90, 1]), (80, 32, [33])])
def test_single_tokens(latent, rope, dtype, heads, page, lengths):
    n = sum(-(-x // page) for x in lengths) + len(lengths) * (max(lengths) // page + 2)
    cache = cache_of(latent, rope, n, page, dtype, page)
    table, lengths = table_of(lengths, page, n, heads)
    B = len(lengths)
    check(cache, normal(1, dtype, B, 1, heads, latent), normal(2, dtype, B, 1, heads, rope), table, lengths)


@pytest.mark.parametrize("latent,rope,dtype", [(512, 64, BF16), (128, 32, F16)])
@pytest.mark.parametrize("heads,page,T,lengths,counts", [
    (16, 64, 4, [4, 5, 333], None), (5, 16, 7, [7, 100, 64], [7, 1, 0]), (1, 32, 130, [130, 200], [130, 77]), (3, 128, 33, [40, 33], None), (20, 64, 9, [3, 70], [9, 9])])
def test_several_tokens(latent, rope, dtype, heads, page, T, lengths, counts):
    """Drafted tokens and chunks; counts, and queries in front of the first key (the last case)."""
    n = 60
    cache = cache_of(latent, rope, n, page, dtype, T)
    table, lengths = table_of(lengths, page, n, T, width=15)
    counts = None if counts is None else ints(counts)
    B = len(lengths)
    ql, qr = normal(3, dtype, B, T, heads, latent), normal(4, dtype, B, T, heads, rope)
    for causal in (True, False):
        y = check(cache, ql, qr, table, lengths, counts=counts, causal=causal)
        for b, c in enumerate(counts.tolist() if counts is not None else []):
            assert not y[b, c:].any()


@pytest.mark.parametrize("B,heads,high", [(1, 16, 20000), (3, 128, 9000), (200, 16, 90), (40, 33, 700), (500, 8, 40)])
def test_long_and_many(B, heads, high):
    """Sequences that many CTAs share, and CTAs that share many sequences, empty ones among them."""
    page, latent, rope, dtype = 64, 256, 64, BF16
    lengths = torch.randint(0, high + 1, (B,), generator=gen_of(B), device="cuda").tolist()
    lengths[0] = high
    n = B * (high // page + 1) + 1
    cache = cache_of(latent, rope, n, page, dtype, 1)
    table, lengths = table_of(lengths, page, n, 2)
    y = check(cache, normal(1, dtype, B, 1, heads, latent), normal(2, dtype, B, 1, heads, rope), table, lengths)
    assert not y[lengths == 0].any()


def test_scores_far_apart_and_references_that_move():
    """Keys that grow along the sequence: every tile's scores exceed the last one's by far; and queries of zeros."""
    latent, rope, page, dtype = 512, 64, 64, F16
    cache = cache_of(latent, rope, 20, page, dtype, 1)
    cache.data.mul_(torch.linspace(0.05, 3, 20 * page, device="cuda").view(20, page, 1).to(dtype))
    table = torch.arange(20, dtype=torch.int32, device="cuda").view(1, 20)
    ql, qr = normal(1, dtype, 1, 1, 16, latent), normal(2, dtype, 1, 1, 16, rope)
    ql[:, :, 3], qr[:, :, 3] = 0, 0
    check(cache, ql, qr, table, ints([20 * page - 3]), scale=0.5)
    check(cache, ql * 4, qr * 4, table, ints([20 * page - 3]), scale=0.5)


def test_what_is_not_seen_does_not_reach_a_query():
    """NaN and infinities behind the end of a sequence, in tokens of the call that earlier queries do not see, in other pages."""
    latent, rope, page, T, heads = 256, 64, 32, 3, 8
    clean = cache_of(latent, rope, 12, page, BF16, 1)
    table, lengths = table_of([70, 65], page, 12, 1)
    ql, qr = normal(1, BF16, 2, T, heads, latent), normal(2, BF16, 2, T, heads, rope)
    want = fa.latent_attention(clean, ql, qr, table, lengths, scale=0.1)
    for what in (float("nan"), float("inf"), -float("inf")):
        data = clean.data.clone()
        for b in range(2):
            held = int(lengths[b])
            data[table[b, held // page].long(), held % page:] = what                      # behind the end
            last = held - 1
            data[table[b, last // page].long(), last % page, 7] = what                    # one value of the last token
        cache = fa.LatentCache(data, latent)
        y = fa.latent_attention(cache, ql, qr, table, lengths, scale=0.1)
        assert torch.equal(y[:, :T - 1], want[:, :T - 1])
        assert not torch.isfinite(y[:, T - 1]).all(-1).any()
        ql2 = ql.clone()
        ql2[0, 1] = what   # a query that is not finite is its own affair
        y = fa.latent_attention(clean, ql2, qr, table, lengths, scale=0.1)
        keep = torch.ones(2, T, dtype=torch.bool, device="cuda")
        keep[0, 1] = False
        assert torch.equal(y[keep], want[keep]) and not torch.isfinite(y[0, 1]).any()


def test_pages_that_are_not_there():
    latent, rope, page = 128, 32, 16
    cache = cache_of(latent, rope, 10, page, F16, 1)
    table, lengths = table_of([150], page, 10, 1)
    broken = table.clone()
    broken[0, 3], broken[0, 5] = -1, 10
    ql, qr = normal(1, F16, 1, 1, 4, latent), normal(2, F16, 1, 1, 4, rope)
    y = fa.latent_attention(cache, ql, qr, broken, lengths, scale=0.1)
    code, reports = cache.read_status()
    assert code == 1 and reports >= 1
    # as if their tokens were not there
    rows = cache.data[table[0].long()].flatten(0, 1)
    keep = torch.ones(160, dtype=torch.bool, device="cuda")
    keep[48:64] = keep[80:96] = keep[150:] = False
    rows = rows[keep].double()
    for h in range(4):
        q = torch.cat((ql[0, :, h], qr[0, :, h]), -1).double()
        within(y[0, :, h], *oracle.attend(q, rows, rows[:, :latent], torch.tensor([len(rows)], device="cuda"), 0.1, 2.0 ** -11, True))
    y = fa.latent_attention(cache, ql, qr, table, ints([-5]), scale=0.1)
    assert not y.any() and cache.read_status()[0] == 2
    y = fa.latent_attention(cache, ql, qr, table, ints([1000]), scale=0.1)   # cut to what the table has room for
    assert cache.read_status()[0] == 2
    assert torch.equal(y, fa.latent_attention(cache, ql, qr, table, ints([160]), scale=0.1))


def test_strides_and_layouts():
    """Heads before tokens, slices of a projection, padded pages and tokens, an output that is given."""
    latent, rope, page, B, T, heads = 256, 32, 32, 2, 3, 6
    wide = normal(1, BF16, 9, 2, page + 1, latent + rope + 24)
    cache = fa.LatentCache(wide[:, 1, :page, 8:8 + latent + rope], latent)
    plain = fa.LatentCache(cache.data.contiguous(), latent)
    table, lengths = table_of([90, 50], page, 9, 1)
    both = normal(2, BF16, B, heads, T, latent + rope).transpose(1, 2)
    ql, qr = both[..., :latent], both[..., latent:]
    want = fa.latent_attention(plain, ql.contiguous(), qr.contiguous(), table, lengths, scale=0.1)
    out = torch.empty_like(want)
    assert fa.latent_attention(cache, ql, qr, table, lengths, scale=0.1, out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, want)
    wide_table = torch.full((B, 9), -1, dtype=torch.int32, device="cuda")
    wide_table[:, 2:2 + table.shape[1]] = table
    assert torch.equal(want, fa.latent_attention(cache, ql, qr, wide_table[:, 2:2 + table.shape[1]], lengths, scale=0.1))


def test_offsets_beyond_32_bits():
    """A page that begins more than 2^32 bytes into the cache."""
    latent, rope, page = 512, 64, 128
    n = (1 << 32) // (page * 1152) + 40
    cache = fa.LatentCache(torch.empty(n, page, latent + rope, dtype=BF16, device="cuda"), latent)
    ids = [n - 1, 3, n - 20, n - 2]
    for p in ids:
        cache.data[p] = normal(p % 1000, BF16, page, latent + rope)
    table = ints([ids[:2], ids[2:]])
    check(cache, normal(1, BF16, 2, 1, 16, latent), normal(2, BF16, 2, 1, 16, rope), table, ints([250, 130]))
    keys, _ = fa.latent_append(cache, normal(3, BF16, 2, 1, latent), normal(4, BF16, 2, 1, rope), table, ints([5, 129]))
    assert torch.equal(cache.data[ids[0], 5, latent:], keys[0, 0]) and torch.equal(cache.data[ids[3], 1, latent:], keys[1, 0])


def test_captured_and_replayed_with_other_lengths():
    latent, rope, page, heads = 256, 64, 64, 16
    cache = cache_of(latent, rope, 30, page, BF16, 1)
    table = torch.randperm(30, generator=gen_of(1), device="cuda").to(torch.int32).view(3, 10)
    lengths, ql, qr = ints([5, 100, 300]), normal(1, BF16, 3, 1, heads, latent), normal(2, BF16, 3, 1, heads, rope)
    out = torch.empty_like(ql)
    fa.latent_attention(cache, ql, qr, table, lengths, scale=0.1)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fa.latent_attention(cache, ql, qr, table, lengths, scale=0.1, out=out)
    other = torch.empty_like(ql)
    with torch.cuda.graph(second, pool=graph.pool()):   # two graphs that share a pool
        fa.latent_attention(cache, ql, qr, table, lengths, scale=0.1, out=other)
    for new in ([640, 1, 0], [64, 65, 639]):
        lengths.copy_(ints(new))
        graph.replay()
        second.replay()
        want = fa.latent_attention(cache, ql, qr, table, lengths, scale=0.1)
        assert torch.equal(out, want) and torch.equal(other, want)


def test_two_streams_at_once():
    latent, rope, page, heads = 512, 64, 64, 32
    cache = cache_of(latent, rope, 200, page, BF16, 1)
    table = torch.randperm(200, generator=gen_of(1), device="cuda").to(torch.int32).view(4, 50)
    lengths = ints([3200, 10, 2000, 777])
    qs = [(normal(i, BF16, 4, 1, heads, latent), normal(i + 9, BF16, 4, 1, heads, rope)) for i in range(2)]
    want = [fa.latent_attention(cache, ql, qr, table, lengths, scale=0.1) for ql, qr in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fa.latent_attention(cache, *qs[i], table, lengths, scale=0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(want[i], y) for y in got[i])


def test_attention_refusals():
    cache = cache_of(256, 32, 4, 32, BF16, 1)
    table, lengths = table_of([90], 32, 4, 1)
    ql, qr = normal(1, BF16, 1, 1, 4, 256), normal(2, BF16, 1, 1, 4, 32)

    def refused(match, *a, **kw):
        args = dict(q_latent=ql, q_rope=qr, table=table, lengths=lengths, scale=0.1)
        args.update(kw)
        with pytest.raises(RuntimeError, match=match):
            fa.latent_attention(cache, args.pop("q_latent"), args.pop("q_rope"), args.pop("table"), args.pop("lengths"), **args)
    refused("float16", q_latent=ql.float())
    refused("type of the others", q_latent=ql.half(), q_rope=qr.half())
    refused("shape", q_latent=ql[..., :128].contiguous())
    refused("shape", q_rope=qr[:, :, :3])
    refused("16-byte", q_latent=normal(1, BF16, 1, 1, 4, 260)[..., 4:])
    refused("contiguous", q_latent=normal(1, BF16, 1, 1, 4, 512)[..., ::2])
    refused("scale", scale=0.0)
    refused("scale", scale=float("nan"))
    refused("int32", table=table.long())
    refused("int32", lengths=lengths.float())
    refused("dimension", counts=ints([1, 1]))
    refused("out must", out=torch.empty(1, 1, 4, 128, dtype=BF16, device="cuda"))
    refused("CUDA tensor", q_latent=ql.cpu())
    with pytest.raises(RuntimeError, match="on top of one another"):
        fa.latent_append(fa.LatentCache(torch.zeros(36, 288, dtype=BF16, device="cuda").as_strided((4, 32, 288), (288, 288, 1)), 256),
                         ql[0, :, :1], qr[0, :, :1], table, lengths)
    with pytest.raises(RuntimeError, match="strides"):
        fa.LatentCache(torch.zeros(4, 32, 292, dtype=BF16, device="cuda")[..., :288], 256)


# ----------------------------------------------------------------------------- append

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("latent,rope,page,T,heads", [(512, 64, 64, 1, 16), (128, 16, 16, 37, 3), (256, 32, 128, 5, 0), (512, 64, 32, 130, 20)])
def test_append(latent, rope, page, T, heads, interleaved, dtype):
    B, W = 3, -(-(T + 90) // page)
    cache = cache_of(latent, rope, B * W + 2, page, dtype, 1)
    before = cache.data.clone()
    table = torch.randperm(B * W, generator=gen_of(2), device="cuda").to(torch.int32).view(B, W)
    lengths, counts = ints([0, 15, 90]), ints([T, T // 2, 0])
    both = normal(3, dtype, B, T, latent + rope)
    q = normal(4, dtype, B, T, heads, rope + 8)[..., 8:] if heads else None
    angle = torch.arange(90 + T, device="cuda")[:, None] * 100.0 ** (-torch.arange(0, rope, 2, device="cuda") / rope)
    rotation = (angle.cos(), angle.sin())
    for counted in (None, counts):
        cache.data.copy_(before)
        keys, rotated = fa.latent_append(cache, both[..., :latent], both[..., latent:], table, lengths, counts=counted, queries=q, rotation=rotation, interleaved=interleaved)
        assert cache.read_status() == (0, 0)
        want = before.clone()
        unit = torch.finfo(dtype).eps / 2
        for b in range(B):
            n = T if counted is None else int(counted[b])
            at = int(lengths[b]) + torch.arange(n, device="cuda")
            for x, y in ((both[b, :n, latent:], keys[b]),) + (((q[b, :n], rotated[b]),) if heads else ()):
                turned, size = oracle.rotate(x.double(), at, rotation, interleaved)
                assert ((y[:n].double() - turned).abs() <= unit * turned.abs() + 2.0 ** -22 * size + 2.0 ** -25).all()
                assert not y[n:].any()
            where = table[b].long()[at // page], at % page
            want[where] = torch.cat((both[b, :n, :latent], keys[b, :n]), -1)
        assert torch.equal(cache.data, want) and (rotated is None) == (heads == 0)


def test_append_without_rotation_and_out_of_reach():
    cache = cache_of(128, 16, 6, 16, F16, 1)
    table, lengths = ints([[0, 1], [2, -1], [3, 4]]), ints([10, 10, 30])
    c, r, q = normal(1, F16, 3, 8, 128), normal(2, F16, 3, 8, 16), normal(3, F16, 3, 8, 2, 16)
    before = cache.data.clone()
    keys, rotated = fa.latent_append(cache, c, r, table, lengths, queries=q)
    assert torch.equal(keys, r) and torch.equal(rotated, q)
    assert cache.read_status() in ((1, 8), (2, 8))   # two tokens without a page, six behind the table's last position; whichever is first
    want = before.clone()
    want[0, 10:] = torch.cat((c, r), -1)[0, :6]
    want[1, :2] = torch.cat((c, r), -1)[0, 6:]
    want[2, 10:] = torch.cat((c, r), -1)[1, :6]
    want[4, 14:] = torch.cat((c, r), -1)[2, :2]
    assert torch.equal(cache.data, want)
    # a rotation that ends: tokens in front of its end are appended, the others are not
    ones = torch.ones(13, 8, device="cuda")
    cache.data.copy_(before)
    keys, rotated = fa.latent_append(cache, c[:1], r[:1], table[:1], lengths[:1], queries=q[:1], rotation=(ones, ones * 0))
    assert cache.read_status() == (2, 5)
    assert torch.equal(keys[0, :3], r[0, :3]) and not keys[0, 3:].any() and not rotated[0, 3:].any()
    want = before.clone()
    want[0, 10:13] = torch.cat((c, r), -1)[0, :3]
    assert torch.equal(cache.data, want)
    fa.latent_append(cache, c[:1], r[:1], table[:1], ints([-3]))
    assert cache.read_status() == (2, 8) and torch.equal(cache.data, want)


# ----------------------------------------------------------------------------- expanded

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nope,rope", [(64, 16), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("B,T,S,heads,lengths,counts", [
    (1, 1, 1, 1, None, None), (2, 130, 130, 3, None, None), (1, 257, 700, 2, None, None), (3, 100, 300, 2, [300, 101, 0], [100, 37, 5]), (2, 300, 300, 1, [300, 128], [299, 300]),
    (1, 3, 900, 5, [777], None)])
def test_prompts(nope, rope, dtype, B, T, S, heads, lengths, counts):
    q, qr = normal(1, dtype, B, T, heads, nope), normal(2, dtype, B, T, heads, rope)
    kv, r = normal(3, dtype, B, S, heads, 2 * nope), normal(4, dtype, B, S, rope)
    lengths, counts = (None if x is None else ints(x) for x in (lengths, counts))
    for causal in (True, False):
        y = fa.latent_prompt(q, qr, kv, r, lengths=lengths, counts=counts, causal=causal)
        within(y, *oracle.prompt(q, qr, kv, r, (nope + rope) ** -0.5, lengths, counts, causal))
        assert torch.equal(y, fa.latent_prompt(q, qr, kv, r, lengths=lengths, counts=counts, causal=causal))
    assert fa.latent_status(0) == (0, 0)


def test_prompt_strides_out_and_scale():
    B, T, heads, nope, rope = 2, 70, 3, 128, 64
    both = normal(1, BF16, B, heads, T, nope + rope).transpose(1, 2)
    kv, r = normal(2, BF16, B, T, heads + 1, 2 * nope)[:, :, 1:], normal(3, BF16, B, T, 512 + rope)[..., 512:]
    want = fa.latent_prompt(both[..., :nope].contiguous(), both[..., nope:].contiguous(), kv.contiguous(), r.contiguous(), scale=0.2)
    within(want, *oracle.prompt(both[..., :nope], both[..., nope:], kv, r, 0.2))
    out = torch.empty_like(want)
    fa.latent_prompt(both[..., :nope], both[..., nope:], kv, r, scale=0.2, out=out)
    assert torch.equal(out, want)


def test_prompt_growing_scores():
    """Scores that grow along the keys, so that references move in every step."""
    B, T, S, heads, nope, rope = 1, 140, 900, 2, 64, 32
    q, qr = normal(1, F16, B, T, heads, nope), normal(2, F16, B, T, heads, rope)
    grow = torch.linspace(0.05, 4, S, device="cuda")
    kv, r = (normal(3, F16, B, S, heads, 2 * nope) * grow.view(1, S, 1, 1)).half(), (normal(4, F16, B, S, rope) * grow.view(1, S, 1)).half()
    within(fa.latent_prompt(q, qr, kv, r, scale=0.6), *oracle.prompt(q, qr, kv, r, 0.6))


@pytest.mark.parametrize("nope", [64, 128])
def test_prompt_what_is_not_seen_does_not_reach_a_query(nope):
    B, T, S, heads, rope = 2, 150, 400, 2, 64
    q, qr = normal(1, BF16, B, T, heads, nope), normal(2, BF16, B, T, heads, rope)
    kv, r = normal(3, BF16, B, S, heads, 2 * nope), normal(4, BF16, B, S, rope)
    lengths = ints([390, 300])
    want = fa.latent_prompt(q, qr, kv, r, lengths=lengths)
    for what in (float("nan"), float("inf"), -float("inf")):
        kv2, r2 = kv.clone(), r.clone()
        for b, held in enumerate(lengths.tolist()):
            kv2[b, held:], r2[b, held:] = what, what
            kv2[b, held - 20, 0, nope + 3] = what        # a value that the last 20 queries see
            kv2[b, held - 10, 1, 5] = what               # a key that the last 10 see
        y = fa.latent_prompt(q, qr, kv2, r2, lengths=lengths)
        assert torch.equal(y[:, :T - 20], want[:, :T - 20])
        assert torch.equal(y[:, :T - 10, 1], want[:, :T - 10, 1])
        assert not torch.isfinite(y[:, T - 20:, 0]).all(-1).any()
        if what != what:   # (an infinity in a key leaves it the largest weight or none, by the query's sign)
            assert not torch.isfinite(y[:, T - 10:, 1]).any()


def test_prompt_reports_and_refusals():
    q, qr, kv, r = normal(1, F16, 2, 9, 2, 64), normal(2, F16, 2, 9, 2, 16), normal(3, F16, 2, 9, 2, 128), normal(4, F16, 2, 9, 16)
    y = fa.latent_prompt(q, qr, kv, r, lengths=ints([20, -4]))
    assert fa.latent_status(0) == (2, 2) and fa.latent_status(0) == (0, 0)
    assert not y[1].any() and torch.equal(y[0], fa.latent_prompt(q, qr, kv, r)[0])
    for match, kw in (("nope_dim", dict(q_nope=normal(1, F16, 2, 9, 2, 96))), ("rope_dim", dict(q_rope=normal(1, F16, 2, 9, 2, 24))), ("shape", dict(expanded=kv[..., :64])),
                      ("shape", dict(rope_keys=r[:, :8])), ("type", dict(expanded=kv.bfloat16())), ("positive", dict(expanded=kv[:1].expand(2, 9, 2, 128))),
                      ("scale", dict(scale=-1.0)), ("int32", dict(lengths=ints([1, 2]).long())), ("shape", dict(counts=ints([1])))):
        args = {**dict(q_nope=q, q_rope=qr, expanded=kv, rope_keys=r), **kw}
        with pytest.raises(RuntimeError, match=match):
            fa.latent_prompt(args.pop("q_nope"), args.pop("q_rope"), args.pop("expanded"), args.pop("rope_keys"), **args)


def test_both_forms_agree():
    """The absorbed form with W_k^T q, multiplied by W_v, is the expanded form: to the activations' roundings (a few of 2^-8 each)."""
    B, T, S, heads, nope, rope, latent, page = 1, 40, 200, 4, 64, 32, 128, 32
    c, r = normal(1, BF16, B, S, latent), normal(2, BF16, B, S, rope)
    w = (torch.randn(latent, heads, 2 * nope, generator=gen_of(3), device="cuda") / latent ** 0.5).to(BF16)
    q, qr = normal(4, BF16, B, T, heads, nope), normal(5, BF16, B, T, heads, rope)
    cache = fa.latent_cache_create(latent, rope, 7, page)
    table = torch.arange(7, dtype=torch.int32, device="cuda").view(1, 7)
    keys, _ = fa.latent_append(cache, c, r, table, ints([0]))
    scale = (nope + rope) ** -0.5
    expanded = fa.latent_prompt(q, qr, torch.einsum("bsc,chd->bshd", c, w).contiguous(), keys, scale=scale)
    y = fa.latent_attention(cache, torch.einsum("bthd,chd->bthc", q, w[..., :nope]).contiguous(), qr, table, ints([S]), scale=scale)
    absorbed = torch.einsum("bthc,chd->bthd", y, w[..., nope:])
    assert float((absorbed.float() - expanded.float()).norm() / expanded.float().norm()) < 4 * 2.0 ** -8
