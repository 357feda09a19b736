"""The operators of a latent cache and of the pages of a cache that are timed, and their plain forms.

A latent cache holds one vector a token for all heads, ``latent`` dimensions that are key and value at once and ``rope`` more that
are rotated by the token's position and belong to the key alone, in pages of ``page`` tokens.  ``table[b, i]`` is the page of the
i-th block of tokens of sequence b, ``lengths[b]`` how many tokens it holds, ``refs[p]`` how many entries of the table hold page p.

  append    writes T new tokens a sequence behind those it holds (counts[b] of them where the sequences differ), the rotation
            applied to the rotary part of the keys on the way and to that of the queries that come with them
  absorbed  softmax attention of T queries a sequence over its tokens' latent vectors, the queries being its last tokens: the score
            of a head is q_latent . latent + q_rope . rope, the values are the latent vectors themselves
  expanded  the same with the keys and values of every head that the latent vectors have been multiplied out to: for prompts
  beams     sequences go on as copies of others that share their pages, get the pages that one more token needs, a page of
            their own in place of one that they would write to and share, and those pages' contents are copied
  compact   the pages that are held move to the front of the cache

A case has an ``op`` and sizes; ``low``..``high`` are the tokens that a sequence holds (before an append; with the queries' own
for attention).
"""
import math

import torch

own = False


def listed():
    return [
        # a token of each of many conversations, as a server appends them between two steps
        dict(name="append_tokens", op="append", B=128, T=1, R=20, latent=512, rope=64, page=64, low=1, high=4000, type="bf16", pairs="neighbours", ragged=False),
        # prompts of different lengths behind what their sequences hold, ends in the middle of pages
        dict(name="append_prompts", op="append", B=4, T=2048, R=32, latent=512, rope=64, page=64, low=0, high=333, type="fp16", pairs="halves", ragged=True),
        # one token of a short conversation: what the launch costs is the time
        dict(name="token_short", op="absorbed", B=1, T=1, R=16, latent=512, rope=64, page=64, low=301, high=301, type="bf16", ragged=False),
        # a token of each conversation of a full batch of all lengths, on the heads that a tensor-parallel rank holds
        dict(name="token_batch", op="absorbed", B=64, T=1, R=16, latent=512, rope=64, page=64, low=100, high=8192, type="bf16", ragged=False),
        # the same with all heads on one device: as many products as the bytes leave time for
        dict(name="token_wide", op="absorbed", B=32, T=1, R=128, latent=512, rope=64, page=64, low=1000, high=8192, type="bf16", ragged=False),
        # four drafted tokens of each sequence, odd heads, a smaller vector, small pages
        dict(name="drafted", op="absorbed", B=16, T=4, R=20, latent=256, rope=32, page=16, low=500, high=4001, type="fp16", ragged=False),
        # a long prompt, its first part known from before
        dict(name="prompt_long", op="expanded", B=1, T=4096, R=20, nope=128, rope=64, low=6000, high=6000, type="bf16", ragged=False),
        # a batch of shorter prompts of odd lengths, small heads
        dict(name="prompt_ragged", op="expanded", B=8, T=777, R=12, nope=64, rope=32, low=777, high=1300, type="fp16", ragged=True),
        # two searches of four beams each over an 8-bit cache
        dict(name="beams_few", op="beams", B=8, beams=4, kind="codes", layers=1, G=8, H=128, page=64, low=900, high=2000, spare=40),
        # many searches over the latent caches of two layers
        dict(name="beams_many", op="beams", B=256, beams=8, kind="latent", layers=2, latent=512, rope=64, page=64, low=100, high=2000, spare=300),
        # a small cache, more than half of it given back
        dict(name="compact_small", op="compact", B=8, kind="latent", layers=1, latent=512, rope=64, page=32, low=100, high=1500, held=0.8),
        # a large 8-bit cache after many conversations have ended
        dict(name="compact_large", op="compact", B=64, kind="codes", layers=1, G=8, H=128, page=64, low=1000, high=8000, held=0.8),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    """One more case of the same kinds; sizes are spread evenly over their logarithms."""
    kind = rng.choice(("append_tokens", "append_prompts", "tokens", "tokens", "drafted", "chunk", "prompts", "prompts", "beams", "compact"))
    c = dict(type=rng.choice(("fp16", "bf16")), ragged=False)
    if kind.startswith("append"):
        c.update(op="append", R=_log_int(rng, 1, 64), latent=rng.choice((128, 256, 512, 512)), rope=rng.choice((16, 32, 64, 64)), page=rng.choice((16, 32, 64, 128)),
                 pairs=rng.choice(("halves", "neighbours")), low=rng.choice((0, 1, 100)), T=1 if kind == "append_tokens" else _log_int(rng, 2, 2048))
        c.update(B=_log_int(rng, 1, 256 if c["T"] == 1 else max(1, 8000 // c["T"])), high=c["low"] + _log_int(rng, 1, 3000 if c["T"] == 1 else 300))
        c["ragged"] = c["T"] > 1 and rng.random() < 0.5
    elif kind in ("tokens", "drafted", "chunk"):
        c.update(op="absorbed", R=rng.choice((1, 5, 8, 16, 16, 20, 32, 64, 128)), latent=rng.choice((128, 256, 512, 512)), rope=rng.choice((16, 32, 64, 64)),
                 page=rng.choice((16, 32, 64, 64, 128)), T={"tokens": 1, "drafted": rng.randint(2, 8), "chunk": _log_int(rng, 20, 300)}[kind])
        high = c["T"] + _log_int(rng, 1, {"tokens": 60000, "drafted": 16000, "chunk": 3000}[kind])
        most = min(64, 260_000 // high, int(30e9 / (4.0 * c["T"] * c["R"] * high * c["latent"])))
        c.update(B=_log_int(rng, 1, max(1, most)), high=high, low=max(c["T"], high // rng.choice((1, 3, 50))))
        c["ragged"] = c["T"] > 1 and rng.random() < 0.5
    elif kind == "prompts":
        c.update(op="expanded", R=rng.choice((1, 4, 12, 16)), nope=rng.choice((64, 128, 128)), rope=rng.choice((16, 32, 64, 64)), T=_log_int(rng, 20, 3000))
        high = c["T"] + rng.choice((0, _log_int(rng, 1, 2000)))
        c.update(B=_log_int(rng, 1, max(1, min(16, int(2e8 / (c["R"] * c["T"] * high))))), high=high, low=max(c["T"], high // rng.choice((1, 2))), ragged=rng.random() < 0.5)
    else:
        c = dict(op=kind, kind=rng.choice(("latent", "codes")), layers=rng.choice((1, 2)), page=rng.choice((16, 32, 64, 128)), low=_log_int(rng, 1, 500))
        c.update(dict(latent=rng.choice((128, 256, 512)), rope=rng.choice((32, 64))) if c["kind"] == "latent" else dict(G=rng.choice((1, 2, 8)), H=rng.choice((32, 64, 128))))
        c["high"] = c["low"] + _log_int(rng, 10, 2000 if kind == "beams" else 6000)
        if kind == "beams":
            c.update(beams=rng.choice((2, 3, 4, 8)), spare=rng.choice((5, 100)))
            c["B"] = c["beams"] * _log_int(rng, 1, 32)
        else:
            c.update(B=_log_int(rng, 1, 64), held=rng.choice((0.5, 0.8, 1.0)))
    return c


# ----------------------------------------------------------------------------- inputs

def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _whole(gen, low, high, *shape):
    return torch.randint(low, high + 1, shape, generator=gen, device="cuda", dtype=torch.int32)


def _normal(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16 if math.prod(shape) > 1 << 27 else torch.float32).to(dtype)


def _contents(case, n, gen):
    """The tensors of the layers' caches, of `n` pages each, as a serving process has filled them."""
    layers = []
    for _ in range(case["layers"]):
        if case["kind"] == "latent":
            layers.append(dict(data=_normal(gen, torch.bfloat16, n, case["page"], case["latent"] + case["rope"])))
            continue
        G, H, page = case["G"], case["H"], case["page"]
        layer = {}
        for name in ("k", "v"):
            layer[name] = torch.empty(n, G, page, H, dtype=torch.float8_e4m3fn, device="cuda")
            for part in layer[name].split(max(1, (1 << 27) // (G * page * H))):
                part.copy_(torch.randn(part.shape, generator=gen, device="cuda", dtype=torch.bfloat16).mul_(80).clamp_(-440, 440))
            layer[name + "_scale"] = torch.exp2(_whole(gen, -9, -6, n, G).float())
        layer["bounds"] = torch.randn(n, G, 2, H, generator=gen, device="cuda").mul_(200).clamp_(-440, 440).to(torch.float8_e4m3fn)
        layers.append(layer)
    return layers


def _prepare_pages(case, gen):
    B, page = case["B"], case["page"]
    if case["op"] == "compact":
        W = -(-case["high"] // page)
        lengths = _whole(gen, case["low"], case["high"], B)
        mine = torch.arange(W, device="cuda") * page < lengths[:, None]
        used = int(mine.sum())
        n = math.ceil(B * W / case["held"])
        table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
        table[mine] = torch.randperm(n, generator=gen, device="cuda")[:used].to(torch.int32)
        # some sequences have begun as others did
        for b in range(1, B, 3):
            shared = int(min(lengths[b], lengths[b - 1])) // page // 2
            table[b, :shared] = table[b - 1, :shared]
        state = dict(table=table, lengths=lengths)
    else:
        beams, groups, W = case["beams"], B // case["beams"], -(-case["high"] // page) + 1
        lengths = _whole(gen, case["low"], case["high"], groups).repeat_interleave(beams)
        blocks = (lengths + page - 1) // page
        # beams of a search share its beginning, a block or more at their ends are their own
        common = (blocks - _whole(gen, 1, 3, groups).repeat_interleave(beams)).clamp(min=0)
        col = torch.arange(W, device="cuda")
        leader = torch.arange(B, device="cuda") % beams == 0
        mine = (col < blocks[:, None]) & ((col >= common[:, None]) | leader[:, None])
        used = int(mine.sum())
        n = groups * W + 4 * B + case["spare"]
        table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
        table[mine] = torch.randperm(n, generator=gen, device="cuda")[:used].to(torch.int32)
        first = table[torch.arange(B, device="cuda") // beams * beams]
        table = torch.where(col < common[:, None], first, table)
        # every beam goes on, or is replaced by one in front of it that goes on
        goes_on = (torch.rand(B, generator=gen, device="cuda") < 0.4) | leader
        at = torch.arange(B, device="cuda")
        parents = torch.where(goes_on, at, -1).cummax(0).values.to(torch.int32)
        state = dict(table=table, lengths=lengths, parents=parents, counts=torch.ones(B, dtype=torch.int32, device="cuda"))
    held = state["table"][state["table"] >= 0].long()
    state["refs"] = torch.bincount(held, minlength=n).to(torch.int32)
    state["layers"] = _contents(case, n, gen)
    return state


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] in ("beams", "compact"):
        return dict(case=case, **_prepare_pages(case, gen))
    B, T, R, rope = case["B"], case["T"], case["R"], case["rope"]
    dtype = torch.float16 if case["type"] == "fp16" else torch.bfloat16
    state = dict(case=case, lengths=_whole(gen, case["low"], case["high"], B), counts=_whole(gen, 1, T, B) if case["ragged"] else None)
    if case["op"] == "expanded":
        nope, S = case["nope"], case["high"]
        # queries as a projection leaves them, the parts of a head beside each other
        state["q_rope"] = _normal(gen, dtype, B, T, R, rope)
        state["q_nope"] = _normal(gen, dtype, B, T, R, nope + rope)[..., :nope]
        state["expanded"] = _normal(gen, dtype, B, S, R, 2 * nope)
        state["rope_keys"] = _normal(gen, dtype, B, S, rope)
        return state
    latent, page = case["latent"], case["page"]
    reach = state["lengths"] + (T if case["op"] == "append" else 0)
    W = -(-(case["high"] + (T if case["op"] == "append" else 0)) // page)
    n = B * W + 3
    # pages in no order, none for what a sequence does not reach
    order = torch.randperm(n, generator=gen, device="cuda")[:B * W].to(torch.int32).view(B, W)
    state["table"] = torch.where(torch.arange(W, device="cuda") * page < reach[:, None], order, -1)
    state["data"] = _normal(gen, dtype, n, page, latent + rope)
    if case["op"] == "append":
        # slices of one projection's result, as a layer has them
        whole = _normal(gen, dtype, B, T, latent + rope)
        state["latents"], state["rope_keys"] = whole[..., :latent], whole[..., latent:]
        state["queries"] = _normal(gen, dtype, B, T, R, 128 + rope)[..., 128:]
        angle = torch.arange(case["high"] + T, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, rope, 2, device="cuda") / rope)
        state["rotation"] = (angle.cos(), angle.sin())
    else:
        state["q_latent"], state["q_rope"] = _normal(gen, dtype, B, T, R, latent), _normal(gen, dtype, B, T, R, rope)
    return state


def _scale(case):
    """Of the scores: that of the heads before their keys were absorbed."""
    return 1 / math.sqrt(case.get("nope", 128) + case["rope"])


# ----------------------------------------------------------------------------- a pass

def _handles(state):
    """The handles that a program keeps beside the tensors."""
    import fused_attention_b200 as fa
    case = state["case"]
    if case["op"] in ("beams", "compact"):
        state["pool"] = fa.PagePool(state["refs"])
        state["caches"] = [fa.LatentCache(x["data"], case["latent"]) if case["kind"] == "latent" else fa.KVCache(x["k"], x["v"], x["k_scale"], x["v_scale"], x["bounds"])
                           for x in state["layers"]]
    elif case["op"] != "expanded":
        state["cache"] = fa.LatentCache(state["data"], case["latent"])


def run(state):
    case = state["case"]
    if own:
        import fused_attention_b200 as fa
        if not ({"pool", "cache"} & state.keys()):
            _handles(state)
        if case["op"] == "append":
            keys, queries = fa.latent_append(state["cache"], state["latents"], state["rope_keys"], state["table"], state["lengths"], counts=state["counts"],
                                             queries=state["queries"], rotation=state["rotation"], interleaved=case["pairs"] == "neighbours")
            return dict(data=state["data"], keys=keys, queries=queries)
        if case["op"] == "absorbed":
            return fa.latent_attention(state["cache"], state["q_latent"], state["q_rope"], state["table"], state["lengths"], scale=_scale(case), counts=state["counts"])
        if case["op"] == "expanded":
            return fa.latent_prompt(state["q_nope"], state["q_rope"], state["expanded"], state["rope_keys"], scale=_scale(case), lengths=state["lengths"],
                                    counts=state["counts"])
        if case["op"] == "beams":
            fa.pages_fork(state["pool"], state["table"], state["lengths"], state["parents"])
            granted, sources, targets = fa.pages_reserve(state["pool"], state["table"], state["lengths"], state["counts"], case["page"])
            fa.cache_copy(state["caches"], sources, targets)
            return _beams_result(state, granted, sources, targets)
        pool, table, sources, targets = fa.pages_compact(state["pool"], state["table"])
        fa.cache_copy(state["caches"], sources, targets)
        return dict(refs=pool.refs, table=table, sources=sources, targets=targets, layers=state["layers"])
    return {"append": _append, "absorbed": _absorbed, "expanded": _expanded, "beams": _beams, "compact": _compact}[case["op"]](state)


def _beams_result(state, granted, sources, targets):
    return dict(granted=granted, sources=sources, targets=targets, **{name: state[name] for name in ("table", "lengths", "refs", "layers")})


# ----------------------------------------------------------------------------- the plain forms

def _rotate(x, cos, sin, pairs):
    """x [..., rope] in 32 bits, cos and sin [..., rope / 2]."""
    if pairs == "halves":
        a, b = x.chunk(2, dim=-1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)


def _append(state):
    case = state["case"]
    T, page = case["T"], case["page"]
    step = torch.arange(T, device="cuda")
    taken = (step < (state["counts"][:, None] if state["counts"] is not None else T)).expand(case["B"], T)
    at = state["lengths"].long()[:, None] + step
    cos, sin = (t[at] for t in state["rotation"])
    keys = _rotate(state["rope_keys"].float(), cos, sin, case["pairs"]).to(state["data"].dtype)
    queries = _rotate(state["queries"].float(), cos[:, :, None], sin[:, :, None], case["pairs"]).to(state["data"].dtype)
    page_of = state["table"].long().gather(1, at // page)
    state["data"][page_of[taken], (at % page)[taken]] = torch.cat((state["latents"], keys), dim=-1)[taken]
    return dict(data=state["data"], keys=torch.where(taken[..., None], keys, 0), queries=torch.where(taken[..., None, None], queries, 0))


def _limits(state):
    """How many keys each query sees, [B, T]; none where its sequence has no such token."""
    T = state["case"]["T"]
    held = state["lengths"].long()[:, None]
    count = state["counts"].long()[:, None] if state["counts"] is not None else T
    step = torch.arange(T, device="cuda")
    return torch.where(step < count, held - count + step + 1, 0).clamp(min=0)


def _weights(scores, limits):
    """Softmax of scores [B, R, T, S] over the keys that each query sees; zeros where it sees none."""
    allowed = torch.arange(scores.shape[-1], device="cuda") < limits[:, None, :, None]
    scores = torch.where(allowed, scores, -math.inf)
    most = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(most > -math.inf, most, 0.0))
    total = weights.sum(-1, keepdim=True)
    return weights / torch.where(total > 0, total, 1.0)


def _absorbed(state):
    case = state["case"]
    B, T, R, latent = case["B"], case["T"], case["R"], case["latent"]
    rows = state["data"][state["table"].long().clamp(min=0)].float().flatten(1, 2)               # [B, S, latent + rope]
    q = torch.cat((state["q_latent"], state["q_rope"]), dim=-1).float().transpose(1, 2)          # [B, R, T, latent + rope]
    scores = torch.matmul(q.reshape(B, R * T, -1), rows.transpose(1, 2)).view(B, R, T, -1) * _scale(case)
    weights = _weights(scores, _limits(state))
    y = torch.matmul(weights.view(B, R * T, -1), rows[..., :latent]).view(B, R, T, latent)
    return y.transpose(1, 2).to(state["q_latent"].dtype)


def _expanded(state):
    case = state["case"]
    nope, R = case["nope"], case["R"]
    q = torch.cat((state["q_nope"], state["q_rope"]), dim=-1).float().transpose(1, 2)
    shared = state["rope_keys"].float()[:, None].expand(-1, R, -1, -1)
    keys, values = state["expanded"].float().transpose(1, 2).split(nope, dim=-1)
    scores = torch.matmul(q, torch.cat((keys, shared), dim=-1).transpose(-1, -2)) * _scale(case)
    return torch.matmul(_weights(scores, _limits(state)), values).transpose(1, 2).to(state["q_nope"].dtype)


def _copy_pages(state, sources, targets):
    taken = (sources >= 0) & (targets >= 0)
    sources, targets = sources[taken].long(), targets[taken].long()
    for layer in state["layers"]:
        for x in layer.values():
            x = x.view(torch.uint8) if x.element_size() == 1 else x
            x[targets] = x[sources]


def _beams(state):
    case = state["case"]
    B, page, table, lengths, refs = case["B"], case["page"], state["table"], state["lengths"], state["refs"]
    n, W = len(refs), table.shape[1]

    def count(entries, by):
        held = entries[entries >= 0].long()
        refs.index_add_(0, held, torch.full_like(held, by, dtype=torch.int32))

    # the rows of the parents
    parents = state["parents"].long()
    count(table, -1)
    table.copy_(torch.where(parents[:, None] >= 0, table[parents.clamp(min=0)], -1))
    lengths.copy_(torch.where(parents >= 0, lengths[parents.clamp(min=0)], 0))
    count(table, 1)
    # the blocks that the tokens need
    held, more = lengths.long()[:, None], state["counts"].long()[:, None]
    block = torch.arange(W, device="cuda")
    need = (held + more + page - 1) // page
    count(torch.where(block >= need, table, -1), -1)
    table.masked_fill_(block >= need, -1)
    written = (block >= held // page) & (block < need) & (more > 0)
    shared = written & (table >= 0) & (refs[table.clamp(min=0).long()] > 1)
    entry = torch.where(shared, table, n).long()
    writers = torch.zeros(n + 1, dtype=torch.int32, device="cuda").index_add_(0, entry.flatten(), shared.flatten().int())
    row = torch.arange(B, device="cuda")[:, None].expand(B, W)
    lowest = torch.full((n + 1,), B, device="cuda").scatter_reduce_(0, entry.flatten(), row.flatten(), "amin")
    keeps = shared & (writers[entry] == torch.cat((refs, refs.new_zeros(1)))[entry]) & (lowest[entry] == row)
    wants = written & ((table < 0) | (shared & ~keeps))
    free = (refs == 0).nonzero()[:, 0]
    rank = (wants.flatten().cumsum(0) - 1).view(B, W)
    given = wants & (rank < len(free))
    new = torch.nn.functional.pad(free, (0, 1))[rank.clamp(0, len(free))].to(torch.int32)
    refused = torch.where(wants & ~given, block, W + 1).amin(1, keepdim=True)
    granted = torch.where(refused <= W, (refused * page - held).clamp(min=0).minimum(more), more)[:, 0].to(torch.int32)
    part = given & (table >= 0) & (block == held // page) & (held % page > 0)
    sources = torch.where(part, table, -1).amax(1)
    targets = torch.where(part, new, -1).amax(1)
    count(torch.where(given, table, -1), -1)
    table.copy_(torch.where(given, new, table))
    count(torch.where(given, table, -1), 1)
    _copy_pages(state, sources, targets)
    return _beams_result(state, granted, sources, targets)


def _compact(state):
    refs, table = state["refs"], state["table"]
    n = len(refs)
    used = refs > 0
    front = torch.arange(n, device="cuda") < used.sum()
    moved, holes = (used & ~front).nonzero()[:, 0], (~used & front).nonzero()[:, 0]
    to = torch.arange(n, device="cuda")
    to[moved] = holes
    sources, targets = (torch.nn.functional.pad(x, (0, n - len(x)), value=-1).to(torch.int32) for x in (moved, holes))
    new_refs = torch.zeros_like(refs)
    new_refs[to[used]] = refs[used]
    new_table = torch.where(table >= 0, to[table.clamp(min=0).long()], -1).to(torch.int32)
    _copy_pages(state, sources, targets)
    return dict(refs=new_refs, table=new_table, sources=sources, targets=targets, layers=state["layers"])


# ----------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "expanded" and case["B"] * case["R"] > 2000 or case["B"] > 2000:
        return None   # too many for a loop over them
    return {"append": _exact_append, "absorbed": _exact_absorbed, "expanded": _exact_expanded, "beams": _exact_beams, "compact": _exact_compact}[case["op"]](state)


def _exact_append(state):
    """Sequence by sequence, pair by pair of dimensions."""
    case = state["case"]
    T, page, latent, rope = case["T"], case["page"], case["latent"], case["rope"]
    first = torch.arange(rope // 2, device="cuda")
    a, b = (first, first + rope // 2) if case["pairs"] == "halves" else (2 * first, 2 * first + 1)
    data = state["data"].double()
    keys, queries = torch.zeros(state["rope_keys"].shape, dtype=torch.float64, device="cuda"), torch.zeros(state["queries"].shape, dtype=torch.float64, device="cuda")
    counts = state["counts"].tolist() if state["counts"] is not None else [T] * case["B"]
    for s, (held, n) in enumerate(zip(state["lengths"].tolist(), counts)):
        cos, sin = (t[held:held + n].double() for t in state["rotation"])
        x = state["rope_keys"][s, :n].double()
        keys[s, :n, a], keys[s, :n, b] = x[:, a] * cos - x[:, b] * sin, x[:, b] * cos + x[:, a] * sin
        x = state["queries"][s, :n].double()
        cos, sin = cos[:, None], sin[:, None]
        queries[s, :n, :, a], queries[s, :n, :, b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
        at = torch.arange(held, held + n, device="cuda")
        pages = state["table"][s].long()[at // page]
        data[pages, at % page, :latent] = state["latents"][s, :n].double()
        data[pages, at % page, latent:] = keys[s, :n]
    return dict(data=data, keys=keys, queries=queries)


def _exact_absorbed(state):
    """Sequence by sequence, a few rows at a time."""
    case = state["case"]
    T, R, latent, page = case["T"], case["R"], case["latent"], case["page"]
    out = torch.zeros(state["q_latent"].shape, dtype=torch.float64, device="cuda")
    counts = state["counts"].tolist() if state["counts"] is not None else [T] * case["B"]
    for s, (held, n) in enumerate(zip(state["lengths"].tolist(), counts)):
        rows = state["data"][state["table"][s, :-(-held // page)].long()].flatten(0, 1)[:held].double()
        c, r = rows[:, :latent], rows[:, latent:]
        for t0 in range(0, n, max(1, (1 << 27) // (R * held))):
            t1 = min(n, t0 + max(1, (1 << 27) // (R * held)))
            scores = (state["q_latent"][s, t0:t1].double() @ c.T + state["q_rope"][s, t0:t1].double() @ r.T) * _scale(case)
            limit = held - n + 1 + torch.arange(t0, t1, device="cuda")
            scores.masked_fill_(torch.arange(held, device="cuda") >= limit[:, None, None], -math.inf)
            y = torch.softmax(scores, dim=-1) @ c
            out[s, t0:t1] = torch.where((limit > 0)[:, None, None], y, 0.0)
    return out


def _exact_expanded(state):
    """Head by head of one sequence at a time."""
    case = state["case"]
    T, nope = case["T"], case["nope"]
    out = torch.zeros(*state["q_nope"].shape, dtype=torch.float64, device="cuda")
    counts = state["counts"].tolist() if state["counts"] is not None else [T] * case["B"]
    for s, (held, n) in enumerate(zip(state["lengths"].tolist(), counts)):
        shared = state["rope_keys"][s, :held].double()
        hidden = torch.arange(held, device="cuda") > held - n + torch.arange(n, device="cuda")[:, None]
        for h in range(case["R"]):
            k, v = state["expanded"][s, :held, h].double().split(nope, dim=-1)
            scores = (state["q_nope"][s, :n, h].double() @ k.T + state["q_rope"][s, :n, h].double() @ shared.T) * _scale(case)
            out[s, :n, h] = torch.softmax(scores.masked_fill_(hidden, -math.inf), dim=-1) @ v
    return out


def _moved(state, pairs):
    """The layers' contents after the moves, one after another."""
    layers = []
    for layer in state["layers"]:
        new = {}
        for name, x in layer.items():
            y = x.view(torch.uint8).clone()
            for source, target in pairs:
                y[target] = x.view(torch.uint8)[source]
            new[name] = y.view(x.dtype)
        layers.append(new)
    return layers


def _exact_beams(state):
    """With lists, sequence by sequence and block by block; the pages suffice in all cases."""
    case = state["case"]
    B, page = case["B"], case["page"]
    parents, old = state["parents"].tolist(), state["table"].tolist()
    held = state["lengths"].tolist()
    table = [list(old[p]) for p in parents]
    lengths = [held[p] for p in parents]

    def holders(p):
        return [b for b in range(B) if p in rows[b]]

    rows = [set(x) for x in table]
    takes = []
    for b in range(B):
        first, need = lengths[b] // page, (lengths[b] + page) // page
        for i in range(len(table[b])):
            if i >= need:
                table[b][i] = -1
        rows[b] = set(table[b])
        takes.append(range(first, need))
    writes = {(b, table[b][i]) for b in range(B) for i in takes[b] if table[b][i] >= 0}
    wanted = []
    for b in range(B):
        for i in takes[b]:
            p = table[b][i]
            if p < 0:
                wanted.append((b, i))
                continue
            all_of_them = holders(p)
            if len(all_of_them) > 1 and not (b == all_of_them[0] and all((o, p) in writes for o in all_of_them)):
                wanted.append((b, i))
    used = {p for row in table for p in row}
    free = iter(p for p in range(len(state["refs"])) if p not in used)
    sources, targets = [-1] * B, [-1] * B
    for b, i in wanted:
        new = next(free)
        if table[b][i] >= 0 and lengths[b] % page and i == lengths[b] // page:
            sources[b], targets[b] = table[b][i], new
        table[b][i] = new
    refs = [0] * len(state["refs"])
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1

    def whole(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    layers = _moved(state, [(s, t) for s, t in zip(sources, targets) if s >= 0])
    return dict(granted=state["counts"], sources=whole(sources), targets=whole(targets), table=whole(table), lengths=whole(lengths), refs=whole(refs), layers=layers)


def _exact_compact(state):
    refs, table = state["refs"].tolist(), state["table"].tolist()
    used = [p for p, r in enumerate(refs) if r > 0]
    moved = [p for p in used if p >= len(used)]
    holes = [p for p in range(len(used)) if refs[p] == 0]
    to = {p: p for p in used if p < len(used)}
    to.update(zip(moved, holes))
    new = [0] * len(refs)
    for p in used:
        new[to[p]] = refs[p]

    def whole(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    rest = [-1] * (len(refs) - len(moved))
    return dict(refs=whole(new), table=whole([[to.get(p, -1) for p in row] for row in table]), sources=whole(moved + rest), targets=whole(holes + rest),
                layers=_moved(state, list(zip(moved, holes))))


# ----------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    B = case["B"]
    mean = (case["low"] + case["high"]) / 2
    if case["op"] in ("beams", "compact"):
        page = case["page"]
        a_page = case["layers"] * (2 * page * (case["latent"] + case["rope"]) if case["kind"] == "latent" else case["G"] * (2 * page * case["H"] + 2 * case["H"] + 8))
        blocks = math.ceil(mean / page)
        if case["op"] == "beams":
            # most beams but the first that goes on in its place write to a shared page; tables read and written once, counts changed
            copies = 0.6 * B * (1 - 1 / case["beams"]) * (1 - 1 / page)
            return dict(bytes=2 * copies * a_page + B * (blocks * 8 + 32), flops=0.0)
        used, n = B * blocks, B * -(-case["high"] // page) / case["held"]
        return dict(bytes=2 * used * (1 - used / n) * a_page + used * 8 + n * 16, flops=0.0)
    T, R, rope = case["T"], case["R"], case["rope"]
    tokens = B * (T / 2 if case["ragged"] else T)
    if case["op"] == "append":
        # read: latents, keys, queries, the angles; written: rows of the cache, the rotated keys and queries
        return dict(bytes=tokens * (4 * case["latent"] + 6 * rope + 4 * R * rope + 4 * rope), flops=tokens * (R + 1) * 3 * rope)
    keys = mean - (tokens / B - 1) / 2        # that a query sees, on average
    if case["op"] == "absorbed":
        latent = case["latent"]
        return dict(bytes=B * mean * 2 * (latent + rope) + tokens * R * 2 * (2 * latent + rope), flops=2.0 * tokens * R * keys * (2 * latent + rope))
    nope = case["nope"]
    return dict(bytes=B * mean * 2 * (2 * R * nope + rope) + tokens * R * 2 * (2 * nope + rope), flops=2.0 * tokens * R * keys * (2 * nope + rope))
