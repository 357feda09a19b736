"""The operators of the paged 8-bit key/value cache that are timed, and their plain forms.

The cache holds the keys and values of sequences in pages of ``page`` tokens.  A page has, for each key/value head, e4m3
codes and one fp32 scale for its keys and one for its values (a value is code * scale), and the lowest and the highest key
code by dimension.  ``table[b, i]`` is the page of the i-th block of tokens of sequence b, ``lengths[b]`` how many tokens it
holds.  Three operators work on it:

  append     writes T new tokens a sequence behind those it holds (counts[b] of them where the sequences differ), the
             position rotation applied to the keys on the way and to the queries that come with them
  select     scores the pages of a sequence for each query by the pages' bounds and takes the best
  attention  softmax attention of T queries a sequence over its tokens, the queries being its last ones; over all pages, or
             over a list of them for each query and head

A case has an ``op`` and sizes: B sequences, T tokens of each, R query heads on G key/value heads of H dimensions, ``page``
tokens a page, ``low``..``high`` tokens that a sequence holds (before an append; with the queries' own for the others).
"""
import math

import torch

own = False


def listed():
    return [
        # one more token of a single conversation: what the launch costs is the time
        dict(name="append_one", op="append", B=1, T=1, R=32, G=8, H=128, page=64, low=777, high=777, type="bf16", pairs="halves", ragged=False),
        # a token of each of many conversations, as a server appends them between two steps
        dict(name="append_batch", op="append", B=256, T=1, R=32, G=8, H=128, page=64, low=1, high=1000, type="fp16", pairs="halves", ragged=False),
        # prompts of different lengths behind what their sequences hold, ends in the middle of pages
        dict(name="append_prompts", op="append", B=4, T=2048, R=32, G=8, H=128, page=64, low=0, high=333, type="fp16", pairs="neighbours", ragged=True),
        # the pages that one token of one long conversation attends to
        dict(name="select_one", op="select", B=1, T=1, R=32, G=8, H=128, page=64, low=20001, high=20001, type="fp16", keep=32),
        # the same for a batch of very long ones: more bounds than the L2 cache holds
        dict(name="select_batch", op="select", B=32, T=1, R=32, G=8, H=128, page=64, low=30000, high=131072, type="bf16", keep=64),
        # one token of a short conversation
        dict(name="token_short", op="attention", B=1, T=1, R=32, G=8, H=128, page=64, low=301, high=301, type="fp16", keep=0),
        # a token of each conversation of a full batch, of all lengths
        dict(name="token_batch", op="attention", B=64, T=1, R=32, G=8, H=128, page=64, low=100, high=8192, type="fp16", keep=0),
        # two very long documents on the few heads that a tensor-parallel rank holds: the keys have to be divided
        dict(name="token_long", op="attention", B=2, T=1, R=32, G=4, H=128, page=128, low=130000, high=131071, type="bf16", keep=0),
        # five drafted tokens of each sequence, five query heads a key head, small pages
        dict(name="drafted", op="attention", B=16, T=5, R=40, G=8, H=128, page=16, low=500, high=4001, type="bf16", keep=0),
        # a long prompt behind a cached beginning
        dict(name="prompt_long", op="attention", B=1, T=4096, R=32, G=8, H=128, page=64, low=8000, high=8000, type="fp16", keep=0),
        # a batch of shorter prompts of odd lengths, a key head for every query head, small heads
        dict(name="prompt_ragged", op="attention", B=16, T=777, R=16, G=16, H=64, page=32, low=777, high=1300, type="fp16", keep=0),
        # the selected pages of long conversations
        dict(name="token_pages", op="attention", B=16, T=1, R=32, G=8, H=128, page=64, low=16000, high=32768, type="bf16", keep=64),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    """One more case of the same kinds; sizes are spread evenly over their logarithms."""
    kind = rng.choice(("append_tokens", "append_prompts", "select_tokens", "select_prompt", "tokens", "drafted", "prompts", "pages"))
    H = rng.choice((64, 128, 128)) if rng.random() < 0.8 else rng.choice((16, 32))
    G = rng.choice((1, 2, 4, 8))
    c = dict(T=1, R=G * rng.choice((1, 2, 4, 5, 8)), G=G, H=H, page=rng.choice((16, 32, 64, 64, 128)), type=rng.choice(("fp16", "bf16")))
    if kind.startswith("append"):
        c.update(op="append", pairs=rng.choice(("halves", "neighbours")), ragged=False, low=rng.choice((0, 1, 100)))
        if kind == "append_tokens":
            c.update(B=_log_int(rng, 1, 256), high=c["low"] + _log_int(rng, 1, 700))
        else:
            c["T"] = _log_int(rng, 2, 2000)
            c.update(B=_log_int(rng, 1, max(1, 6000 // c["T"])), high=c["low"] + _log_int(rng, 1, 300), ragged=rng.random() < 0.5)
    elif kind.startswith("select"):
        c["T"] = 1 if kind == "select_tokens" else _log_int(rng, 2, 300)
        high = _log_int(rng, 300, 100000 if c["T"] == 1 else 6000)
        tokens = high * c["T"] * c["R"] * 128 // c["page"]
        c.update(op="select", B=_log_int(rng, 1, max(1, min(32, 120_000_000 // tokens))), keep=rng.choice((4, 16, 33, 64)), high=high, low=max(c["T"], high // 3))
    else:
        c["T"] = {"tokens": 1, "drafted": rng.randint(2, 9), "prompts": _log_int(rng, 100, 2000), "pages": rng.choice((1, 1, 2, 5))}[kind]
        most = {"tokens": 100000, "drafted": 20000, "prompts": 4000, "pages": 30000}[kind]
        high = c["T"] + _log_int(rng, 1, most)
        cost = high * (c["T"] * c["R"] // 8 + G)
        c.update(op="attention", B=_log_int(rng, 1, max(1, min(64, 8_000_000 // cost))), high=high, low=max(c["T"], high // rng.choice((1, 3, 50))), keep=rng.choice((4, 16, 33)) if kind == "pages" else 0)
    return c


def _pages(case):
    """How many pages a sequence needs at most."""
    return -(-(case["high"] + (case["T"] if case["op"] == "append" else 0)) // case["page"])


def _codes(shape, gen):
    """Codes as an append leaves them: keys and values of a normal distribution, the largest of a page near the end of the range."""
    codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    for part in codes.split(max(1, (1 << 27) // max(1, codes[0].numel()))):
        x = torch.randn(part.shape, generator=gen, device="cuda", dtype=torch.bfloat16)
        part.copy_(x.mul_(80).clamp_(-440, 440))
    return codes


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    B, T, R, G, H, page, W = (case["B"], case["T"], case["R"], case["G"], case["H"], case["page"], _pages(case))
    dtype = torch.float16 if case["type"] == "fp16" else torch.bfloat16

    def whole(low, high, *shape):
        return torch.randint(low, high + 1, shape, generator=gen, device="cuda", dtype=torch.int32)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    state = dict(case=case, lengths=whole(case["low"], case["high"], B), queries=normal(B, T, R * H))
    n = B * W + 3
    # pages in no order, none for what a sequence does not reach
    order = torch.randperm(n, generator=gen, device="cuda")[:B * W].to(torch.int32).view(B, W)
    reach = state["lengths"] + (T if case["op"] == "append" else 0)
    state["table"] = torch.where(torch.arange(W, device="cuda") * page < reach[:, None], order, -1)
    for name in ("k_scale", "v_scale"):
        state[name] = torch.exp2(whole(-9, -6, n, G).float())
    if case["op"] == "select":
        # the bounds alone are read; the pages that they describe are not made
        bounds = torch.randn(n, G, 2, H, generator=gen, device="cuda").abs_().mul_(60).add_(90)
        bounds[:, :, 0].neg_()
        state["bounds"] = bounds.clamp_(-440, 440).to(torch.float8_e4m3fn)
        state["k"] = state["v"] = torch.empty(1, 1, page, H, dtype=torch.float8_e4m3fn, device="cuda").expand(n, G, page, H)
        return state
    state["k"], state["v"] = _codes((n, G, page, H), gen), _codes((n, G, page, H), gen)
    state["bounds"] = torch.zeros(n, G, 2, H, dtype=torch.float8_e4m3fn, device="cuda")
    if case["op"] == "append":
        state["bounds"][:, :, 0].fill_(-416)
        state["bounds"][:, :, 1].fill_(416)
        state["keys"], state["values"] = normal(B, T, G * H), normal(B, T, G * H)
        state["counts"] = whole(1, T, B) if case["ragged"] else None
        angle = torch.arange(case["high"] + T, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, H, 2, device="cuda") / H)
        state["rotation"] = (angle.cos(), angle.sin())
    elif case["keep"]:
        state["pages"] = _some_pages(state["lengths"], T, G, case["keep"], page, W, gen)
    return state


def _some_pages(lengths, T, G, keep, page, W, gen):
    """For each query and head `keep` of the pages up to its own, which is among them; ascending, the rest -1."""
    at = lengths[:, None] - T + torch.arange(T, device="cuda")
    last = (at // page)[:, :, None, None]
    key = torch.rand(len(lengths), T, G, W, generator=gen, device="cuda")
    index = torch.arange(W, device="cuda")
    key = torch.where(index == last, 2.0, torch.where(index < last, key, -1.0))
    best, chosen = key.topk(min(keep, W), dim=-1)
    chosen = torch.where(best >= 0, chosen, W).sort(dim=-1).values
    chosen = torch.nn.functional.pad(chosen, (0, keep - chosen.shape[-1]), value=W)
    return torch.where(chosen < W, chosen, -1).to(torch.int32)


# ----------------------------------------------------------------------------- a pass

def run(state):
    case = state["case"]
    if own:
        import fused_attention_b200 as fa
        if "cache" not in state:   # the handle that a program keeps beside the tensors
            state["cache"] = fa.KVCache(state["k"], state["v"], state["k_scale"], state["v_scale"], state["bounds"])
        cache = state["cache"]
        if case["op"] == "append":
            rotated = fa.cache_append(cache, state["keys"], state["values"], state["table"], state["lengths"], counts=state["counts"],
                                      queries=state["queries"], rotation=state["rotation"], interleaved=case["pairs"] == "neighbours")
            return _updated(state, rotated)
        if case["op"] == "select":
            return fa.cache_select(cache, state["queries"], state["table"], state["lengths"], case["keep"], first=1, last=2)
        return fa.cache_attention(cache, state["queries"], state["table"], state["lengths"], pages=state.get("pages"))
    if case["op"] == "append":
        return _updated(state, _append(state))
    if case["op"] == "select":
        return _select(state)
    return _attention_pages(state) if case["keep"] else _attention(state)


def _updated(state, rotated):
    return dict(queries=rotated, **{name: state[name] for name in ("k", "v", "k_scale", "v_scale", "bounds")})


# ----------------------------------------------------------------------------- the plain forms

def _rotate(x, cos, sin, pairs):
    """x [B, T, heads, H] in 32 bits, cos and sin [B, T, 1, H/2]."""
    if pairs == "halves":
        a, b = x.chunk(2, dim=-1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)


def _power(k):
    """2^k in 32 bits for whole k."""
    return (k + 127).to(torch.int32).bitwise_left_shift(23).view(torch.float32)


def _scale_of(most):
    """The smallest power of two, 2^-100 at least, that brings `most` to 448 or below."""
    part, exponent = torch.frexp(most)
    k = exponent - 9 + (part > 0.875)
    return _power(torch.where(most > 0, k, -100).clamp(min=-100))


def _append(state):
    case = state["case"]
    B, T, R, G, H, page, W = (case["B"], case["T"], case["R"], case["G"], case["H"], case["page"], _pages(case))
    lengths, table = state["lengths"].long(), state["table"].long()
    step = torch.arange(T, device="cuda")
    taken = step < (state["counts"][:, None] if state["counts"] is not None else T)
    taken = taken.expand(B, T)
    at = lengths[:, None] + step
    cos, sin = (t[at][:, :, None] for t in state["rotation"])
    queries = _rotate(state["queries"].view(B, T, R, H).float(), cos, sin, case["pairs"]).to(state["queries"].dtype).view(B, T, R * H)
    queries = torch.where(taken[:, :, None], queries, 0)
    keys = _rotate(state["keys"].view(B, T, G, H).float(), cos, sin, case["pairs"])
    values = state["values"].view(B, T, G, H).float()
    # the blocks from the first touched one on, every token at its place in them
    blocks = (T + page - 2) // page + 1
    begin, inside = lengths // page, lengths % page
    slot = torch.arange(blocks * page, device="cuda").view(blocks, page)
    fresh = (slot >= inside[:, None, None]) & (slot < (inside + taken.sum(1))[:, None, None])
    old = (slot < inside[:, None, None]) & (slot < page)
    touched = fresh.any(-1)
    which = (begin[:, None] + torch.arange(blocks, device="cuda")).clamp(max=W - 1)
    page_of = table.gather(1, which)[touched]
    source = (slot.view(1, -1) - inside[:, None]).clamp(0, T - 1)[:, :, None, None].expand(B, blocks * page, G, H)
    fresh, old = fresh[touched][:, None, :, None], old[touched][:, None, :, None]
    holds = old.any(2)[..., 0]
    for name, x in (("k", keys), ("v", values)):
        x = x.gather(1, source).view(B, blocks, page, G, H).transpose(2, 3)[touched]
        x = torch.where(fresh, x, 0.0)
        before = state[name + "_scale"][page_of]
        scale = _scale_of(x.abs().amax(dim=(2, 3)))
        scale = torch.where(holds, torch.maximum(before, scale), scale)
        shrink = torch.where(holds, before / scale, 1.0)
        codes = state[name].view(torch.uint8)[page_of].view(torch.float8_e4m3fn)
        moved = (codes.float() * shrink[:, :, None, None]).to(torch.float8_e4m3fn)
        codes = torch.where(old, moved.view(torch.uint8), codes.view(torch.uint8))
        new = (x / scale[:, :, None, None]).to(torch.float8_e4m3fn)
        codes = torch.where(fresh, new.view(torch.uint8), codes)
        state[name].view(torch.uint8)[page_of] = codes
        state[name + "_scale"][page_of] = scale
        if name == "k":
            bounds = state["bounds"].view(torch.uint8)[page_of].view(torch.float8_e4m3fn).float()
            bounds = (bounds * shrink[:, :, None, None]).to(torch.float8_e4m3fn).float()
            low, high = (torch.where(fresh, new.float(), end) for end in (math.inf, -math.inf))
            low, high = low.amin(2), high.amax(2)
            low = torch.where(holds[..., None], torch.minimum(low, bounds[:, :, 0]), low)
            high = torch.where(holds[..., None], torch.maximum(high, bounds[:, :, 1]), high)
            state["bounds"].view(torch.uint8)[page_of] = torch.stack((low, high), dim=2).to(torch.float8_e4m3fn).view(torch.uint8)
    return queries


def _position(state):
    """Where each query stands in its sequence, [B, T]."""
    T = state["case"]["T"]
    return state["lengths"].long()[:, None] - T + torch.arange(T, device="cuda")


def _select(state):
    case = state["case"]
    B, T, R, G, H, page, W = (case["B"], case["T"], case["R"], case["G"], case["H"], case["page"], _pages(case))
    table = state["table"].long().clamp(min=0)
    x = state["queries"].view(B, T, G, R // G, H).float()
    most = x.abs().amax(-1, keepdim=True)
    q8 = torch.where(most > 0, torch.round(x * (127.0 / most)), 0.0)
    bounds = torch.round(state["bounds"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * 0.25)
    low, high = bounds[:, :, :, 0], bounds[:, :, :, 1]   # [B, W, G, H]
    dots = torch.einsum("btgrd,bwgd->btgrw", q8.clamp(min=0), high) + torch.einsum("btgrd,bwgd->btgrw", q8.clamp(max=0), low)
    score = (dots * (most / 127.0)).amax(3) * state["k_scale"][table].transpose(1, 2)[:, None]
    index = torch.arange(W, device="cuda")
    last = (_position(state) // page)[:, :, None, None]
    score = torch.where((index < 1) | (index > last - 2), math.inf, score)
    score = torch.where(index > last, -math.inf, score)
    best, chosen = score.sort(dim=-1, descending=True, stable=True)
    chosen = torch.where(best > -math.inf, chosen, W)[..., :case["keep"]].sort(dim=-1).values
    chosen = torch.nn.functional.pad(chosen, (0, case["keep"] - chosen.shape[-1]), value=W)
    return torch.where(chosen < W, chosen, -1).to(torch.int32)


def _softmax_product(scores, allowed, product):
    """Softmax of the allowed scores along the last axis and its product with the values; zeros where nothing is allowed."""
    scores = torch.where(allowed, scores, -math.inf)
    most = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(most > -math.inf, most, 0.0))
    total = weights.sum(-1, keepdim=True)
    return product(weights) / torch.where(total > 0, total, 1.0)


def _attention(state):
    case = state["case"]
    B, T, R, G, H, page, W = (case["B"], case["T"], case["R"], case["G"], case["H"], case["page"], _pages(case))
    table = state["table"].long().clamp(min=0)

    def whole(name):
        x = state[name].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * state[name + "_scale"][table][..., None, None]
        return x.transpose(1, 2).reshape(B, G, 1, W * page, H)

    x = state["queries"].view(B, T, G, R // G, H).permute(0, 2, 3, 1, 4).float()
    scores = torch.matmul(x, whole("k").transpose(-1, -2)) / math.sqrt(H)
    allowed = torch.arange(W * page, device="cuda") <= _position(state)[:, None, None, :, None]
    y = _softmax_product(scores, allowed, lambda w: torch.matmul(w, whole("v")))
    return y.permute(0, 3, 1, 2, 4).reshape(B, T, R * H).to(state["queries"].dtype)


def _attention_pages(state):
    case = state["case"]
    B, T, R, G, H, page = (case["B"], case["T"], case["R"], case["G"], case["H"], case["page"])
    chosen = state["pages"].long()
    keep = chosen.shape[-1]
    page_of = state["table"].long()[torch.arange(B, device="cuda")[:, None, None, None], chosen.clamp(min=0)]
    head = torch.arange(G, device="cuda")[:, None]

    def some(name):
        x = state[name].view(torch.uint8)[page_of, head].view(torch.float8_e4m3fn).float() * state[name + "_scale"][page_of, head][..., None, None]
        return x.reshape(B, T, G, keep * page, H)

    x = state["queries"].view(B, T, G, R // G, H).float()
    scores = torch.matmul(x, some("k").transpose(-1, -2)) / math.sqrt(H)
    at = chosen[..., None] * page + torch.arange(page, device="cuda")
    allowed = (chosen[..., None] >= 0) & (at <= _position(state)[:, :, None, None, None])
    y = _softmax_product(scores, allowed.reshape(B, T, G, 1, keep * page), lambda w: torch.matmul(w, some("v")))
    return y.reshape(B, T, R * H).to(state["queries"].dtype)


# ----------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "select":
        return None   # whole numbers
    return _exact_append(state) if case["op"] == "append" else _exact_attention(state)


def _to_codes(x):
    """The e4m3 number nearest to each x of at most 448, ties to the even one."""
    exponent = (torch.frexp(x).exponent - 1).clamp(min=-6)
    grain = torch.exp2((exponent - 3).double())
    return torch.round(x / grain) * grain


def _exact_append(state):
    """Sequence by sequence and block by block, from the definition."""
    case = state["case"]
    T, R, G, H, page = (case["T"], case["R"], case["G"], case["H"], case["page"])
    out = {name: state[name].double() for name in ("k", "v", "k_scale", "v_scale", "bounds")}
    out["queries"] = torch.zeros_like(state["queries"], dtype=torch.float64)
    lengths, table = state["lengths"].tolist(), state["table"].tolist()
    counts = state["counts"].tolist() if state["counts"] is not None else [T] * len(lengths)
    first = torch.arange(H // 2, device="cuda")
    a, b = (first, first + H // 2) if case["pairs"] == "halves" else (2 * first, 2 * first + 1)
    for s, (held, n) in enumerate(zip(lengths, counts)):
        cos, sin = (t[held:held + n].double()[:, None] for t in state["rotation"])

        def turned(x, heads):
            x = x[s, :n].double().view(n, heads, H)
            y = torch.empty_like(x)
            y[..., a] = x[..., a] * cos - x[..., b] * sin
            y[..., b] = x[..., b] * cos + x[..., a] * sin
            return y

        out["queries"][s, :n] = turned(state["queries"], R).reshape(n, R * H)
        new = dict(k=turned(state["keys"], G), v=state["values"][s, :n].double().view(n, G, H))
        for block in range(held // page, (held + n - 1) // page + 1):
            p = table[s][block]
            kept = max(0, held - block * page)
            rows = slice(max(0, block * page - held), min(n, (block + 1) * page - held))
            for name in ("k", "v"):
                x = new[name][rows].transpose(0, 1)          # [G, tokens, H]
                most = x.abs().amax(dim=(1, 2))
                scale = torch.exp2(torch.ceil(torch.log2(most / 448)).clamp(min=-100))
                if kept:
                    before = out[name + "_scale"][p].clone()
                    scale = torch.maximum(scale, before)
                    shrink = (before / scale)[:, None, None]
                    out[name][p][:, :kept] = _to_codes(out[name][p][:, :kept] * shrink)
                    if name == "k":
                        out["bounds"][p] = _to_codes(out["bounds"][p] * shrink)
                codes = _to_codes(x / scale[:, None, None])
                out[name][p][:, kept:kept + codes.shape[1]] = codes
                out[name + "_scale"][p] = scale
                if name == "k":
                    low, high = codes.amin(1), codes.amax(1)
                    if kept:
                        low, high = torch.minimum(low, out["bounds"][p][:, 0]), torch.maximum(high, out["bounds"][p][:, 1])
                    out["bounds"][p] = torch.stack((low, high), dim=1)
    return out


def _exact_attention(state):
    """Head by head: one key/value head of one sequence at a time."""
    case = state["case"]
    B, T, R, G, H, page = (case["B"], case["T"], case["R"], case["G"], case["H"], case["page"])
    group = R // G
    if B * G * (T if case["keep"] else 1) > 8000:
        return None   # too many heads for a loop over them
    out = torch.zeros(B, T, G, group, H, dtype=torch.float64, device="cuda")
    for s, held in enumerate(state["lengths"].tolist()):
        pages = state["table"][s, :-(-held // page)].long()
        x = state["queries"][s].double().view(T, G, group, H)
        at = held - T + torch.arange(T, device="cuda")
        for g in range(G):
            k, v = (state[n].view(torch.uint8)[pages, g].view(torch.float8_e4m3fn).double() * state[n + "_scale"][pages, g].double()[:, None, None]
                    for n in ("k", "v"))
            k, v = k.reshape(-1, H)[:held], v.reshape(-1, H)[:held]
            scores = torch.einsum("trd,ld->trl", x[:, g], k) / math.sqrt(H)
            seen = torch.arange(held, device="cuda") <= at[:, None]
            if case["keep"]:
                chosen = state["pages"][s, :, g].long()
                mine = torch.zeros(T, len(pages) + 1, dtype=torch.bool, device="cuda")
                mine.scatter_(1, torch.where(chosen >= 0, chosen, len(pages)), True)
                seen = seen & mine[:, :-1].repeat_interleave(page, dim=1)[:, :held]
            scores.masked_fill_(~seen[:, None], -math.inf)
            out[s, :, g] = torch.softmax(scores, dim=-1) @ v
    return out.view(B, T, R * H)


# ----------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    B, T, R, G, H, page = (case["B"], case["T"], case["R"], case["G"], case["H"], case["page"])
    mean = (case["low"] + case["high"]) / 2
    if case["op"] == "append":
        tokens = B * (T / 2 if case["ragged"] else T)
        pages = B * (1 + (tokens / B - 1) / page)
        # read: keys, values, queries, the angles; written: codes, queries, a scale and bounds a page
        return dict(bytes=tokens * (2 * G * H * 3 + 2 * R * H * 2 + 4 * H) + pages * G * (8 + 2 * H), flops=tokens * (R + G) * 3 * H)
    if case["op"] == "select":
        pages = mean / page
        return dict(bytes=B * (pages * G * (2 * H + 4) + T * (2 * R * H + 4 * G * case["keep"])), flops=B * T * R * pages * 2 * H)
    keys = mean - (T - 1) / 2                 # that a query sees, on average
    read = mean
    if case["keep"]:
        keys = min(keys, case["keep"] * page)
        read = min(mean, keys * T)
    return dict(bytes=B * (2 * read * G * H + 8 * read / page * G + T * R * H * 4), flops=4.0 * B * T * R * H * keys)
