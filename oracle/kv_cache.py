"""The paged 8-bit key/value cache in 64 bits, sequence by sequence and head by head: what the tests hold the kernels to.

Works on any device; codes are e4m3 tensors, everything else is float64.
"""
from __future__ import annotations

import math

import torch

LOW_SCALE = 2.0 ** -100


def codes_of(x: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to each x of magnitude 448 at most, ties to the even one."""
    e = (torch.frexp(x).exponent - 1).clamp(min=-6)
    grain = torch.exp2((e - 3).double())
    return torch.round(x / grain) * grain


def scale_of(most: float) -> float:
    """Smallest power of two, LOW_SCALE at least, with most / scale <= 448; NaN if `most` is not finite."""
    if not math.isfinite(most):
        return math.nan
    scale = LOW_SCALE
    if most > 448 * LOW_SCALE:
        m, e = math.frexp(most / 448)
        scale = math.ldexp(1.0, e - 1 if m == 0.5 else e)
    return scale


def rotate(x: torch.Tensor, position: torch.Tensor, rotation, interleaved: bool):
    """x float64 [n, heads, H] at `position` [n]; the result and, for error bounds, the sum of the products' magnitudes."""
    if rotation is None:
        return x, torch.zeros_like(x)
    c, s = (t.double()[position][:, None] for t in rotation)
    H = x.shape[-1]
    i = torch.arange(H // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + H // 2)
    y, size = torch.empty_like(x), torch.empty_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a], size[..., b] = (x[..., a] * c).abs() + (x[..., b] * s).abs(), (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


def values_of(codes: torch.Tensor, scale: torch.Tensor, pages: torch.Tensor, head: int) -> tuple:
    """(codes, scale by token) in float64 of one head of the given pages, their tokens in a row."""
    page = codes.shape[2]
    c = codes.view(torch.uint8)[pages, head].view(torch.float8_e4m3fn).double().reshape(-1, codes.shape[3])
    return c, scale[pages, head].double().repeat_interleave(page)


def attention(cache, queries, table, lengths, counts=None, pages=None, causal=True, unit=2.0 ** -11):
    """(y, bound): the attention in float64 and how far a kernel may be from it that holds scores and sums in 32 bits, rounds
    the weights to fp16 and the result once to a type whose rounding error is `unit`."""
    B, T, F = queries.shape
    H, G, page = cache.head_dim, cache.kv_heads, cache.page_size
    group = F // H // G
    y = torch.zeros(B, T, G, group, H, dtype=torch.float64, device=queries.device)
    bound = torch.zeros_like(y)
    for b in range(B):
        held = int(lengths[b])
        n = T if counts is None else int(counts[b])
        if held == 0 or n == 0:
            continue
        ids = table[b, :-(-held // page)].long()
        at = held - n + torch.arange(n, device=queries.device)
        x = queries[b, :n].double().view(n, G, group, H)
        for g in range(G):
            (kc, ks), (vc, vs) = (values_of(c, s, ids, g) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            k, v = (kc * ks[:, None])[:held], (vc * vs[:, None])[:held]
            seen = torch.arange(held, device=queries.device)[None] <= (at[:, None] if causal else held)
            if pages is not None:
                chosen = pages[b, :n, g].long()
                mine = torch.zeros(n, len(ids) + 1, dtype=torch.bool, device=queries.device)
                mine.scatter_(1, torch.where((chosen >= 0) & (chosen < len(ids)), chosen, len(ids)), True)
                seen = seen & mine[:, :-1].repeat_interleave(page, dim=1)[:, :held]
            s = torch.einsum("trd,ld->trl", x[:, g], k) / math.sqrt(H)
            size = torch.einsum("trd,ld->trl", x[:, g].abs(), k.abs()) / math.sqrt(H)
            s = s.masked_fill(~seen[:, None], -math.inf)
            some = seen.any(-1)[:, None, None]
            p = torch.where(some, torch.softmax(torch.where(some, s, 0.0), dim=-1), 0.0)
            y[b, :n, g] = p @ v
            # weights: fp16 (2^-11; below its normal numbers 2^-25 of the largest weight), the exponent's fp32 error (sums of
            # products, and numbers up to 2^8 with an error of 2^-24 of themselves); the result: `unit`
            spread = 2.0 ** -11 + 2.0 ** -15 + 2.0 ** -21 * torch.where(seen[:, None], size, 0.0).amax(-1, keepdim=True)
            tail = 2.0 ** -25 * (p * vs[:held]).amax(-1, keepdim=True) * vc[:held].abs().sum(0)
            bound[b, :n, g] = spread * (p @ v.abs()) + tail + unit * y[b, :n, g].abs() + 2.0 ** -25
    return y.view(B, T, F), bound.view(B, T, F)


def select(cache, queries, table, lengths, keep, counts=None, first=1, last=1):
    """The selected pages, with the definition's roundings (1 / max |q| * 127, its product with q, max |q| * (1 / 127) and the
    products of scores and scales) in float32 and whole numbers otherwise."""
    B, T, F = queries.shape
    H, G, page = cache.head_dim, cache.kv_heads, cache.page_size
    out = torch.full((B, T, G, keep), -1, dtype=torch.int32)
    bounds = torch.round(cache.bounds.float() / 4)
    for b in range(B):
        held, n = int(lengths[b]), T if counts is None else int(counts[b])
        if held == 0:
            continue
        ids = table[b, :-(-held // page)].long()
        for t in range(n):
            own = (held - n + t) // page
            if held - n + t < 0:
                continue
            x = queries[b, t].float().view(G, -1, H)
            most = x.abs().amax(-1, keepdim=True)
            q8 = torch.where(most > 0, torch.round(x * (most.reciprocal() * 127.0)), 0.0)
            for g in range(G):
                bg = bounds[ids[:own + 1], g].double()                                   # [pages, 2, H]
                whole = torch.maximum(q8[g].double()[:, None] * bg[None, :, 0], q8[g].double()[:, None] * bg[None, :, 1]).sum(-1)
                score = (whole.float() * (most[g] * torch.tensor(1.0 / 127.0, device=most.device))).amax(0) * cache.k_scale[ids[:own + 1], g]
                score[:first] = math.inf
                score[max(0, own + 1 - last):] = math.inf
                score = score.tolist()
                best = sorted(range(own + 1), key=lambda i: (-score[i], i))[:keep]
                out[b, t, g, :len(best)] = torch.tensor(sorted(best), dtype=torch.int32)
    return out
