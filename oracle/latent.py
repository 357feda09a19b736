"""Attention over latent vectors in 64 bits, and appending to their cache: what the tests hold the kernels to.  Works on any device."""
from __future__ import annotations

import math

import torch


def attend(q, k, v, limits, scale: float, unit: float, half: bool):
    """(y, bound) of queries q [n, dk] on keys k [S, dk] and values v [S, dv] in float64, query i seeing keys [0, limits[i]).

    The bound is for a kernel that holds scores, maxima and sums in 32 bits, rounds weights to a type whose rounding error is `unit` and
    sums them as rounded, and rounds the result once.  A weight is off by its rounding, by the exponent's fp32 error (sums of products;
    numbers up to 2^8 with an error of 2^-24 of themselves) and, with fp16 (`half`), below its normal numbers by 2^-25 of the largest weight; in
    numerator and sum alike, so that each counts twice.
    """
    seen = torch.arange(k.shape[0], device=q.device) < limits[:, None]
    s = (q @ k.T) * scale
    size = (q.abs() @ k.abs().T) * scale
    s = s.masked_fill(~seen, -math.inf)
    some = seen.any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, s, 0.0), dim=-1), 0.0)
    y = p @ v
    spread = unit + 2.0 ** -15 + 2.0 ** -21 * torch.where(seen, size, 0.0).amax(-1, keepdim=True)
    # what is behind a query's limit is not read: a value there may be anything
    held = torch.where(torch.isfinite(v), v.abs(), 0.0)
    tail = 2.0 ** -25 * p.amax(-1, keepdim=True) * (seen.double() @ held) if half else 0.0
    bound = 2 * (spread * (p @ held + y.abs()) / 2 + tail) + spread * (p @ held) + unit * y.abs() + 2.0 ** -25
    return y, bound


def limits_of(held: int, count: int, T: int, causal: bool, device):
    """Keys [0, ...) that each of T queries sees; 0 for one that the sequence does not have."""
    t = torch.arange(T, device=device)
    return torch.where(t < count, (held - count + t + 1 if causal else torch.full_like(t, held)).clamp(0, held), 0)


def attention(data, latent: int, q_latent, q_rope, table, lengths, scale: float, counts=None, causal: bool = True):
    """The absorbed form over pages [n_pages, page, latent + rope]; (y, bound) [B, T, heads, latent]."""
    B, T, heads, _ = q_latent.shape
    unit, half = torch.finfo(q_latent.dtype).eps / 2, q_latent.dtype == torch.float16
    y = torch.zeros(q_latent.shape, dtype=torch.float64, device=data.device)
    bound = torch.full_like(y, 0.0)
    page = data.shape[1]
    for b in range(B):
        held = int(lengths[b])
        if held == 0:
            continue
        rows = data[table[b, :-(-held // page)].long()].flatten(0, 1)[:held].double()
        limits = limits_of(held, T if counts is None else int(counts[b]), T, causal, data.device)
        for h in range(heads):
            q = torch.cat((q_latent[b, :, h], q_rope[b, :, h]), dim=-1).double()
            y[b, :, h], bound[b, :, h] = attend(q, rows, rows[:, :latent], limits, scale, unit, half)
    return y, bound


def prompt(q_nope, q_rope, expanded, rope_keys, scale: float, lengths=None, counts=None, causal: bool = True):
    """The expanded form; (y, bound) [B, T, heads, nope]."""
    B, T, heads, nope = q_nope.shape
    S = expanded.shape[1]
    unit, half = torch.finfo(q_nope.dtype).eps / 2, q_nope.dtype == torch.float16
    y = torch.zeros(q_nope.shape, dtype=torch.float64, device=q_nope.device)
    bound = torch.zeros_like(y)
    for b in range(B):
        held = S if lengths is None else int(lengths[b])
        if held == 0:
            continue
        limits = limits_of(held, T if counts is None else int(counts[b]), T, causal, q_nope.device)
        for h in range(heads):
            q = torch.cat((q_nope[b, :, h], q_rope[b, :, h]), dim=-1).double()
            k = torch.cat((expanded[b, :held, h, :nope], rope_keys[b, :held]), dim=-1).double()
            y[b, :, h], bound[b, :, h] = attend(q, k, expanded[b, :held, h, nope:].double(), limits, scale, unit, half)
    return y, bound


def rotate(x, position, rotation, interleaved: bool):
    """x float64 [n, ..., rope] at `position` [n]; the result, and the sum of the products' magnitudes."""
    if rotation is None:
        return x, torch.zeros_like(x)
    shape = (len(position),) + (1,) * (x.dim() - 2) + (x.shape[-1] // 2,)
    c, s = (t.double()[position].view(shape) for t in rotation)
    half = x.shape[-1] // 2
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, size = torch.empty_like(x), torch.empty_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a], size[..., b] = (x[..., a] * c).abs() + (x[..., b] * s).abs(), (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size
