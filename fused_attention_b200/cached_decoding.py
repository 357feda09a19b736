"""Answering from the key/value cache: a small decoder with random weights that reads prompts and goes on token by token.

  python -m fused_attention_b200.cached_decoding [--batch 8 --prompt 2000 --new 64 --layers 4 --keep 0]

Every layer appends the keys and values of its new tokens to its cache (rotating them and the queries on the way) and attends
over the cache; with ``--keep N`` a token attends to the N pages that the bounds of the pages' keys select.  A token's step is
captured in a CUDA graph once and replayed: lengths live on the device.  Prompts of different lengths share a call.
"""
from __future__ import annotations

import argparse
import math
from typing import List, Optional

import torch

from .cache import KVCache, cache_append, cache_attention, cache_create, cache_select


def rotation_angles(positions: int, head_dim: int, base: float = 10000.0, device="cuda"):
    """(cos, sin) [positions, head_dim / 2] of the position rotation."""
    angle = torch.arange(positions, device=device)[:, None] * base ** (-torch.arange(0, head_dim, 2, device=device) / head_dim)
    return angle.cos(), angle.sin()


class CachedDecoder:
    """``layers`` of norm, attention over the cache, norm, feed-forward, with the caches of a batch of sequences."""

    def __init__(self, batch: int, most_tokens: int, *, layers: int = 4, heads: int = 16, kv_heads: int = 4, head_dim: int = 128, vocabulary: int = 1000,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, seed: int = 179):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim, self.dtype = heads, kv_heads, head_dim, dtype
        width = heads * head_dim

        def weight(rows: int, cols: int) -> torch.Tensor:
            return (torch.randn(rows, cols, generator=gen, device="cuda") / math.sqrt(rows)).to(dtype)
        self.embedding = torch.randn(vocabulary, width, generator=gen, device="cuda").to(dtype)
        self.layers = [dict(qkv=weight(width, (heads + 2 * kv_heads) * head_dim), out=weight(width, width), up=weight(width, 2 * width), down=weight(2 * width, width))
                       for _ in range(layers)]
        pages = -(-most_tokens // page_size)
        self.caches: List[KVCache] = [cache_create(head_dim, kv_heads, batch * pages, page_size) for _ in range(layers)]
        # which page a sequence's blocks lie in: any order will do
        self.table = torch.randperm(batch * pages, generator=gen, device="cuda").to(torch.int32).view(batch, pages)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.rotation = rotation_angles(pages * page_size, head_dim)

    @staticmethod
    def _norm(x: torch.Tensor) -> torch.Tensor:
        return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def forward(self, tokens: torch.Tensor, counts: Optional[torch.Tensor] = None, keep: int = 0) -> torch.Tensor:
        """tokens int64 [B, T], of which sequence b has counts[b]: appended to the sequences; the logits, [B, T, vocabulary]."""
        q_width, kv_width = self.heads * self.head_dim, self.kv_heads * self.head_dim
        x = self.embedding[tokens]
        after = self.lengths + (tokens.shape[1] if counts is None else counts)
        for layer, cache in zip(self.layers, self.caches):
            # slices of one product: rows that are farther apart than they are long
            q, k, v = (self._norm(x) @ layer["qkv"]).split((q_width, kv_width, kv_width), dim=-1)
            q = cache_append(cache, k, v, self.table, self.lengths, counts=counts, queries=q, rotation=self.rotation)
            pages = cache_select(cache, q, self.table, after, keep, counts=counts, last=2) if keep else None
            x = x + cache_attention(cache, q, self.table, after, counts=counts, pages=pages) @ layer["out"]
            x = x + torch.nn.functional.silu(self._norm(x) @ layer["up"]) @ layer["down"]
        self.lengths.copy_(after)
        return self._norm(x) @ self.embedding.T

    def capture_step(self, keep: int = 0):
        """(graph, tokens): a replay takes tokens [B, 1], appends them and leaves the most likely next ones in their place."""
        tokens = torch.zeros(len(self.lengths), 1, dtype=torch.int64, device="cuda")

        def step(counts: Optional[torch.Tensor] = None) -> None:
            tokens.copy_(self.forward(tokens, counts, keep=keep).argmax(-1))
        # Library handles and allocations come into being ahead of the capture, in a step without a token for any sequence: one that is
        # appended and taken back would leave its page's scale enlarged and its bounds widened.
        none = torch.zeros_like(self.lengths)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(none)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        return graph, tokens


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("batch", 8), ("prompt", 2000), ("new", 64), ("layers", 4), ("heads", 16), ("kv-heads", 4), ("head-dim", 128), ("keep", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    model = CachedDecoder(a.batch, a.prompt + a.new + 1, layers=a.layers, heads=a.heads, kv_heads=a.kv_heads, head_dim=a.head_dim)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    counts = torch.randint(max(1, a.prompt // 2), a.prompt + 1, (a.batch,), generator=gen, device="cuda", dtype=torch.int32)
    prompts = torch.randint(0, len(model.embedding), (a.batch, a.prompt), generator=gen, device="cuda")
    begin, middle, end = (torch.cuda.Event(enable_timing=True) for _ in range(3))
    model.forward(prompts, counts)   # (first calls)
    model.lengths.zero_()
    begin.record()
    logits = model.forward(prompts, counts)
    middle.record()
    graph, tokens = model.capture_step(a.keep)
    tokens.copy_(logits[torch.arange(a.batch), counts.long() - 1].argmax(-1, keepdim=True))
    torch.cuda.synchronize()
    out = []
    start = torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(a.new):
        graph.replay()
        out.append(tokens.clone())
    end.record()
    torch.cuda.synchronize()
    for cache in model.caches:
        assert cache.read_status() == (0, 0)
    per = start.elapsed_time(end) / a.new
    print(f"prompts of {int(counts.min())} to {int(counts.max())} tokens in {begin.elapsed_time(middle):.2f} ms; {a.new} tokens each for {a.batch} sequences, "
          f"{per * 1000:.0f} us a step, {a.batch / per * 1000:.0f} tokens/s; the first sequence goes on {torch.cat(out, 1)[0, :8].tolist()}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
