"""Answering from a cache of latent vectors: a small decoder with random weights that reads prompts, goes on token by token, forks and lets go.

  python -m fused_attention_b200.latent_decoding [--batch 4 --beams 2 --prompt 1000 --new 32 --layers 3]

Keys and values of all heads come from one latent vector a token.  A prompt is read with them multiplied out (``latent_prompt``), a token with its
queries multiplied into the latent space instead (``latent_attention``), so that the cache holds latent vectors and rotated rotary keys alone.
Pages belong to a pool: a step reserves what its tokens need, sequences that fork share pages until they write to them, and sequences that
end give theirs back.  A token's step, pages and all, is captured in a CUDA graph once and replayed.
"""
from __future__ import annotations

import argparse
import math
from typing import List, Optional

import torch

from .cached_decoding import CachedDecoder, rotation_angles
from .latent import LatentCache, latent_append, latent_attention, latent_cache_create, latent_prompt
from .pages import cache_copy, page_pool_create, pages_compact, pages_fork, pages_reserve


class LatentDecoder:
    """``layers`` of norm, attention over the latent cache, norm, feed-forward, with the caches of up to ``batch`` sequences."""

    def __init__(self, batch: int, most_tokens: int, *, layers: int = 3, heads: int = 8, nope: int = 64, rope: int = 32, latent: int = 256, width: int = 512,
                 vocabulary: int = 1000, page_size: int = 32, n_pages: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, seed: int = 179):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.heads, self.nope, self.rope, self.latent, self.dtype, self.page_size = heads, nope, rope, latent, dtype, page_size

        def weight(rows: int, cols: int) -> torch.Tensor:
            return (torch.randn(rows, cols, generator=gen, device="cuda") / math.sqrt(rows)).to(dtype)
        self.embedding = torch.randn(vocabulary, width, generator=gen, device="cuda").to(dtype)
        # kv: what a latent vector is multiplied by for a head's own part of the key, and for its value behind it
        self.layers = [dict(q=weight(width, heads * (nope + rope)), down_kv=weight(width, latent + rope), kv=weight(latent, heads * 2 * nope), out=weight(heads * nope, width),
                            up=weight(width, 2 * width), down=weight(2 * width, width)) for _ in range(layers)]
        pages = -(-most_tokens // page_size)
        self.pool = page_pool_create(batch * pages if n_pages is None else n_pages)
        self.caches: List[LatentCache] = [latent_cache_create(latent, rope, self.pool.n_pages, page_size, dtype) for _ in range(layers)]
        self.table = torch.full((batch, pages), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.rotation = rotation_angles(pages * page_size, rope)

    def forward(self, tokens: torch.Tensor, counts: Optional[torch.Tensor] = None, *, fresh: bool = False) -> torch.Tensor:
        """tokens int64 [B, T], of which sequence b has counts[b]: appended to the sequences as far as there are pages; the logits, [B, T,
        vocabulary].  ``fresh``: the sequences hold nothing yet, and attention is over this call's keys and values multiplied out."""
        B, T = tokens.shape
        if counts is None:
            counts = torch.full((B,), T, dtype=torch.int32, device="cuda")
        counts, sources, targets = pages_reserve(self.pool, self.table, self.lengths, counts, self.page_size)
        cache_copy(self.caches, sources, targets)
        after, scale = self.lengths + counts, (self.nope + self.rope) ** -0.5
        x = self.embedding[tokens]
        for layer, cache in zip(self.layers, self.caches):
            h = CachedDecoder._norm(x)
            q_nope, q_rope = (h @ layer["q"]).view(B, T, self.heads, -1).split((self.nope, self.rope), dim=-1)
            c, r = (h @ layer["down_kv"]).split((self.latent, self.rope), dim=-1)
            r, q_rope = latent_append(cache, c, r, self.table, self.lengths, counts=counts, queries=q_rope, rotation=self.rotation)
            w = layer["kv"].view(self.latent, self.heads, 2 * self.nope)
            if fresh:
                y = latent_prompt(q_nope, q_rope, (c @ layer["kv"]).view(B, T, self.heads, -1), r, scale=scale, lengths=after, counts=counts)
            else:
                q = torch.einsum("bthd,chd->bthc", q_nope, w[..., :self.nope]).contiguous()
                y = latent_attention(cache, q, q_rope, self.table, after, scale=scale, counts=counts)
                y = torch.einsum("bthc,chd->bthd", y, w[..., self.nope:])
            x = x + y.reshape(B, T, -1) @ layer["out"]
            x = x + torch.nn.functional.silu(CachedDecoder._norm(x) @ layer["up"]) @ layer["down"]
        self.lengths.copy_(after)
        return CachedDecoder._norm(x) @ self.embedding.T

    def fork(self, parents: torch.Tensor) -> None:
        """Sequence b goes on as a copy of sequence parents[b]; -1: it is let go."""
        pages_fork(self.pool, self.table, self.lengths, parents)

    def compact(self) -> None:
        """Pages that are held move to the front of the caches.  (Captured steps go on with the same table and counts.)"""
        pool, table, sources, targets = pages_compact(self.pool, self.table)
        cache_copy(self.caches, sources, targets)
        self.table.copy_(table)
        self.pool.refs.copy_(pool.refs)

    def capture_step(self):
        """(graph, tokens): a replay takes tokens [B, 1], appends them and leaves the most likely next ones in their place."""
        tokens = torch.zeros(len(self.lengths), 1, dtype=torch.int64, device="cuda")

        def step(counts: Optional[torch.Tensor] = None) -> None:
            tokens.copy_(self.forward(tokens, counts).argmax(-1))
        # (library handles and allocations come into being ahead of the capture, in a step without a token for any sequence)
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
    for name, value in (("batch", 4), ("beams", 2), ("prompt", 1000), ("new", 32), ("layers", 3)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    B = a.batch * a.beams
    model = LatentDecoder(B, a.prompt + a.new + 1, layers=a.layers)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    # the first beam of each search reads the prompt, the others fork from it
    counts = torch.randint(max(1, a.prompt // 2), a.prompt + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    leader = torch.arange(B, device="cuda", dtype=torch.int32) // a.beams * a.beams
    counts = torch.where(leader == torch.arange(B, device="cuda"), counts, 0).to(torch.int32)
    logits = model.forward(torch.randint(0, len(model.embedding), (B, a.prompt), generator=gen, device="cuda"), counts, fresh=True)
    first = logits[leader.long(), counts[leader.long()].long() - 1].topk(a.beams).indices   # a beam's own next token
    graph, tokens = model.capture_step()
    model.fork(leader)
    tokens.copy_(first[torch.arange(B, device="cuda"), torch.arange(B, device="cuda") % a.beams][:, None])
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    torch.cuda.synchronize()
    begin.record()
    for _ in range(a.new):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    held = int((model.pool.refs > 0).sum())
    model.fork(torch.where(leader == torch.arange(B, device="cuda"), leader, -1).to(torch.int32))   # the first beams have won
    model.compact()
    torch.cuda.synchronize()
    assert model.pool.read_status() == (0, 0) and all(c.read_status() == (0, 0) for c in model.caches)
    print(f"{a.batch} searches of {a.beams} beams, prompts of up to {a.prompt} tokens: {begin.elapsed_time(end) / a.new * 1000:.0f} us a step; {held} pages held, "
          f"{int((model.pool.refs > 0).sum())} after the other beams were let go")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
