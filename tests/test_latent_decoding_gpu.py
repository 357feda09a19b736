"""A decoder that answers from the cache of latent vectors: pages, appending and both forms of attention together, as the example module runs them.

Tolerance: 16-bit activations (bf16: 2^-8 of themselves a rounding, some forty of them in a row through three layers and two forms that
round in different places, adding up like a random walk: 2^-8 * sqrt(40) = 2.5 %) against the spread of the logits.
"""
import pytest
import torch

from fused_attention_b200.latent_decoding import LatentDecoder

pytestmark = pytest.mark.gpu


def prompts(B, T):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    return torch.randint(0, 300, (B, T), generator=gen, device="cuda")


def model(B=3, **kw):
    return LatentDecoder(B, 260, **{**dict(layers=2, vocabulary=300), **kw})


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def spread(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def clean(m):
    assert m.pool.read_status() == (0, 0) and all(c.read_status() == (0, 0) for c in m.caches)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_prompt_at_once_and_in_chunks(dtype):
    """The expanded form of the whole against the absorbed one of its chunks."""
    tokens, counts = prompts(3, 200), ints([200, 77, 1])
    whole, parts = model(dtype=dtype), model(dtype=dtype)
    logits = whole.forward(tokens, counts, fresh=True)
    first = torch.minimum(counts, ints(60))
    a = parts.forward(tokens[:, :60].contiguous(), first, fresh=True)
    b = parts.forward(tokens[:, 60:].contiguous(), counts - first)
    assert whole.lengths.tolist() == parts.lengths.tolist() == [200, 77, 1]
    for s, n in enumerate(counts.tolist()):
        assert spread(a[s, :min(n, 60)], logits[s, :min(n, 60)]) < 0.05
        if n > 60:
            assert spread(b[s, :n - 60], logits[s, 60:n]) < 0.05
    clean(whole), clean(parts)


def test_forks_go_on_as_their_parents_would():
    """Three beams of one prompt, in few pages: they share its beginning, each goes on as a sequence of its own does; then two are let go."""
    tokens = prompts(3, 90)
    forked, apart = model(n_pages=14), model()
    forked.forward(tokens[:1].expand(3, 90).contiguous(), ints([90, 0, 0]), fresh=True)
    assert int((forked.pool.refs > 0).sum()) == 3                       # 90 tokens, pages of 32
    forked.fork(ints([0, 0, 0]))
    apart.forward(tokens[:1].expand(3, 90).contiguous(), fresh=True)
    nxt = prompts(3, 60)
    for t in range(50):
        a, b = forked.forward(nxt[:, t:t + 1].contiguous()), apart.forward(nxt[:, t:t + 1].contiguous())
        assert torch.equal(a, b)                                        # the same rows in other pages: the same bits
    held = int((forked.pool.refs > 0).sum())
    assert held == 2 + 3 * 3                                            # two full pages for all, three of one's own each
    forked.fork(ints([2, -1, -1]))
    before = forked.pool.refs.clone()
    forked.compact()
    assert int((forked.pool.refs > 0).sum()) == 5 and forked.pool.refs[:5].all() and not torch.equal(before, forked.pool.refs)
    a = forked.forward(nxt[2:].expand(3, 60)[:, 50:51].contiguous(), ints([1, 0, 0]))
    b = apart.forward(nxt[:, 50:51].contiguous())
    assert torch.equal(a[0], b[2])
    clean(forked), clean(apart)


def test_steps_in_a_graph_are_the_steps():
    tokens = prompts(3, 151)
    eager, graphed = model(), model()
    for m in (eager, graphed):
        m.forward(tokens[:, :150].contiguous(), fresh=True)
    graph, at = graphed.capture_step()
    at.copy_(tokens[:, 150:])
    now = tokens[:, 150:].clone()
    for _ in range(20):
        graph.replay()
        now = eager.forward(now).argmax(-1)
        assert torch.equal(now, at)
    assert eager.lengths.tolist() == graphed.lengths.tolist() == [170] * 3
    clean(eager), clean(graphed)


def test_pages_that_run_out():
    """A sequence whose tokens find no page gets none of them, and the others go on."""
    m = model(n_pages=4)
    m.forward(prompts(3, 60), ints([60, 60, 60]), fresh=True)           # two pages each: the third finds none
    assert m.lengths.tolist() == [60, 60, 0] and m.pool.read_status()[0] == 3
    m.fork(ints([0, -1, -1]))
    m.forward(prompts(3, 60), ints([0, 0, 60]))
    assert m.lengths.tolist() == [60, 0, 60]
    clean(m)


def test_the_module_runs(capsys):
    import sys
    from fused_attention_b200 import latent_decoding
    old = sys.argv
    sys.argv = ["latent_decoding", "--batch", "2", "--beams", "2", "--prompt", "100", "--new", "8", "--layers", "1"]
    try:
        assert latent_decoding.main() == 0
    finally:
        sys.argv = old
    assert "us a step" in capsys.readouterr().out
