"""A decoder that answers from the key/value cache: appending, selecting and attending together, as the example module runs them.

Tolerances: bf16 activations (2^-8 of themselves a rounding, some thirty of them in a row through two layers, adding up like a random
walk: 2^-8 * sqrt(30) = 2 %) against the spread of the logits; pages that are filled in two ways differ by codes that are one e4m3
step apart where bf16 rounding moved a value across a boundary, 6 % of single values, which a softmax over hundreds of keys averages out.
"""
import pytest
import torch

from fused_attention_b200.cached_decoding import CachedDecoder

pytestmark = pytest.mark.gpu


def model(**kw):
    return CachedDecoder(3, 400, **{**dict(layers=2, heads=8, kv_heads=2, head_dim=64, vocabulary=300, page_size=32), **kw})


def prompts():
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    return torch.randint(0, 300, (3, 200), generator=gen, device="cuda")


def spread(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_at_once_and_in_parts_agree(dtype):
    tokens, counts = prompts(), torch.tensor([200, 77, 1], dtype=torch.int32, device="cuda")
    whole, parts = model(dtype=dtype), model(dtype=dtype)
    logits = whole.forward(tokens, counts)
    first = torch.minimum(counts, torch.tensor(60, device="cuda", dtype=torch.int32))
    a = parts.forward(tokens[:, :60].contiguous(), first)
    b = parts.forward(tokens[:, 60:].contiguous(), counts - first)
    assert torch.equal(whole.lengths, parts.lengths) and whole.lengths.tolist() == [200, 77, 1]
    for s, n in enumerate(counts.tolist()):
        assert spread(a[s, :min(n, 60)], logits[s, :min(n, 60)]) < 0.05
        if n > 60:
            assert spread(b[s, :n - 60], logits[s, 60:n]) < 0.05
    for c in whole.caches + parts.caches:
        assert c.read_status() == (0, 0)


def test_steps_in_a_graph_are_the_steps():
    tokens = prompts()
    eager, graphed = model(), model()
    for m in (eager, graphed):
        m.forward(tokens[:, :150].contiguous())
    graph, at = graphed.capture_step()
    at.copy_(tokens[:, 150:151])
    now = tokens[:, 150:151].clone()
    for _ in range(20):
        graph.replay()
        now = eager.forward(now).argmax(-1)
        assert torch.equal(now, at)
    assert torch.equal(eager.lengths, graphed.lengths) and eager.lengths.tolist() == [170] * 3


def test_all_pages_selected_is_all_pages():
    tokens = prompts()
    dense, some, few = model(), model(), model()
    for m in (dense, some, few):
        m.forward(tokens[:, :199].contiguous())
    last = tokens[:, 199:].contiguous()
    want = dense.forward(last)
    assert spread(some.forward(last, keep=7), want) < 0.02            # 200 tokens are seven pages
    assert 1e-4 < spread(few.forward(last, keep=3), want)             # three of them are something else
