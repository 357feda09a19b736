"""Capturing a decoder's step leaves its caches as they were, bit for bit."""
import pytest
import torch

from test_cached_decoding_gpu import model, prompts

pytestmark = pytest.mark.gpu


def contents(m):
    return [t.clone() for c in m.caches for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale, c.bounds.view(torch.uint8))] + [m.lengths.clone()]


@pytest.mark.parametrize("keep", [0, 3])
@pytest.mark.parametrize("held", [1, 150, 159])
def test_capturing_a_step_appends_nothing(held, keep):
    m = model()
    tokens = prompts()
    m.forward(tokens[:, :held].contiguous())
    for c in m.caches:   # pages whose scales a token would enlarge, and whose bounds it would widen
        c.k_scale.mul_(2.0 ** -6), c.v_scale.mul_(2.0 ** -6)
        c.bounds.view(torch.uint8).zero_()
    before = contents(m)
    m.capture_step(keep)
    for a, b in zip(before, contents(m)):
        assert torch.equal(a, b)


def test_a_step_can_be_captured_when_the_sequences_are_full():
    m = model()
    m.lengths.fill_(m.table.shape[1] * 32)
    m.capture_step()
    assert all(c.read_status() == (0, 0) for c in m.caches)
