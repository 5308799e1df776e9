"""Rotary positions that a caller gives, of any size: a table of the sequence's length must not be what they index."""
import pytest
import torch

from linear_moe_b200 import ops
from test_softmax_layers import EOD, documents, model

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kw", [dict(), dict(rotary_percent=0.5, rotary_seq_len_interpolation_factor=2.0), dict(rotary_interleaved=True)])
def test_any_positions(device, kw):
    """Scores depend on differences of positions: moved all together, beyond the sequence or below zero, they give the same logits; the sequence's own give those without any."""
    m, tok = model(device, **kw), documents(device)
    at = torch.arange(tok.shape[1], device=device).expand_as(tok)
    with torch.no_grad():
        plain = m(tok)
        assert torch.equal(m(tok, positions=at), plain)
        for move in (40, 1000, -7):
            assert torch.allclose(m(tok, positions=at + move), plain, atol=5e-3)
        assert not torch.allclose(m(tok, positions=at * 3), plain, atol=1e-2)
        # one document of a packed pair goes on behind the other's positions
        first = ops.document_first(tok, EOD)
        a, b = m(tok, key_first=first, positions=at - first), m(tok, key_first=first, positions=at - first + 64 * (first > 0))
        assert torch.allclose(a, b, atol=5e-3)


def test_as_many_positions_as_tokens():
    m, tok = model(), documents()
    for bad in (torch.arange(40), torch.zeros(2, 39, dtype=torch.long), torch.zeros(1, 40, dtype=torch.long)):
        with pytest.raises(ValueError):
            m(tok, positions=bad)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_are_those_of_the_table(device):
    m, tok = model(device, recompute_granularity="full", recompute_method="uniform").train(), documents(device)
    at = torch.arange(tok.shape[1], device=device).expand_as(tok)
    a, b = (torch.autograd.grad(m(tok, tok.roll(-1, 1), positions=p).mean(), list(m.parameters())) for p in (at, None))
    assert all(torch.equal(x, y) or (x - y).norm() <= 1e-5 * y.norm() for x, y in zip(a, b))
