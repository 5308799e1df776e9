"""What a beam search may take for a state with a row per beam."""
import pytest
import torch

from linear_moe_b200.config.model_config import LA_MODULES
from linear_moe_b200.infer import generation as G
from linear_moe_b200.infer.paged_cache import PagedCache
from test_softmax_layers import EOD, model, prompts


def hybrid(la="retention"):
    return model(use_la_module=True, la_module=la, layer_type_list="LN", hidden_size=256)


def keep(m, make):
    """A linear layer that keeps one more tensor."""
    mixer = m.decoder.layers[0]._mixer()
    inner = mixer.forward

    def forward(h, cache=None, **kw):
        out = inner(h, cache=cache, **kw)
        if cache is not None:
            cache["kept"] = make(h)
        return out
    mixer.forward = forward
    return m


@pytest.mark.parametrize("make,ok", [(lambda h: h[:, -1].detach(), True), (lambda h: h[:1].mean((0, 1)).detach()[None], False), (lambda h: h[:, -1].t().detach(), False),
                                     (lambda h: torch.tensor(1.0), False)])
def test_states_without_a_row_per_beam_are_refused(make, ok):
    """A leading dimension of one is a row of the single prompt, or something else altogether."""
    prompt = prompts()[0][:1, :5]
    m = keep(hybrid(), make)
    if ok:
        a, b = G.beam_search(m, prompt, 3, 4, EOD, paged=True), G.beam_search(hybrid(), prompt, 3, 4, EOD)
        assert torch.equal(a[0], b[0])
    else:
        with pytest.raises(ValueError, match="follow a beam"):
            G.beam_search(m, prompt, 3, 4, EOD, paged=True)
    G.beam_search(keep(hybrid(), lambda h: h[:, -1].detach()), prompt, 1, 4, EOD, paged=True)


@pytest.mark.parametrize("la", [x for x in LA_MODULES if not x.startswith("mom_")])
def test_linear_layers_keep_a_row_per_request(la):
    """Every linear layer's states, reordered, go on as the rows that they came from."""
    m = hybrid(la)
    tok = prompts(rows=3, P=7, L=12)[0]
    with torch.no_grad():
        cache = PagedCache(m, 3, 12)
        cache.advance(6)
        m(tok[:, :6], caches=cache)
        assert cache.reorderable()
        want = m(torch.cat([tok[[2, 0, 2], :6], tok[:, 6:7]], 1))[:, -1]
        cache.reorder([2, 0, 2])
        cache.advance(1)
        got = m(tok[:, 6:7], caches=cache, position_offset=6)[:, -1]
        assert torch.allclose(got, want, atol=2e-3)
