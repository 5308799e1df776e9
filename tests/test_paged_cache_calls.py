"""Calls of a model on a paged cache that has no room for them."""
import pytest
import torch

from linear_moe_b200.infer.paged_cache import PagedCache
from test_softmax_layers import documents, model


@pytest.mark.parametrize("T", [1, 5])
def test_no_call_ahead_of_its_room(T):
    m, tok = model(), documents(T=12)
    cache = PagedCache(m, 2, 70)
    with torch.no_grad():
        with pytest.raises(ValueError, match="advance"):
            m(tok[:, :T], caches=cache)
        cache.advance(T)
        m(tok[:, :T], caches=cache)
        with pytest.raises(ValueError, match="advance"):
            m(tok[:, T:T + 3], caches=cache, position_offset=T)
        cache.advance(3)
        got = m(tok[:, T:T + 3], caches=cache, position_offset=T)
        assert torch.allclose(got, m(tok[:, :T + 3])[:, T:], atol=1e-3)
        with pytest.raises(ValueError, match="advance"):
            m(tok[:, T + 3:T + 4], caches=cache, position_offset=T + 3)


def test_rows_are_the_cache_s():
    m, tok = model(), documents(rows=3)
    cache = PagedCache(m, 3, 70, live=2)
    cache.advance(4)
    with torch.no_grad():
        with pytest.raises(ValueError, match="rows"):
            m(tok[:, :4], caches=cache)
        m(tok[:2, :4], caches=cache)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_pages_have_the_layers_type(device):
    """A model built in one type and brought to another one."""
    from linear_moe_b200.infer import generation as G
    from test_softmax_layers import EOD, prompts
    m = model(device, params_dtype=torch.bfloat16).float()
    base, lengths = prompts(device, L=20)
    a, b = (G.generate_tokens(m, base.clone(), lengths, top_k=1, paged=p)[0] for p in (False, True))
    assert torch.equal(a, b)
    a, b = (G.beam_search(m, base[:1, :9], 3, 5, EOD, paged=p)[0] for p in (False, True))
    assert torch.equal(a, b)
