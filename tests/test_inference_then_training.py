"""A model that has run under torch.inference_mode is trained: what its layers keep from call to call must be fit for autograd."""
import pytest
import torch

from test_softmax_layers import documents, model


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kw", [dict(), dict(position_embedding_type="alibi"), dict(position_embedding_type="alibi", attn_logit_softcapping=5.0)])
def test_training_goes_on(device, kw):
    kw = dict(kw, params_dtype=torch.bfloat16, hidden_size=256) if device == "cuda" else kw
    m, other, tok = model(device, **kw), model(device, **kw), documents(device)
    other.load_state_dict(m.state_dict())
    with torch.inference_mode():
        m(tok)
    for layer in m.decoder.layers:
        slopes = layer._mixer()._slopes
        assert slopes is None or not slopes.is_inference()
    a, b = (torch.autograd.grad(x.train()(tok, tok.roll(-1, 1)).float().mean(), list(x.parameters())) for x in (m, other))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
