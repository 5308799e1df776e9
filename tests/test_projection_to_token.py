"""From a softmax layer's projection to the next token through the framework's own paths: heads in one pass, pages of 4 bits a number, tokens by one random number each."""
import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.infer import generation as G
from linear_moe_b200.infer.paged_cache import PagedCache
from linear_moe_b200.models.transformer import CausalLM
from linear_moe_b200.ops import gemm
from linear_moe_b200.ref import ops as R
from test_softmax_layers import EOD, config, documents, model, prompts

gpu = pytest.mark.gpu
KINDS = [dict(), dict(qk_layernorm=True), dict(qk_layernorm=True, rotary_percent=0.5, rotary_interleaved=True), dict(qk_layernorm=True, position_embedding_type="alibi", attn_logit_softcapping=2.0),
         dict(qk_layernorm=True, use_la_module=True, la_module="retention", layer_type_list="LN"), dict(add_qkv_bias=True, num_query_groups=1)]


def fused(m):
    """The same model with its heads in one pass."""
    f = CausalLM(m.cfg.replace(fused_qkv_heads=True), device=str(next(m.parameters()).device)).to(next(m.parameters()).device)
    f.load_state_dict(m.state_dict())
    return f.train(m.training)


# ---- heads in one pass --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", KINDS)
def test_heads_in_one_pass(kw):
    """fp32: the same logits and gradients but for the order of a few roundings, with and without packed documents, and the same greedy tokens from either cache."""
    m, tok = model(**kw), documents()
    f = fused(m)
    cases = [dict()]
    if not kw.get("use_la_module"):
        first = ops.document_first(tok, EOD)
        cases.append(dict(key_first=first, positions=torch.arange(tok.shape[1]) - first))
    for c in cases:
        a, b = (x(tok, tok.roll(-1, 1), **c).sum() for x in (m, f))
        assert torch.allclose(a, b, rtol=1e-4)
        for (n, _), x, y in zip(m.named_parameters(), torch.autograd.grad(a, list(m.parameters())), torch.autograd.grad(b, list(f.parameters()))):
            assert (x - y).norm() <= 1e-4 * x.norm() + 1e-7, n
    base, lengths = prompts()
    for paged in (False, True):
        a, b = (G.generate_tokens(x, base.clone(), lengths, top_k=1, return_log_probs=True, paged=paged) for x in (m, f))
        assert torch.equal(a[0], b[0]) and torch.allclose(a[2], b[2], atol=1e-3)


@gpu
@pytest.mark.parametrize("kw", KINDS)
def test_heads_in_one_pass_on_gpu(kw):
    """Gradients of a bf16 model against the same model in fp32 on the CPU: one rounding in the place of three, so the fused model may be off by as much as the other one, in other directions; twice that
    and a rounding (2^-8) is the bound."""
    if kw.get("use_la_module"):
        kw = {**kw, "num_attention_heads": 4}
    m = model(params_dtype=torch.bfloat16, device="cuda", hidden_size=256, vocab_size=512, **kw).train()
    f = fused(m)
    c = CausalLM(m.cfg.replace(params_dtype=torch.float32)).train()
    c.load_state_dict({k: v.float().cpu() for k, v in m.state_dict().items()})
    tok = documents(rows=3, T=300)
    lab = tok.roll(-1, 1)

    def step(x):
        dev = next(x.parameters()).device
        return [g.float().cpu() for g in torch.autograd.grad(x(tok.to(dev), lab.to(dev)).float().mean(), list(x.parameters()))]
    got, other, want = step(f), step(m), step(c)
    for (n, _), g, e, w in zip(m.named_parameters(), got, other, want):
        assert (g - w).norm() <= 2 * (e - w).norm() + 2.0 ** -8 * w.norm(), n
    gemm.check_error()


# ---- pages of 4 bits ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device,dtype", [("cpu", torch.float32), pytest.param("cuda", torch.bfloat16, marks=gpu), pytest.param("cuda", torch.float32, marks=gpu)])
def test_a_layer_on_pages_of_four_bits(device, dtype):
    """A prompt, a portion behind it and single tokens: attention over what the pages give back (a portion's own rows as they were)."""
    m = model(device=device, num_layers=1, params_dtype=dtype, qk_layernorm=True, fused_qkv_heads=True)
    att = m.decoder.layers[0]._mixer()
    seen = []
    orig = ops.qkv_heads

    def watch(*a, **kw):
        seen.append(orig(*a, **kw))
        return seen[-1]
    cache = PagedCache(m, 2, 200, bits=4)
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(2, 150, 128, generator=gen).to(device, dtype)
    at, tol = 0, 1e-5 if dtype == torch.float32 else 2.0 ** -7         # bf16: attention and what comes behind it round once each on either way
    with pytest.MonkeyPatch.context() as mp, torch.no_grad():
        mp.setattr(ops, "qkv_heads", watch)
        for n in (70, 63, 1, 1, 1):
            cache.advance(n)
            out = att(x[:, at:at + n], cache=cache[0], position_offset=at)
            q, k, v = seen[-1]
            old = ops.read_rows_int4(cache[0]["k_pages"], cache[0]["v_pages"], cache[0]["table"], cache[0]["lengths"], at + n, att.D, torch.float32)
            k, v = (torch.cat([o[:, :at], t.float()], 1) if n > 1 else o for o, t in zip(old, (k, v)))
            want = att.linear_proj(R.softmax_attention(q.float(), k, v, None, True, at).to(dtype).reshape(2, n, -1))
            assert (out.float() - want.float()).norm() <= tol * want.float().norm()
            # what is stored is within half a size of what went in
            for o, t in zip(old, seen[-1][1:]):
                span = t.float().unflatten(-1, (-1, 32))
                span = (span.amax(-1) - span.amin(-1) + 2.0 ** -7 * span.amin(-1).abs()) / 15 * 1.01
                assert ((o[:, at:] - t.float()).unflatten(-1, (-1, 32)).abs().amax(-1) <= span / 2 + 1e-6).all()
            at += n
    gemm.check_error()


def test_pages_of_four_bits_of_beams():
    """Beams share pages and get copies of the last one; one beam is greedy decoding."""
    m = model(qk_layernorm=True)
    prompt = prompts(P=62, L=70)[0][:1, :62]
    for n in (4, 6):
        beams, scores = G.beam_search(m, prompt, 4, n, EOD, num_return=4, paged=True, cache_bits=4)
        assert beams.shape[0] == 4 and (scores[:-1] >= scores[1:]).all() and torch.equal(beams[:, :62], prompt.expand(4, -1))
    one, _ = G.beam_search(m, prompt, 1, 6, eod=-1, paged=True, cache_bits=4)
    base = torch.cat([prompt, torch.zeros(1, 6, dtype=torch.long)], 1)
    assert torch.equal(one, G.generate_tokens(m, base, torch.tensor([62]), top_k=1, paged=True, cache_bits=4)[0])


def test_refusals():
    m = model()
    base, lengths = prompts()
    for kw in (dict(cache_bits=4), dict(cache_bits=8, paged=True), dict(min_p=1.5), dict(min_p=-0.1)):
        with pytest.raises(ValueError):
            G.generate_tokens(m, base.clone(), lengths, top_k=1, **kw)
    with pytest.raises(ValueError):
        G.beam_search(m, base[:1, :4], 2, 3, EOD, cache_bits=4)
    with pytest.raises(ValueError):
        PagedCache(model(kv_channels=24, hidden_size=96), 1, 10, bits=4)
    from linear_moe_b200.config.arguments import parse_args
    args, cfg, _, _ = parse_args("--fused-qkv-heads --qk-layernorm --paged-kv-cache --kv-cache-bits 4 --min-p 0.05 --fused-sampling".split())
    assert cfg.fused_qkv_heads and args.kv_cache_bits == 4 and args.min_p == 0.05 and args.fused_sampling
    assert not config().fused_qkv_heads


# ---- tokens by one random number each -----------------------------------------------------------------------------------------------
def test_sampled_generation():
    """The same generator gives the same tokens; each is the one that its random number falls to."""
    m = model()
    base, lengths = prompts(L=40)
    kw = dict(top_k=8, top_p=0.9, min_p=0.01, temperature=1.3)
    out = [G.generate_tokens(m, base.clone(), lengths, generator=torch.Generator().manual_seed(s), fused_sampling=True, **kw)[0] for s in (1, 1, 2)]
    assert torch.equal(out[0], out[1]) and not torch.equal(out[0], out[2])
    greedy = G.generate_tokens(m, base.clone(), lengths, top_k=1)[0]
    assert torch.equal(G.generate_tokens(m, base.clone(), lengths, top_k=1, fused_sampling=True)[0], greedy)
    gen = torch.Generator().manual_seed(1)
    ids, P = out[0], int(lengths.min())
    with torch.no_grad():
        logits = m(ids)
    for t in range(P, 40):
        draw = torch.rand(2, generator=gen)
        want = ops.sample_tokens(logits[:, t - 1], draw, kw["temperature"], kw["top_k"], kw["top_p"], kw["min_p"])[0]
        assert all(int(want[b]) == int(ids[b, t]) for b in range(2) if t >= int(lengths[b]))


def test_a_padded_vocabulary_is_not_drawn_from():
    logits = torch.zeros(4, 80)
    logits[:, 64:] = 50.0
    for s in range(20):
        assert int(G.sample_fused(logits, vocab_size=64, generator=torch.Generator().manual_seed(s)).max()) < 64


def test_requests_with_min_p():
    from fastapi.testclient import TestClient
    from linear_moe_b200.data.tokenizer import NullTokenizer
    from linear_moe_b200.infer.server import build_app
    m, tok = model(), NullTokenizer(64)
    with TestClient(build_app(m, tok, paged=True, cache_bits=4)) as c:
        body = {"prompts": ["1 2 3 4"], "tokens_to_generate": 6, "min_p": 0.1, "temperature": 2.0, "random_seed": 3}
        a, b = (c.put("/api", json=body) for _ in range(2))
        assert a.status_code == 200 and a.json() == b.json()
        with torch.no_grad():
            want = G.generate_and_post_process(m, tok, body["prompts"], 6, min_p=0.1, temperature=2.0, random_seed=3, paged=True, cache_bits=4)
        assert a.json()["tokens"] == want[1]
        assert c.put("/api", json={**body, "min_p": 2}).status_code == 400
        assert c.put("/api", json={"prompts": ["1 2 3 4"], "tokens_to_generate": 4, "beam_width": 2}).status_code == 200


# ---- together -------------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("kw", KINDS)
def test_captured_steps(kw):
    """Sampled tokens from a captured step on pages of 4 bits are those of eager steps, and so are their log-probabilities."""
    m = model(params_dtype=torch.bfloat16, device="cuda", hidden_size=256, vocab_size=512, fused_qkv_heads=True, **kw)
    base, lengths = prompts("cuda")
    out = [G.generate_tokens(m, base.clone(), lengths, return_log_probs=True, paged=True, cache_bits=4, cuda_graph=graph, top_k=50, top_p=0.95, min_p=0.001, temperature=0.9, fused_sampling=True,
                             generator=torch.Generator("cuda").manual_seed(5)) for graph in (False, True)]
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][2], out[1][2])


@gpu
def test_train_then_sample():
    """The operators as they are used together: steps on packed documents, then tokens sampled from captured steps on pages of 4 bits."""
    torch.manual_seed(0)
    m = model(params_dtype=torch.bfloat16, device="cuda", hidden_size=256, vocab_size=512, qk_layernorm=True, fused_qkv_heads=True).train()
    opt = torch.optim.SGD(m.parameters(), lr=0.05)
    for seed in range(3):
        tok = documents("cuda", 4, 257, seed)
        first = ops.document_first(tok[:, :-1], EOD)
        loss = m(tok[:, :-1], tok[:, 1:], key_first=first, positions=torch.arange(256, device="cuda") - first).float().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        assert torch.isfinite(loss) and all(torch.isfinite(p.grad).all() for p in m.parameters())
    m.eval()
    P, n = 30, 100
    base = torch.cat([documents("cuda", 3, P), torch.zeros(3, n, dtype=torch.long, device="cuda")], 1)
    out, _, lp = G.generate_tokens(m, base, torch.full((3,), P, device="cuda"), return_log_probs=True, paged=True, cache_bits=4, cuda_graph=True, top_p=0.9, fused_sampling=True,
                                   generator=torch.Generator("cuda").manual_seed(1))
    assert out.shape == (3, P + n) and torch.isfinite(lp).all() and int(out.max()) < 512
    gemm.check_error()


def test_requests_with_top_k_and_top_p():
    """Together where the tokens are drawn by one random number each: a server started with fused sampling, or a request with a min_p."""
    from fastapi.testclient import TestClient
    from linear_moe_b200.data.tokenizer import NullTokenizer
    from linear_moe_b200.infer.server import build_app
    m, tok = model(), NullTokenizer(64)
    body = {"prompts": ["1 2 3 4"], "tokens_to_generate": 6, "top_k": 8, "top_p": 0.8, "temperature": 2.0, "random_seed": 3}
    for fused in (False, True):
        with TestClient(build_app(m, tok, fused_sampling=fused)) as c:
            for extra in (dict(), dict(min_p=0.0), dict(min_p=0.05)):
                got = c.put("/api", json={**body, **extra})
                if not fused and not extra.get("min_p"):
                    assert got.status_code == 400 and "top_k and top_p" in got.json()["message"]
                    continue
                with torch.no_grad():
                    want = G.generate_and_post_process(m, tok, body["prompts"], 6, top_k_sampling=8, top_p_sampling=0.8, temperature=2.0, random_seed=3, fused_sampling=fused, **extra)
                assert got.status_code == 200 and got.json()["tokens"] == want[1]
            assert c.put("/api", json={**body, "min_p": "x"}).status_code == 400


@pytest.mark.parametrize("one_pass", [False, True])
def test_single_tokens_from_pages_take_their_own_positions(one_pass):
    """A layer's step over pages turns by the pages' lengths, whatever tables come along; elsewhere these have a row for every token."""
    m = model(num_layers=1, fused_qkv_heads=one_pass)
    att = m.decoder.layers[0]._mixer()
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(2, 12, 128, generator=gen)
    tables = att.rope.get(5, 0, x.device)
    with torch.no_grad():
        out = []
        for rotary in (None, tables):
            cache = PagedCache(m, 2, 40)
            cache.advance(11)
            att(x[:, :11], cache=cache[0])
            cache.advance(1)
            out.append(att(x[:, 11:], cache=cache[0], position_offset=11, rotary=rotary))
        assert torch.equal(*out)
        with pytest.raises(ValueError, match="positions for"):
            att(x, rotary=tables)
