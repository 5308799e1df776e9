"""Models whose softmax layers cap their scores, bias them by distance, keep packed documents apart, and decode from pages: training, generation and beam search through the
framework's own paths."""
import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.config.model_config import ModelConfig, ParallelConfig, TrainConfig
from linear_moe_b200.infer import generation as G
from linear_moe_b200.infer.paged_cache import PagedCache
from linear_moe_b200.models.transformer import CausalLM

gpu = pytest.mark.gpu
EOD = 63


def config(**kw):
    base = dict(base_model="llama3", num_layers=2, hidden_size=128, num_attention_heads=4, num_query_groups=2, ffn_hidden_size=256, vocab_size=64)
    return ModelConfig(**{**base, **kw})


def model(device="cpu", **kw):
    m = CausalLM(config(**kw), device=device).to(device).eval()
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "word_embeddings" in n or "output_layer" in n:
                p.mul_(20.0)                                  # logits far enough apart that rounding decides nothing
            elif "linear_qkv" in n or "linear_proj" in n:
                p.mul_(8.0)                                   # scores of the size of the caps, and attention that matters beside the stream
    return m


def documents(device="cpu", rows=2, T=40, seed=0):
    gen = torch.Generator().manual_seed(seed)
    tok = torch.randint(0, EOD, (rows, T), generator=gen)
    for b in range(rows):
        tok[b, torch.randperm(T - 1, generator=gen)[:3]] = EOD
    return tok.to(device)


KINDS = [dict(), dict(attn_logit_softcapping=2.0), dict(position_embedding_type="alibi"), dict(attn_logit_softcapping=2.0, position_embedding_type="alibi", sliding_window=7)]


@pytest.mark.parametrize("kw", KINDS)
def test_documents_are_apart(kw):
    """A packed sequence gives the logits of its documents by themselves."""
    m, tok = model(**kw), documents()
    first = ops.document_first(tok, EOD)
    with torch.no_grad():
        got = m(tok, key_first=first, positions=torch.arange(tok.shape[1]) - first)
        for b in range(tok.shape[0]):
            ends = (tok[b] == EOD).nonzero()[:, 0].add(1).tolist() + [tok.shape[1]]
            at = 0
            for e in ends:
                if e > at:
                    assert torch.allclose(got[b, at:e], m(tok[b:b + 1, at:e])[0], atol=1e-4)
                at = e
        assert not torch.allclose(got, m(tok), atol=1e-2)


def test_capped_and_biased_scores_change_the_model():
    tok = documents()
    with torch.no_grad():
        plain = model()(tok)
        for kw in KINDS[1:]:
            assert not torch.allclose(plain, model(**kw)(tok), atol=1e-2)


def test_slopes():
    assert ops.alibi_slopes(8).tolist() == [2.0 ** -(i + 1) for i in range(8)]
    assert torch.allclose(ops.alibi_slopes(12)[8:], torch.tensor([2.0 ** -(0.5 + i) for i in range(4)]))
    assert ops.alibi_slopes(1).tolist() == [2.0 ** -8]


def test_configuration():
    for kw in (dict(attn_logit_softcapping=0.0), dict(base_model="deepseek_v2", attn_logit_softcapping=5.0), dict(base_model="deepseek_v2", position_embedding_type="alibi")):
        with pytest.raises(ValueError):
            config(**kw)
    from linear_moe_b200.config.arguments import parse_args
    _, cfg, _, tc = parse_args("--attn-logit-softcapping 50 --position-embedding-type alibi --reset-attention-mask --reset-position-ids".split())
    assert cfg.attn_logit_softcapping == 50.0 and cfg.position_embedding_type == "alibi" and tc.reset_attention_mask and tc.reset_position_ids
    tok = documents()
    m = model()
    with pytest.raises(ValueError):
        m(tok, key_first=ops.document_first(tok, EOD), caches=m.new_cache())
    hybrid = model(use_la_module=True, la_module="retention", layer_type_list="LN")
    with pytest.raises(ValueError):
        hybrid(tok, key_first=ops.document_first(tok, EOD))


@pytest.mark.parametrize("recompute", [None, "full"])
def test_training_on_packed_documents(recompute):
    """The trainer's step with the reset flags has the gradients of a step over the documents one by one."""
    from linear_moe_b200.data.datasets import SyntheticTokenDataset
    from linear_moe_b200.train.loop import Trainer

    class Packed(SyntheticTokenDataset):
        def __getitem__(self, i):
            row = super().__getitem__(i)
            row["text"] = row["text"].clone()
            row["text"][[7, 8, 20]] = EOD
            return row

        def __getitems__(self, idx):
            return [self[i] for i in idx]
    cfg = config(attn_logit_softcapping=3.0, recompute_granularity=recompute, recompute_method="uniform" if recompute else None)
    tc = TrainConfig(seq_length=32, micro_batch_size=2, global_batch_size=2, train_iters=1, eod_token=EOD, reset_attention_mask=True, reset_position_ids=True)
    tr = Trainer(cfg, ParallelConfig(), tc, device=torch.device("cpu"), dataset=Packed(64, 32, seed=1))
    batch = next(tr.data_iter)
    tr.model.train()
    out, loss_fn = tr.forward_step(batch, tr.model, None)
    got = torch.autograd.grad(loss_fn(out)[0], list(tr.model.parameters()))
    total = 0.0
    for b in range(2):
        tok, lab = batch["tokens"][b], batch["labels"][b]
        ends = (tok == EOD).nonzero()[:, 0].add(1).tolist() + [32]
        at = 0
        for e in ends:
            if e > at:
                total = total + tr.model(tok[None, at:e], lab[None, at:e]).sum()
            at = e
    want = torch.autograd.grad(total / batch["loss_mask"].sum(), list(tr.model.parameters()))
    for g, w in zip(got, want):
        assert (g - w).norm() <= 1e-4 * w.norm() + 1e-8
    assert torch.isfinite(torch.as_tensor(float(tr.train_step()["lm loss"])))


def test_trainer_refusals():
    from linear_moe_b200.train.loop import Trainer
    tc = dict(seq_length=32, micro_batch_size=1, global_batch_size=1, train_iters=1)
    with pytest.raises(ValueError, match="end-of-document"):
        Trainer(config(), ParallelConfig(), TrainConfig(reset_attention_mask=True, **tc), device=torch.device("cpu"))
    with pytest.raises(ValueError, match="softmax layers"):
        Trainer(config(use_la_module=True, la_module="gla", layer_type_list="LN"), ParallelConfig(), TrainConfig(reset_position_ids=True, eod_token=1, **tc),
                device=torch.device("cpu"))


MODELS = [dict(), dict(attn_logit_softcapping=2.0), dict(position_embedding_type="alibi", sliding_window=20), dict(qk_layernorm=True, rotary_percent=0.5),
          dict(use_la_module=True, la_module="retention", layer_type_list="LN"), dict(use_la_module=True, la_module="gla", layer_type_list="LL")]


def prompts(device="cpu", rows=2, P=9, L=90, seed=2):
    gen = torch.Generator().manual_seed(seed)
    base = torch.zeros(rows, L, dtype=torch.long)
    base[:, :P + 3] = torch.randint(0, EOD, (rows, P + 3), generator=gen)
    return base.to(device), torch.tensor([P, P + 3][:rows] + [P] * (rows - 2), device=device)


@pytest.mark.parametrize("kw", MODELS)
def test_generation_from_pages(kw):
    """Greedy tokens and their log-probabilities from pages are those from the dense cache, over a page's border."""
    m = model(**kw)
    base, lengths = prompts()
    a = G.generate_tokens(m, base.clone(), lengths, top_k=1, return_log_probs=True)
    b = G.generate_tokens(m, base.clone(), lengths, top_k=1, return_log_probs=True, paged=True)
    assert torch.equal(a[0], b[0]) and torch.allclose(a[2], b[2], atol=1e-3)


@pytest.mark.parametrize("kw", MODELS)
def test_beam_search_from_pages(kw):
    """Beams and scores from pages and reordered states are those of beams that are run again from their first token."""
    m = model(**kw)
    for P, n in ((3, 6), (62, 5), (64, 4)):
        prompt = prompts(P=P, L=P + 3)[0][:1, :P]
        a, sa = G.beam_search(m, prompt, 4, n, EOD, num_return=4)
        b, sb = G.beam_search(m, prompt, 4, n, EOD, num_return=4, paged=True)
        assert torch.equal(a, b) and torch.allclose(sa, sb, atol=1e-3)


def test_pages_of_beams():
    """Shared pages, copies where a row writes, pages given back: rows of random reorderings hold what their history wrote."""
    m = model(num_layers=1, kv_channels=8, hidden_size=32)
    cache = PagedCache(m, 4, 300, live=1)
    hist = [[]]
    gen = torch.Generator().manual_seed(0)
    for step in range(280):
        cache.advance(1)
        c, n = cache[0], len(hist)
        assert c["table"].shape[0] == c["lengths"].shape[0] == n and (c["lengths"] == step + 1).all()
        for b in range(n):
            page = int(c["table"][b, step // 64])
            assert cache.uses[page] == 1                       # nobody else's page is written
            c["k_pages"][page, step % 64], c["v_pages"][page, step % 64] = float(step * 4 + b), -float(step * 4 + b)
            hist[b] = hist[b] + [step * 4 + b]
        for b in range(n):
            at = c["table"][b, : step // 64 + 1].long()
            rows = c["k_pages"][at].flatten(0, 1)[: step + 1, 0, 0]
            assert rows.tolist() == hist[b] and (c["v_pages"][at].flatten(0, 1)[: step + 1, 0, 0] == -rows).all()
        parents = torch.randint(0, n, (4 if step != 100 else 2,), generator=gen).tolist()
        cache.reorder(parents)
        hist = [list(hist[p]) for p in parents]
        assert sum(cache.uses.values()) == sum(len(p) for p in cache.owned)
        assert len(cache.uses) + len(cache.free) == c["k_pages"].shape[0] and not set(cache.uses) & set(cache.free)
    for bad in ([], [4], [-1], [0] * 5):
        with pytest.raises(ValueError):
            cache.reorder(bad)
    with pytest.raises(ValueError):
        cache.advance(21)


def test_caches_that_are_not_paged():
    mla = CausalLM(ModelConfig(base_model="deepseek_v2", num_layers=1, hidden_size=64, num_attention_heads=2, ffn_hidden_size=64, vocab_size=64, q_lora_rank=None,
                               kv_lora_rank=16, qk_nope_head_dim=16, qk_rope_head_dim=8, v_head_dim=16)).eval()
    with pytest.raises(ValueError):
        PagedCache(mla, 1, 10)
    with pytest.raises(ValueError):
        G.generate_tokens(mla, *prompts(), paged=True)
    mom = model(use_la_module=True, la_module="mom_gla", layer_type_list="LN")
    assert not G.can_page_beams(mom)
    with pytest.raises(ValueError):
        G.beam_search(mom, prompts()[0][:1, :4], 2, 3, EOD, paged=True)


# ---- on the GPU -----------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("kw", KINDS)
def test_training_step_on_gpu(kw, monkeypatch):
    """Gradients of a bf16 model over packed documents, with the kernels and with the eager definition of attention in their place, against the same model in fp32 on the CPU: all
    other roundings are the same ones, so the kernels' model may be off by as much as the other one, in other directions; twice that and a rounding (2^-8) is the bound."""
    from linear_moe_b200.ref import ops as R
    m = model(params_dtype=torch.bfloat16, device="cuda", hidden_size=256, vocab_size=512, **kw).train()
    c = CausalLM(m.cfg.replace(params_dtype=torch.float32)).train()
    c.load_state_dict({k: v.float().cpu() for k, v in m.state_dict().items()})
    tok = documents(rows=3, T=300)
    lab = tok.roll(-1, 1)

    def step(m, tok, lab):
        first = ops.document_first(tok, EOD)
        loss = m(tok, lab, key_first=first, positions=torch.arange(tok.shape[1], device=tok.device) - first).float().mean()
        return [g.float().cpu() for g in torch.autograd.grad(loss, list(m.parameters()))]
    got, want = step(m, tok.cuda(), lab.cuda()), step(c, tok, lab)
    monkeypatch.setattr(ops, "scored_attention", R.softmax_attention)
    eager = step(m, tok.cuda(), lab.cuda())
    for (n, _), g, e, w in zip(m.named_parameters(), got, eager, want):
        assert (g - w).norm() <= 2 * (e - w).norm() + 2.0 ** -8 * w.norm(), n
        assert (e - w).norm() < 0.3 * w.norm(), n


@gpu
@pytest.mark.parametrize("kw", MODELS)
def test_captured_generation_from_pages(kw):
    """Replayed and eager steps from pages have the same bits.  Steps from pages and from the dense cache run the same roundings but those of attention: the first are as near
    to an fp32 model as the others, or within twice that and a rounding (2^-8)."""
    m = model(params_dtype=torch.bfloat16, device="cuda", hidden_size=256, vocab_size=512, **kw)
    base, lengths = prompts("cuda")
    a = G.generate_tokens(m, base.clone(), lengths, top_k=1, return_log_probs=True, paged=True)
    b = G.generate_tokens(m, base.clone(), lengths, top_k=1, return_log_probs=True, paged=True, cuda_graph=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    c = CausalLM(m.cfg.replace(params_dtype=torch.float32)).eval()
    c.load_state_dict({k: v.float().cpu() for k, v in m.state_dict().items()})
    ids, B, P = a[0], 2, 9
    with torch.no_grad():
        full = c(ids.cpu()).cuda()
        cache, dense = PagedCache(m, B, ids.shape[1]), m.new_cache()
        cache.advance(P)
        m(ids[:, :P], caches=cache)
        m(ids[:, :P], caches=dense)
        step, off = None, torch.zeros(2)
        for t in range(P, ids.shape[1]):
            cache.advance(1)
            tok = ids[:, t:t + 1].contiguous()
            other = m(tok, caches=dense, position_offset=t)
            if t < P + 2:
                out = m(tok, caches=cache, position_offset=t)
            else:
                if step is None:
                    assert G.GraphedDecodeStep.supported(m, cache, tok.device)
                    step = G.GraphedDecodeStep(m, cache, B, tok.device)
                out = step(tok)
                assert step.graph is not None
            off += torch.stack([(x[:, 0].float() - full[:, t]).norm() / full[:, t].norm() for x in (out, other)]).cpu()
        off /= ids.shape[1] - P
        assert off[0] <= 2 * off[1] + 2.0 ** -8 and off[1] < 0.2, off
    from linear_moe_b200.ops import gemm
    gemm.check_error()


@gpu
@pytest.mark.parametrize("kw", MODELS)
def test_beam_search_on_gpu(kw):
    """fp32 beams from pages against beams run again from their first token."""
    if kw.get("use_la_module"):
        kw = {**kw, "hidden_size": 256}                        # 64-wide heads, which the linear kernels take
    m = model(device="cuda", vocab_size=500, **kw)
    prompt = prompts("cuda", P=62, L=80)[0][:1, :62]
    a, sa = G.beam_search(m, prompt, 5, 8, EOD, num_return=5)
    b, sb = G.beam_search(m, prompt, 5, 8, EOD, num_return=5, paged=True)
    assert torch.equal(a, b) and torch.allclose(sa, sb, atol=2e-3)


@gpu
def test_train_then_generate_then_search():
    """The operators as they are used together: steps on packed documents, then greedy tokens from a captured step, then a beam search whose first beam is at least as likely."""
    from linear_moe_b200.ops import gemm
    torch.manual_seed(0)
    m = model(params_dtype=torch.bfloat16, device="cuda", hidden_size=256, vocab_size=512, attn_logit_softcapping=20.0).train()
    opt = torch.optim.SGD(m.parameters(), lr=0.05)
    for seed in range(3):
        tok = documents("cuda", 4, 257, seed)
        loss = m(tok[:, :-1], tok[:, 1:], key_first=ops.document_first(tok[:, :-1], EOD)).float().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        assert torch.isfinite(loss) and all(torch.isfinite(p.grad).all() for p in m.parameters())
    m.eval()
    P, n = 30, 40
    prompt = documents("cuda", 1, P)
    base = torch.cat([prompt, torch.zeros(1, n, dtype=torch.long, device="cuda")], 1)
    out, _, lp = G.generate_tokens(m, base, torch.tensor([P], device="cuda"), top_k=1, return_log_probs=True, paged=True, cuda_graph=True)
    beams, scores = G.beam_search(m, prompt, 4, n, eod=-1, length_penalty=0.0, num_return=4, paged=True)
    assert beams.shape == (4, P + n) and (scores[:-1] >= scores[1:]).all() and torch.equal(beams[:, :P], prompt.expand(4, P))
    own = G.score_tokens(m, beams)[:, P - 1:].sum(-1)
    assert torch.allclose(own, scores, rtol=0.03, atol=1.0)
    gemm.check_error()
