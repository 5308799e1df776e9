"""Operators of the softmax layers that are timed on their own, each through the call that a user makes.

* ``attention``  softmax attention whose scores are capped, biased by distance, or seen through a range of keys per query (documents
                 packed into a sequence, a prefix that sees itself whole, padding); ``train`` asks for the gradients too
* ``step``       the same attention for one new token of every request, over a paged cache; it stores the token's key and value
* ``beam``       one step of a beam search: the best continuations over beams and vocabulary, and the states of the beams in
                 their new order

``run`` makes the calls of :mod:`linear_moe_b200.ops` where ``own`` is true, and computes the plain form in 32 bits (candidates'
scores, which lie next to one another, in 64) where it is not.  ``exact`` is the definition in 64 bits.
"""
import math
import random

import torch

own = False
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # two short sequences of packed documents: the smallest training call, where the launches count
        dict(name="attention_train_130", kind="attention", B=2, T=130, ctx=0, H=4, HKV=2, D=64, dtype="bf16", mask="documents", mean=40, window=0, cap=30.0,
             slopes=False, train=True),
        # packed pretraining: documents of about 700 tokens in sequences of 4096, capped scores, 16 query heads on 4
        dict(name="attention_train_docs_2x4k", kind="attention", B=2, T=4096, ctx=0, H=16, HKV=4, D=128, dtype="bf16", mask="documents", mean=700, window=0,
             cap=50.0, slopes=False, train=True),
        # fine-tuning on prompts that see themselves whole, in a padded batch of an odd length, in fp16
        dict(name="attention_train_prefix_3x1531", kind="attention", B=3, T=1531, ctx=0, H=32, HKV=8, D=64, dtype="fp16", mask="prefix", mean=1200, window=0,
             cap=0.0, slopes=False, train=True),
        # long documents with a distance bias and a sliding window
        dict(name="attention_train_slopes_8k", kind="attention", B=1, T=8192, ctx=0, H=16, HKV=16, D=128, dtype="bf16", mask="documents", mean=5000,
             window=2048, cap=0.0, slopes=True, train=True),
        # the next portion of two prompts against what the cache holds, capped, with heads of 96
        dict(name="attention_prefill_777", kind="attention", B=2, T=777, ctx=2556, H=24, HKV=8, D=96, dtype="bf16", mask="causal", mean=0, window=0, cap=50.0,
             slopes=False, train=False),
        # one request at the beginning of its answer
        dict(name="step_1x300", kind="step", B=1, most=300, least=300, H=16, HKV=4, D=128, dtype="bf16", window=0, cap=0.0, slopes=False),
        # eight requests of different lengths, 64-wide heads, capped, in fp16
        dict(name="step_8x2k", kind="step", B=8, most=2048, least=77, H=32, HKV=8, D=64, dtype="fp16", window=0, cap=50.0, slopes=False),
        # two long contexts with few key heads: the cache's length is all there is to split
        dict(name="step_2x100k", kind="step", B=2, most=100001, least=60000, H=16, HKV=2, D=128, dtype="bf16", window=0, cap=0.0, slopes=True),
        # a full batch of long requests, capped
        dict(name="step_64x8k", kind="step", B=64, most=8192, least=1000, H=32, HKV=8, D=128, dtype="bf16", window=0, cap=50.0, slopes=False),
        # a single prompt with four beams and a small vocabulary
        dict(name="beam_1x4", kind="beam", N=1, K=4, V=32000, dtype="bf16", layers=2, H=4, D=64),
        # four prompts, an odd vocabulary and an odd number of beams
        dict(name="beam_4x5", kind="beam", N=4, K=5, V=50257, dtype="bf16", layers=4, H=8, D=128),
        # sixteen prompts with eight beams over the vocabulary of the 1B model, states of four of its layers
        dict(name="beam_16x8", kind="beam", N=16, K=8, V=128256, dtype="fp32", layers=4, H=16, D=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "step", "step", "beam"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    cap = rng.choice([0.0, 20.0, 50.0])
    if kind == "attention":
        HKV = rng.choice([1, 2, 4, 8])
        H, D = HKV * rng.choice([1, 2, 3, 4]), rng.choice([64, 64, 80, 96, 128, 128])
        mask, T = rng.choice(["documents", "documents", "prefix", "causal"]), _log(rng, 64, 4096)
        B = max(1, min(4, 6000 // T))
        ctx = _log(rng, 1, 4096) if mask == "causal" else 0
        return dict(kind=kind, B=B, T=T, ctx=ctx, H=H, HKV=HKV, D=D, dtype=dtype, mask=mask, mean=max(1, int(T * rng.uniform(0.05, 0.9))),
                    window=0 if mask == "prefix" else rng.choice([0, 0, _log(rng, 16, 2048)]), cap=cap, slopes=rng.random() < 0.3, train=rng.random() < 0.7)
    if kind == "step":
        B, HKV = _log(rng, 1, 48), rng.choice([1, 2, 4, 8])
        most = _log(rng, 64, min(65536, 400000 // B))
        return dict(kind=kind, B=B, most=most, least=max(1, int(most * rng.uniform(0.01, 1.0))), H=HKV * rng.choice([1, 3, 4, 8, 16]), HKV=HKV,
                    D=rng.choice([64, 96, 128, 128]), dtype=dtype, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), cap=cap, slopes=rng.random() < 0.3)
    N, K = _log(rng, 1, 16), rng.randint(2, 8)
    return dict(kind=kind, N=N, K=K, V=_log(rng, 2000, 128256), dtype=rng.choice(["bf16", "fp32"]), layers=rng.randint(1, 4), H=rng.choice([4, 8, 16]),
                D=rng.choice([64, 128]))


# ---- what follows from a case alone: the lengths that its seed only shuffles -----------------------------------------------------
def _documents(c):
    """Lengths of the documents of every sequence."""
    rng, rows = random.Random(c["T"] * 31 + c["mean"]), []
    for _ in range(c["B"]):
        left, row = c["T"], []
        while left > 0:
            n = min(left, max(1, int(rng.expovariate(1.0 / c["mean"]))))
            row.append(n)
            left -= n
        rows.append(row)
    return rows


def _padded(c):
    """(length, prefix) of every sequence of a padded batch; the last sequence is full."""
    rng = random.Random(c["T"] * 17 + c["mean"])
    ls = [max(1, min(c["T"], int(rng.uniform(0.5, 1.5) * c["mean"]))) for _ in range(c["B"] - 1)] + [c["T"]]
    return [(n, int(n * rng.uniform(0.1, 0.7))) for n in ls]


def _lengths(c):
    rng = random.Random(c["most"] * 13 + c["B"])
    return [c["most"]] + [rng.randint(c["least"], c["most"]) for _ in range(c["B"] - 1)]


def _pairs(n, ctx, window):
    """Visible (query, key) pairs of n causal queries behind ctx keys."""
    if not window:
        return n * ctx + n * (n + 1) // 2
    short = max(0, min(n, window - ctx))                                # queries that see fewer keys than the window
    return short * ctx + short * (short + 1) // 2 + (n - short) * window


def _visible(c):
    if c["mask"] == "documents":
        return sum(_pairs(n, 0, c["window"]) for row in _documents(c) for n in row)
    if c["mask"] == "prefix":
        return sum(p * p + (n * (n + 1) - p * (p + 1)) // 2 for n, p in _padded(c))
    return c["B"] * _pairs(c["T"], c["ctx"], c["window"])


def work(case):
    c = case
    if c["kind"] == "attention":
        size, Tk = TYPES[c["dtype"]].itemsize, c["T"] + c["ctx"]
        qs, ks = c["B"] * c["T"] * c["H"] * c["D"] * size, c["B"] * Tk * c["HKV"] * c["D"] * size
        passes = 3 if c["train"] else 1
        return {"bytes": (4 * qs + 4 * ks) if c["train"] else 2 * qs + 2 * ks,
                "flops": (14 if passes > 1 else 4) * _visible(c) * c["H"] * c["D"]}
    if c["kind"] == "step":
        size = TYPES[c["dtype"]].itemsize
        keys = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c))
        return {"bytes": (2 * keys * c["HKV"] + 2 * c["B"] * (c["H"] + c["HKV"])) * c["D"] * size, "flops": 4 * keys * c["H"] * c["D"]}
    rows, state = c["N"] * c["K"], c["layers"] * c["H"] * c["D"] * c["D"] * 4
    # a state that two beams go on from is read once; about half of the beams have a successor
    return {"bytes": rows * c["V"] * TYPES[c["dtype"]].itemsize + (rows + (rows + 1) // 2) * state, "flops": 3 * rows * c["V"]}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
PAGE = 64


def _ranges(c, shuffle):
    """First visible key and the key behind the last one, int32 [B, T]; None where nothing but causality limits a query."""
    B, T = c["B"], c["T"]
    if c["mask"] == "causal":
        return None, None
    at = torch.arange(T, dtype=torch.int32)
    if c["mask"] == "documents":
        first = torch.zeros(B, T, dtype=torch.int32)
        for b, row in enumerate(_documents(c)):
            shuffle.shuffle(row)
            lens = torch.tensor(row)
            first[b] = torch.repeat_interleave(torch.cumsum(lens, 0) - lens, lens).int()
        return first.cuda(), None
    stop = torch.zeros(B, T, dtype=torch.int32)
    rows = _padded(c)
    shuffle.shuffle(rows)
    for b, (n, p) in enumerate(rows):
        stop[b] = torch.where(at < n, torch.clamp(at + 1, min=p), 0)
    return None, stop.cuda()


def _slopes(c):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / c["H"]) for h in range(c["H"])], device="cuda") if c["slopes"] else None


def prepare(case, seed):
    c, gen, shuffle = case, torch.Generator(device="cuda").manual_seed(seed), random.Random(seed)
    dt = TYPES[c["dtype"]]

    def normal(*shape, dtype=dt, size=1.0):
        return (torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen) * size)

    if c["kind"] == "attention":
        B, T, Tk, D = c["B"], c["T"], c["T"] + c["ctx"], c["D"]
        first, stop = _ranges(c, shuffle)
        # capped layers have larger scores: about 6 in root mean square against 1.5
        q = normal(B, T, c["H"], D, size=6.0 if c["cap"] else 1.5).requires_grad_(c["train"])
        k, v = (normal(B, Tk, c["HKV"], D).requires_grad_(c["train"]) for _ in range(2))
        return dict(case=c, q=q, k=k, v=v, do=normal(B, T, c["H"], D) if c["train"] else None, first=first, stop=stop, slopes=_slopes(c))
    if c["kind"] == "step":
        B, lens = c["B"], _lengths(c)
        shuffle.shuffle(lens)
        need = [-(-n // PAGE) for n in lens]
        order = list(range(sum(need) + B))                              # a few pages are free
        shuffle.shuffle(order)
        table = torch.zeros(B, max(need), dtype=torch.int32)
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(order[:n], dtype=torch.int32)
            order = order[n:]
        P = sum(need) + B
        k, v = (normal(P, PAGE, c["HKV"], c["D"]) for _ in range(2))
        return dict(case=c, q=normal(B, c["H"], c["D"], size=6.0 if c["cap"] else 1.5), k=k, v=v, table=table.cuda(),
                    lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"), k_new=normal(B, c["HKV"], c["D"]), v_new=normal(B, c["HKV"], c["D"]),
                    slopes=_slopes(c))
    N, K = c["N"], c["K"]
    logits = normal(N, K, c["V"], size=3.0)
    scores = torch.sort(normal(N, K, dtype=torch.float32).abs() * -4 - 5, dim=-1, descending=True).values
    return dict(case=c, logits=logits, scores=scores, states=[normal(N * K, c["H"], c["D"], c["D"], dtype=torch.float32) for _ in range(c["layers"])])


# ---- one pass -------------------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if own:
        from linear_moe_b200 import ops
        options = {"window": c.get("window") or None, "softcap": c.get("cap") or None, "slopes": s.get("slopes")}
        if c["kind"] == "attention":
            o = ops.softmax_attention(s["q"], s["k"], s["v"], None, c["mask"] != "prefix", c["ctx"], key_first=s["first"], key_stop=s["stop"], **options)
            return (o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])) if c["train"] else o
        if c["kind"] == "step":
            return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], k_new=s["k_new"], v_new=s["v_new"], **options), s["k"], s["v"]
        scores, beam, token = ops.beam_select(s["logits"], s["scores"], 2 * c["K"])
        return scores, beam, token, ops.reorder_states(s["states"], _parents(beam, c["K"]))
    with torch.no_grad():
        return _plain_attention(s, c) if c["kind"] == "attention" else _plain_step(s, c) if c["kind"] == "step" else _plain_beam(s, c)


def _parents(beam, K):
    """Rows of the first K candidates' beams."""
    return (beam[:, :K] + K * torch.arange(beam.shape[0], device=beam.device)[:, None]).reshape(-1)


def _hidden(s, c):
    """[B or 1, Tq, Tk]: is the key out of the query's sight?"""
    T, Tk = c["T"], c["T"] + c["ctx"]
    i, j = torch.arange(T, device="cuda")[:, None] + c["ctx"], torch.arange(Tk, device="cuda")[None, :]
    h = (j > i) if c["mask"] != "prefix" else torch.zeros(T, Tk, dtype=torch.bool, device="cuda")
    if c["window"]:
        h = h | (j <= i - c["window"])
    h = h[None]
    if s["first"] is not None:
        h = h | (j[None] < s["first"][:, :, None])
    if s["stop"] is not None:
        h = h | (j[None] >= s["stop"][:, :, None])
    return h, (i - j).abs().float()


def _plain_attention(s, c):
    q, rep, scale = s["q"].float(), c["H"] // c["HKV"], c["D"] ** -0.5
    k, v = (t.float().repeat_interleave(rep, dim=2) for t in (s["k"], s["v"]))
    hidden, distance = _hidden(s, c)
    x = torch.einsum("bihd,bjhd->bhij", q, k).mul_(scale)
    if c["cap"]:
        t = torch.tanh(x.div_(c["cap"]))
        x = t * c["cap"]
    if s["slopes"] is not None:
        x -= s["slopes"][:, None, None] * distance
    x.masked_fill_(hidden[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    p = x.div_(x.sum(-1, keepdim=True).clamp_min(1e-30))
    o = torch.einsum("bhij,bjhd->bihd", p, v)
    if not c["train"]:
        return o.to(s["q"].dtype)
    do = s["do"].float()
    ds = torch.einsum("bihd,bjhd->bhij", do, v).sub_((do * o).sum(-1).transpose(1, 2)[..., None]).mul_(p)
    if c["cap"]:
        ds.mul_(1 - t * t)
    B, Tk = c["B"], c["T"] + c["ctx"]
    dv = torch.einsum("bhij,bihd->bjhd", p, do).reshape(B, Tk, c["HKV"], rep, c["D"]).sum(3)
    dk = torch.einsum("bhij,bihd->bjhd", ds, q).reshape(B, Tk, c["HKV"], rep, c["D"]).sum(3) * scale
    dq = torch.einsum("bhij,bjhd->bihd", ds, k) * scale
    return tuple(t.to(s["q"].dtype) for t in (o, dq, dk, dv))


def _plain_step(s, c):
    B, G, D, n = c["B"], c["HKV"], c["D"], s["lengths"].long()
    last = n - 1
    page = s["table"].gather(1, (last // PAGE)[:, None])[:, 0].long()
    s["k"][page, last % PAGE], s["v"][page, last % PAGE] = s["k_new"], s["v_new"]
    j = torch.arange(s["table"].shape[1] * PAGE, device="cuda")
    row = s["table"].long()[:, j // PAGE] * PAGE + j % PAGE
    k, v = (t.view(-1, G, D)[row].float() for t in (s["k"], s["v"]))
    q = s["q"].float().view(B, G, -1, D)
    x = torch.einsum("bgrd,bjgd->bgrj", q, k) * D ** -0.5
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, G, -1, 1) * (last[:, None] - j)[:, None, None].float()
    hidden = j[None] > last[:, None]
    if c["window"]:
        hidden = hidden | (j[None] <= last[:, None] - c["window"])
    x = x.masked_fill(hidden[:, None, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True)).exp()
    o = torch.einsum("bgrj,bjgd->bgrd", p, v) / p.sum(-1, keepdim=True)
    return o.reshape(B, c["H"], D).to(s["q"].dtype), s["k"], s["v"]


def _plain_beam(s, c):
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    total = (x - top).exp().sum(-1, keepdim=True).log() + top
    best, at = torch.sort((s["scores"].double()[..., None] + (x - total)).reshape(c["N"], -1), dim=-1, descending=True, stable=True)
    n = 2 * c["K"]
    beam = at[:, :n] // c["V"]
    parents = _parents(beam, c["K"])
    return best[:, :n].float(), beam, at[:, :n] % c["V"], [t[parents] for t in s["states"]]


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    with torch.no_grad():
        if c["kind"] == "beam":
            z = s["logits"].double()
            score = s["scores"].double().unsqueeze(-1) + z - torch.logsumexp(z, -1, keepdim=True)
            return score.flatten(1).topk(2 * c["K"], dim=-1).values, None, None, None
        q, D = s["q"].double(), c["D"]
        if c["kind"] == "step":
            out = torch.zeros(c["B"], c["H"], D, dtype=torch.float64, device="cuda")
            for b, n in enumerate(s["lengths"].tolist()):
                k, v = (torch.cat([pages[s["table"][b].long()].flatten(0, 1)[: n - 1], new[b][None]]).double()
                        for pages, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])))
                lo = max(0, n - c["window"]) if c["window"] else 0
                for h in range(c["H"]):
                    g = h * c["HKV"] // c["H"]
                    x = k[lo:, g] @ q[b, h] / math.sqrt(D)
                    if c["cap"]:
                        x = c["cap"] * torch.tanh(x / c["cap"])
                    if s["slopes"] is not None:
                        x = x - s["slopes"][h].double() * torch.arange(n - 1 - lo, -1, -1, device="cuda").double()
                    out[b, h] = torch.softmax(x, 0) @ v[lo:, g]
            return out, None, None
        T, Tk = c["T"], c["T"] + c["ctx"]
        i, j = torch.arange(T, device="cuda") + c["ctx"], torch.arange(Tk, device="cuda")
        res = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (s["q"], s["q"], s["k"], s["v"])]
        for b in range(c["B"]):
            lo, hi = torch.zeros_like(i), torch.full_like(i, Tk)
            if c["mask"] != "prefix":
                hi = i + 1
            if c["window"]:
                lo = (i - c["window"] + 1).clamp_min(0)
            if s["first"] is not None:
                lo = torch.maximum(lo, s["first"][b].long())
            if s["stop"] is not None:
                hi = torch.minimum(hi, s["stop"][b].long())
            seen = (j >= lo[:, None]) & (j < hi[:, None])
            for h in range(c["H"]):
                g = h * c["HKV"] // c["H"]
                qh, kh, vh = q[b, :, h], s["k"][b, :, g].double(), s["v"][b, :, g].double()
                x = qh @ kh.T / math.sqrt(D)
                slope = 1.0
                if c["cap"]:
                    y = torch.tanh(x / c["cap"])
                    x, slope = c["cap"] * y, 1 - y ** 2
                if s["slopes"] is not None:
                    x = x - s["slopes"][h].double() * (i[:, None] - j).abs()
                p = torch.nan_to_num(torch.softmax(torch.where(seen, x, -math.inf), -1))      # a query that sees nothing: zeros
                o = res[0][b, :, h] = p @ vh
                if c["train"]:
                    g_o = s["do"][b, :, h].double()
                    ds = p * (g_o @ vh.T - (g_o * o).sum(-1, keepdim=True)) * slope / math.sqrt(D)
                    res[1][b, :, h] = ds @ kh
                    res[2][b, :, g] += ds.T @ qh
                    res[3][b, :, g] += p.T @ g_o
        return tuple(res) if c["train"] else res[0]
