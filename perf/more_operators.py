"""Operators between a softmax layer's projection and the next token that are timed on their own, each through the call that a user makes.

* ``heads``   queries, keys and values out of a fused projection: RMS norm of every query and key head and rotation by its position;
              ``train`` asks for the gradients too
* ``cache``   keys and values into a paged cache of 4 bits a number, and what the requests' pages hold back out of it (a prompt's next
              portion attends to the ones in front of it)
* ``step``    attention of one new token of every request over such a cache
* ``sample``  the next token of every request: temperature, top-k, top-p and min-p from given random numbers

``run`` makes the calls of :mod:`linear_moe_b200.ops` where ``own`` is true, and computes the plain form in 32 bits (64 for the sums
and borders of the sampling) where it is not.  ``exact`` is the definition in 64 bits.

A row of 4-bit numbers goes in groups of 32, x = low + size * code with ``low`` the least number of the group, rounded down to bf16,
and ``size`` a fifteenth of what is left up to the greatest one, rounded up to bf16.  A page holds, head by head, the codes of its rows
and then every row's lows and sizes; the 16 bytes of a group lie at ``_place`` of their row.
"""
import math
import random

import torch

own = False
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PAGE, UNIT = 64, 32                       # rows of a page, numbers of a group
FIFTEENTH = float(torch.tensor(1.0 / 15.0))


def listed():
    return [
        # two short sequences of a small layer: the smallest training call, where the launches count
        dict(name="heads_train_2x65", kind="heads", B=2, T=65, H=4, HKV=2, D=64, rot=64, norm=True, inter=False, at=0, dtype="bf16", train=True),
        # pretraining at 16384 tokens, 32 query heads on 8
        dict(name="heads_train_16k", kind="heads", B=1, T=16384, H=32, HKV=8, D=128, rot=128, norm=True, inter=False, at=0, dtype="bf16", train=True),
        # fine-tuning in fp32: an odd length, heads of 96 of which a third turns, in neighbouring pairs
        dict(name="heads_train_3x1531", kind="heads", B=3, T=1531, H=12, HKV=4, D=96, rot=32, norm=True, inter=True, at=0, dtype="fp32", train=True),
        # one token of 64 requests at positions of their own
        dict(name="heads_step_64", kind="heads", B=64, T=1, H=32, HKV=8, D=128, rot=128, norm=True, inter=False, at=8192, dtype="bf16", train=False),
        # one new token of 64 requests of up to 200 tokens: stored, and the short contexts read back
        dict(name="cache_64x1", kind="cache", B=64, T=1, most=200, HKV=8, D=128, dtype="bf16"),
        # the next portion of four long prompts behind what the cache holds of them, heads of 96 in fp16
        dict(name="cache_4x1531", kind="cache", B=4, T=1531, most=6000, HKV=8, D=96, dtype="fp16"),
        # one request at the beginning of its answer
        dict(name="step_1x300", kind="step", B=1, most=300, least=300, H=16, HKV=4, D=128, dtype="bf16", window=0, cap=0.0, slopes=False),
        # two long contexts with few key heads, a distance bias: the cache's length is all there is to split
        dict(name="step_2x100k", kind="step", B=2, most=100001, least=60000, H=16, HKV=2, D=64, dtype="fp16", window=0, cap=0.0, slopes=True),
        # a full batch of long requests, capped
        dict(name="step_64x8k", kind="step", B=64, most=8192, least=1000, H=32, HKV=8, D=128, dtype="bf16", window=0, cap=50.0, slopes=False),
        # a single request, nucleus sampling over a small vocabulary
        dict(name="sample_1x32000", kind="sample", B=1, V=32000, dtype="bf16", k=0, p=0.9, least=0.0, own_settings=False),
        # requests with settings of their own over an odd vocabulary
        dict(name="sample_17x50257", kind="sample", B=17, V=50257, dtype="bf16", k=200, p=0.95, least=0.02, own_settings=True),
        # a full batch over the vocabulary of the 1B model, logits in fp32
        dict(name="sample_128x128256", kind="sample", B=128, V=128256, dtype="fp32", k=0, p=0.95, least=0.0, own_settings=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["heads", "heads", "cache", "step", "step", "sample", "sample"])
    if kind == "heads":
        HKV, D, train = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 96, 128, 128]), rng.random() < 0.7
        H = HKV * rng.choice([1, 2, 3, 4, 7])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = min(10000, 200_000_000 // ((H + 2 * HKV) * D * TYPES[dtype].itemsize))          # rows
        T = _log(rng, 33, most) if train else rng.choice([1, 1, _log(rng, 2, 2000)])
        B = max(1, min(4, most // T)) if train else _log(rng, 1, max(1, min(128, most // T)))
        return dict(kind=kind, B=B, T=T, H=H, HKV=HKV, D=D, rot=rng.choice([D, D, D // 2, 32, 0]), norm=rng.random() < 0.8, inter=rng.random() < 0.3,
                    at=rng.choice([0, _log(rng, 2048, 65536)]), dtype=dtype, train=train)
    if kind == "cache":
        T = rng.choice([1, _log(rng, 2, 2000)])
        B = max(1, min(64, _log(rng, 1, 4000 // T)))
        return dict(kind=kind, B=B, T=T, most=T + rng.choice([0, _log(rng, 1, 20000 // B)]), HKV=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 96, 128, 128]),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if kind == "step":
        B, HKV = _log(rng, 1, 64), rng.choice([1, 2, 4, 8])
        most = _log(rng, 64, min(100000, 500000 // B))
        return dict(kind=kind, B=B, most=most, least=max(1, int(most * rng.uniform(0.01, 1.0))), H=HKV * rng.choice([1, 3, 4, 8, 16]), HKV=HKV,
                    D=rng.choice([64, 96, 128, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]), window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                    cap=rng.choice([0.0, 20.0, 50.0]), slopes=rng.random() < 0.3)
    return dict(kind=kind, B=_log(rng, 1, 128), V=_log(rng, 1000, 128256), dtype=rng.choice(["bf16", "fp16", "fp32"]), k=rng.choice([0, 1, _log(rng, 2, 1000)]),
                p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]), least=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]),
                own_settings=rng.random() < 0.4)


# ---- what follows from a case alone: the lengths that its seed only shuffles -----------------------------------------------------
def _lengths(c):
    """Tokens of every request, the new one counted."""
    rng = random.Random(c["most"] * 13 + c["B"])
    least = c.get("least", c.get("T"))
    return [c["most"]] + [rng.randint(least, c["most"]) for _ in range(c["B"] - 1)]


def _row_bytes(D):
    return D // 2 + D // UNIT * 4


def work(case):
    c = case
    size = TYPES[c["dtype"]].itemsize
    if c["kind"] == "heads":
        rows, tables = c["B"] * c["T"], min(c["B"] * c["T"], c["at"] or c["T"]) * c["rot"] * 4
        numbers = rows * (c["H"] + 2 * c["HKV"]) * c["D"]
        turned = rows * (c["H"] + c["HKV"]) * c["D"]
        return {"bytes": (4 if c["train"] else 2) * numbers * size + tables, "flops": turned * (22 if c["train"] else 7)}
    if c["kind"] == "cache":
        new, all_ = (n * c["HKV"] * 2 for n in (c["B"] * c["T"], sum(_lengths(c))))
        # a read of the pages gives the longest request's rows for everyone
        return {"bytes": new * (c["D"] * size + _row_bytes(c["D"])) + all_ * _row_bytes(c["D"]) + c["B"] * c["most"] * c["HKV"] * 2 * c["D"] * size,
                "flops": (new * 6 + all_ * 2) * c["D"]}
    if c["kind"] == "step":
        keys = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c))
        return {"bytes": 2 * keys * c["HKV"] * _row_bytes(c["D"]) + 2 * c["B"] * c["H"] * c["D"] * size, "flops": 4 * keys * c["H"] * c["D"]}
    return {"bytes": c["B"] * c["V"] * size + c["B"] * 12, "flops": 4 * c["B"] * c["V"]}


# ---- a cache of 4 bits a number ---------------------------------------------------------------------------------------------------
def _place(D, device):
    """Where the 16 bytes of a row's groups lie, [PAGE, D / 32]: two groups change places every four rows, four go round every two."""
    n = D // UNIT
    row, at = torch.arange(PAGE, device=device)[:, None], torch.arange(n, device=device)[None, :]
    return at ^ ((row // 2) % 4) if n == 4 else at ^ ((row // 4) % 2) if n == 2 else at.expand(PAGE, n)


def _codes(x):
    """x [..., D] fp32 -> codes [..., D / 32, 32] (whole numbers), lows and sizes [..., D / 32] (numbers that bf16 holds)."""
    g = x.unflatten(-1, (-1, UNIT))
    bits = g.amin(-1).view(torch.int32)
    low = (torch.where(bits < 0, bits + 0xffff, bits) & -65536).view(torch.float32)
    size = (((g.amax(-1) - low) * FIFTEENTH).view(torch.int32) + 0xffff & -65536).view(torch.float32)
    code = torch.round((g - low[..., None]) / torch.where(size > 0, size, 1.0)[..., None]).clamp_(0, 15)
    return code, low, size


def _rows_to_bytes(x, rows):
    """x [n, heads, D] fp32 that go to rows ``rows`` [n] of their pages -> bytes of the codes [n, heads, D / 2] and of the scales."""
    D = x.shape[-1]
    code, low, size = _codes(x)
    code = code.to(torch.uint8)
    packed = code[..., 0::2] | code[..., 1::2] << 4
    place = _place(D, x.device)[rows][:, None, :, None].expand(packed.shape)
    scales = torch.cat([low, size], dim=-1).to(torch.bfloat16)
    return torch.empty_like(packed).scatter_(2, place, packed).flatten(2), scales.view(torch.uint8)


def _split(pool, D):
    """The pages' codes [P, heads, PAGE, D / 2] and scales [P, heads, PAGE, D / 8], as views."""
    P, G = pool.shape[:2]
    return pool[:, :, : PAGE * D // 2].view(P, G, PAGE, D // 2), pool[:, :, PAGE * D // 2:].view(P, G, PAGE, D // 8)


def _values(pages, D):
    """Bytes [..., heads, page bytes] of whole pages -> their numbers [..., heads, PAGE, D] in fp32."""
    n = D // UNIT
    packed = pages[..., : PAGE * D // 2].unflatten(-1, (PAGE, n, 16))
    place = _place(D, pages.device)[:, :, None].expand(PAGE, n, 16)
    packed = packed.gather(-2, place.expand(packed.shape))
    scales = pages[..., PAGE * D // 2:].contiguous().view(torch.bfloat16).unflatten(-1, (PAGE, 2, n)).float()
    code = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2).float()
    return (scales[..., 0, :, None] + scales[..., 1, :, None] * code).flatten(-2)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _pool(c, pages, gen):
    """Pages of the numbers that a layer's keys and values are like, already in 4 bits."""
    G, D = c["HKV"], c["D"]
    pool = torch.empty(pages, G, PAGE * _row_bytes(D), dtype=torch.uint8, device="cuda")
    rows = torch.arange(PAGE, device="cuda")
    codes, scales = _split(pool, D)
    for at in range(0, pages, 512):
        n = min(512, pages - at)
        x = torch.empty(n * PAGE, G, D, device="cuda").normal_(generator=gen)
        a, b = _rows_to_bytes(x, rows.repeat(n))
        codes[at:at + n] = a.view(n, PAGE, G, -1).transpose(1, 2)
        scales[at:at + n] = b.view(n, PAGE, G, -1).transpose(1, 2)
    return pool


def _pages(lens, shuffle):
    """A table of pages in no order, and how many pages the pool has (a few are free)."""
    need = [-(-n // PAGE) for n in lens]
    order = list(range(sum(need) + len(lens)))
    shuffle.shuffle(order)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[:n], dtype=torch.int32)
        order = order[n:]
    return table.cuda(), sum(need) + len(lens)


def prepare(case, seed):
    c, gen, shuffle = case, torch.Generator(device="cuda").manual_seed(seed), random.Random(seed)
    dt = TYPES[c["dtype"]]

    def normal(*shape, dtype=dt, size=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen) * size

    if c["kind"] == "heads":
        B, T, H, G, D = c["B"], c["T"], c["H"], c["HKV"], c["D"]
        s = dict(case=c, qkv=normal(B, T, G, H // G + 2, D, size=1.3).requires_grad_(c["train"]), wq=None, wk=None, cos=None, sin=None, at=None)
        if c["norm"]:
            s["wq"], s["wk"] = ((1 + normal(D, dtype=torch.float32, size=0.2)).to(dt).requires_grad_(c["train"]) for _ in range(2))
        if c["rot"]:
            turn = torch.arange(c["at"] or T, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda").double() / c["rot"])
            s["cos"], s["sin"] = turn.cos().float(), turn.sin().float()
            if c["at"]:                                                 # every request goes on from a position of its own
                first = torch.randint(0, max(1, c["at"] - T), (B, 1), generator=gen, device="cuda")
                s["at"] = (first + torch.arange(T, device="cuda")) % c["at"]
        if c["train"]:
            s["grads"] = [normal(B, T, n, D) for n in (H, G, G)]
        return s
    if c["kind"] in ("cache", "step"):
        lens = _lengths(c)
        shuffle.shuffle(lens)
        table, pages = _pages(lens, shuffle)
        s = dict(case=c, k=_pool(c, pages, gen), v=_pool(c, pages, gen), table=table, lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
        if c["kind"] == "cache":
            s["k_new"], s["v_new"] = (normal(c["B"], c["T"], c["HKV"], c["D"]) for _ in range(2))
        else:
            s["q"] = normal(c["B"], c["H"], c["D"], size=6.0 if c["cap"] else 1.5)
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / c["H"]) for h in range(c["H"])], device="cuda") if c["slopes"] else None
        return s
    B, V = c["B"], c["V"]
    logits = normal(B, V, dtype=torch.float32, size=2.0)                # a broad floor, and a few dozen tokens that stand out of it
    some = torch.randint(0, V, (B, 40), generator=gen, device="cuda")
    logits.scatter_add_(1, some, torch.empty(B, 40, device="cuda").exponential_(0.25, generator=gen))
    s = dict(case=c, logits=logits.to(dt), draw=torch.rand(B, generator=gen, device="cuda"), temperature=0.8, top_k=c["k"], top_p=c["p"], min_p=c["least"])
    if c["own_settings"]:
        def spread(lo, hi):
            return torch.empty(B, device="cuda").uniform_(lo, hi, generator=gen)
        s.update(temperature=spread(0.5, 1.5), top_k=torch.randint(1, 2 * c["k"] + 2, (B,), generator=gen, device="cuda", dtype=torch.int32),
                 top_p=spread(c["p"] / 2, 1.0), min_p=spread(0.0, 2 * c["least"]))
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if own:
        from linear_moe_b200 import ops
        if c["kind"] == "heads":
            q, k, v = ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"], positions=s["at"], interleaved=c["inter"])
            if not c["train"]:
                return q, k, v
            leaves = [t for t in (s["qkv"], s["wq"], s["wk"]) if t is not None]
            return (q, k, v, *torch.autograd.grad((q, k, v), leaves, s["grads"]))
        if c["kind"] == "cache":
            ops.store_rows_int4(s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["lengths"])
            return ops.read_rows_int4(s["k"], s["v"], s["table"], s["lengths"], c["most"], c["D"], TYPES[c["dtype"]])
        if c["kind"] == "step":
            return ops.paged_attention_int4(s["q"], s["k"], s["v"], s["table"], s["lengths"], None, c["window"] or None, softcap=c["cap"] or None, slopes=s["slopes"])
        return ops.sample_tokens(s["logits"], s["draw"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    with torch.no_grad():
        return {"heads": _plain_heads, "cache": _plain_cache, "step": _plain_step, "sample": _plain_sample}[c["kind"]](s, c)


def _turn(x, cos, sin, inter):
    """Pairs of the first numbers of x [B, T, n, D] turned by cos, sin [B or 1, T, 1, R / 2]."""
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if inter else (x[..., : R // 2], x[..., R // 2:R])
    y = torch.empty_like(x)
    y[..., R:] = x[..., R:]
    if inter:
        y[..., 0:R:2], y[..., 1:R:2] = a * cos - b * sin, a * sin + b * cos
    else:
        y[..., : R // 2], y[..., R // 2:R] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_heads(s, c):
    B, T, G, r, D = s["qkv"].shape
    dt, x = s["qkv"].dtype, s["qkv"].float()
    parts = [x[:, :, :, : r - 2].reshape(B, T, -1, D), x[:, :, :, r - 2]]
    cos, sin = s["cos"], s["sin"]
    if cos is not None:
        cos, sin = ((t[s["at"]] if s["at"] is not None else t[None, :T])[:, :, None] for t in (cos, sin))
    weights = [None if w is None else w.float() for w in (s["wq"], s["wk"])]
    outs, kept = [], []
    for h, w in zip(parts, weights):
        inv = None
        if w is not None:
            inv = torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6)
            h = h * inv
        y = h if w is None else h * w
        outs.append((y if cos is None else _turn(y, cos, sin, c["inter"])).to(dt))
        kept.append((h, inv))
    outs.append(s["qkv"][:, :, :, r - 1].contiguous())
    if not c["train"]:
        return tuple(outs)
    dx, dws = torch.empty_like(x), []
    dx[:, :, :, r - 1] = s["grads"][2].float()
    for i, (h, inv) in enumerate(kept):
        d = s["grads"][i].float()
        if cos is not None:
            d = _turn(d, cos, -sin, c["inter"])
        if weights[i] is not None:
            dws.append((d * h).sum((0, 1, 2)).to(dt))
            d = d * weights[i]
            d = (d - h * (d * h).mean(-1, keepdim=True)) * inv
        if i == 0:
            dx[:, :, :, : r - 2] = d.view(B, T, G, r - 2, D)
        else:
            dx[:, :, :, r - 2] = d
    return (*outs, dx.to(dt), *dws)


def _plain_cache(s, c):
    T, D = c["T"], c["D"]
    at = s["lengths"].long()[:, None] - T + torch.arange(T, device="cuda")                # rows of the new tokens
    page, row = s["table"].long().gather(1, at // PAGE).flatten(), (at % PAGE).flatten()
    for pool, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        codes, scales = _split(pool, D)
        codes[page, :, row], scales[page, :, row] = _rows_to_bytes(new.float().flatten(0, 1), row)
    hidden = torch.arange(c["most"], device="cuda") >= s["lengths"][:, None]
    out = []
    for pool in (s["k"], s["v"]):
        x = _values(pool[s["table"].long()], D).transpose(2, 3).flatten(1, 2)[:, : c["most"]]
        out.append(x.masked_fill(hidden[:, :, None, None], 0.0).to(TYPES[c["dtype"]]))
    return tuple(out)


def _plain_step(s, c):
    B, G, D, n = c["B"], c["HKV"], c["D"], s["lengths"].long()
    k, v = (_values(pool[s["table"].long()], D).transpose(2, 3).flatten(1, 2) for pool in (s["k"], s["v"]))
    j = torch.arange(k.shape[1], device="cuda")
    x = torch.einsum("bgrd,bjgd->bgrj", s["q"].float().view(B, G, -1, D), k) * D ** -0.5
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, G, -1, 1) * (n[:, None] - 1 - j)[:, None, None].float()
    hidden = j[None] >= n[:, None]
    if c["window"]:
        hidden = hidden | (j[None] < n[:, None] - c["window"])
    x = x.masked_fill(hidden[:, None, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True)).exp()
    o = torch.einsum("bgrj,bjgd->bgrd", p, v) / p.sum(-1, keepdim=True)
    return o.reshape(B, c["H"], D).to(s["q"].dtype)


def _plain_sample(s, c):
    B, V = s["logits"].shape

    def setting(x):
        return (x if torch.is_tensor(x) else torch.full((B,), x, dtype=torch.float32, device="cuda"))[:, None].double()

    z, k, p = s["logits"].double(), setting(s["top_k"]), setting(s["top_p"])
    z, order = torch.sort(z, dim=-1, descending=True, stable=True)
    w = ((z - z[:, :1]) / setting(s["temperature"])).exp()
    upto = w.cumsum(-1)
    before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], dim=-1)             # what comes ahead of a token
    keep = (torch.arange(V, device="cuda") < torch.where(k > 0, k, V)) & ((before < p * upto[:, -1:]) | (p >= 1)) & (w >= setting(s["min_p"]))
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))               # back in the vocabulary's order
    upto = kept.cumsum(-1)
    total = upto[:, -1:]
    token = (upto <= s["draw"].double()[:, None] * total).sum(-1)
    return token, (kept.gather(1, token[:, None]) / total).log()[:, 0].float()


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------
def _numbers(pool, page, row, D):
    """What rows ``row`` [n] of the pages ``page`` hold: [n, heads, D]."""
    n, every = D // UNIT, torch.arange(len(row), device="cuda")
    shift = {4: row // 2 % 4, 2: row // 4 % 2}.get(n, row * 0)
    code, scale = _split(pool, D)
    code = code[page, :, row].unflatten(-1, (n, 16))                                       # [rows, heads, place, 16]
    code = torch.stack([code[every, :, i ^ shift] if n in (2, 4) else code[:, :, i] for i in range(n)], 2)
    scale = scale[page, :, row].contiguous().view(torch.bfloat16).double().unflatten(-1, (2, n))
    nibbles = torch.stack([code % 16, code // 16], -1).flatten(-2).double()
    return (nibbles * scale[:, :, 1, :, None] + scale[:, :, 0, :, None]).flatten(-2)


def _in_four_bits(x):
    """x [..., D] as four bits a number give it back.  The steps that pick the codes have 32 bits by definition: 64 rounded to them."""
    def bf16(y, up):                                                    # the next number of 8 bits, up or down
        m, e = torch.frexp(y)
        return torch.ldexp((torch.ceil if up else torch.floor)(m * 256), e - 8)

    x = x.double().unflatten(-1, (-1, UNIT))
    low = bf16(x.amin(-1, keepdim=True), False)
    size = bf16(((x.amax(-1, keepdim=True) - low).float().double() * FIFTEENTH).float().double(), True)
    code = torch.where(size > 0, ((x - low).float().double() / size).float().double(), 0.0).round().clamp(0, 15)
    return (low + size * code).flatten(-2)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "heads":
        x = s["qkv"].detach().double().requires_grad_(c["train"])
        ws = [None if w is None else w.detach().double().requires_grad_(c["train"]) for w in (s["wq"], s["wk"])]
        outs = []
        for part, w in zip((x[..., :-2, :].flatten(2, 3), x[..., -2, :]), ws):
            if w is not None:
                part = part * w / torch.sqrt(part.square().mean(-1, keepdim=True) + 1e-6)
            if c["rot"]:
                R, pos = c["rot"], s["at"] if s["at"] is not None else torch.arange(c["T"], device="cuda")[None]
                turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, :, None]
                pairs = part[..., :R].unflatten(-1, (R // 2, 2) if c["inter"] else (2, R // 2))
                if not c["inter"]:
                    pairs = pairs.transpose(-1, -2)
                turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
                turned = turned.flatten(-2) if c["inter"] else turned.transpose(-1, -2).flatten(-2)
                part = torch.cat([turned, part[..., R:]], dim=-1)
            outs.append(part)
        outs.append(x[..., -1, :])
        if not c["train"]:
            return tuple(outs)
        leaves = [x] + [w for w in ws if w is not None]
        return (*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, [g.double() for g in s["grads"]]))
    with torch.no_grad():
        if c["kind"] == "step":
            D = c["D"]
            out = torch.zeros(c["B"], c["H"], D, dtype=torch.float64, device="cuda")
            for b, length in enumerate(s["lengths"].tolist()):
                lo = max(0, length - c["window"]) if c["window"] else 0
                rows = torch.arange(lo, length, device="cuda")
                kv = [_numbers(pool, s["table"][b].long()[rows // PAGE], rows % PAGE, D) for pool in (s["k"], s["v"])]
                for h in range(c["H"]):
                    g = h * c["HKV"] // c["H"]
                    x = kv[0][:, g] @ s["q"][b, h].double() / math.sqrt(D)
                    if c["cap"]:
                        x = c["cap"] * torch.tanh(x / c["cap"])
                    if s["slopes"] is not None:
                        x = x - s["slopes"][h].double() * (length - 1 - rows).double()
                    out[b, h] = torch.softmax(x, 0) @ kv[1][:, g]
            return out
        if c["kind"] == "cache":
            res = torch.zeros(2, c["B"], c["most"], c["HKV"], c["D"], dtype=torch.float64, device="cuda")
            for b, length in enumerate(s["lengths"].tolist()):
                rows = torch.arange(length - c["T"], device="cuda")
                for i, (pool, new) in enumerate(((s["k"], s["k_new"]), (s["v"], s["v_new"]))):
                    res[i, b, : length - c["T"]] = _numbers(pool, s["table"][b].long()[rows // PAGE], rows % PAGE, c["D"])
                    res[i, b, length - c["T"]: length] = _in_four_bits(new[b])
            return res[0], res[1]
        res = torch.zeros(c["B"], dtype=torch.float64, device="cuda")
        for b in range(c["B"]):
            t, k, p, least = (float(x[b] if torch.is_tensor(x) else torch.tensor(x, dtype=torch.float32)) for x in (s["temperature"], s["top_k"], s["top_p"], s["min_p"]))
            z, order = torch.sort(s["logits"][b].double(), descending=True, stable=True)
            prob = torch.softmax(z / t, 0)
            n = len(prob) if p >= 1 else int(torch.searchsorted(prob.cumsum(0), p)) + 1     # the first n tokens reach p
            n = max(1, min(n, int(k) if k else n, int((prob >= least * prob[0]).sum())))
            # back in the vocabulary's order, where the draw falls into the token that it reaches
            place, rank = torch.sort(order[:n])
            share = prob[:n][rank] / prob[:n].sum()
            i = min(int(torch.searchsorted(share.cumsum(0), s["draw"][b].double(), right=True)), n - 1)
            res[b] = share[i].log()
        return None, res
