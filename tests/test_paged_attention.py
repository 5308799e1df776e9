"""One-token attention over a paged cache, against the formula in 64 bits.

Bounds.  u = finfo(type).eps / 2 is the largest relative error of one rounding.  On the tensor cores the weights are rounded once and the output is rounded once:
elementwise |error| <= 2 u sum p |v|, and 2 u in the 2-norm (errors of single roundings have no common sign).  A quarter of u covers the 32-bit part (scores to 2^-24 of their
terms, 2e-7 of the cap in tanh, exp2 to 2^-22).  fp16 numbers below 2^-14 are rounded by up to 2^-25 whatever their size, which adds 2^-25 sum |v|.
The general kernel rounds the output alone (u); in fp32 it is the sums of 512 terms at most that count: 64 times 2^-24 of the terms' magnitudes."""
import math

import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.ops import paged_attn as PA

gpu = pytest.mark.gpu


def make(lens, H, G, D, page=64, dtype=torch.bfloat16, device="cuda", size=1.5, seed=0, stale=float("nan"), spare=3):
    """Pages in no order whose rows behind a request's last key hold `stale`, as do the pages of nobody."""
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen)            # noqa: E731
    need = [-(-x // page) for x in lens]
    P, width = sum(need) + spare, max(need + [1]) + 1
    order = torch.randperm(P, generator=gen).tolist()
    table = torch.randint(-9, P + 9, (len(lens), width), generator=gen, dtype=torch.int32)       # entries behind the length: anything
    k, v = torch.full((P, page, G, D), stale), torch.full((P, page, G, D), stale)
    for b, x in enumerate(lens):
        at = [order.pop() for _ in range(need[b])]
        table[b, :need[b]] = torch.tensor(at, dtype=torch.int32)
        for i in range(x - 1):
            k[at[i // page], i % page], v[at[i // page], i % page] = n(G, D), n(G, D)
    B = len(lens)
    t = dict(q=(n(B, H, D) * size).to(dtype), k=k.to(dtype), v=v.to(dtype), table=table, lengths=torch.tensor(lens, dtype=torch.int32), k_new=n(B, G, D).to(dtype),
             v_new=n(B, G, D).to(dtype))
    return {x: y.to(device) for x, y in t.items()}


def formula(s, window=None, cap=None, slopes=None, scale=None):
    """(output, sum p |v|, sum |v|, pages with the new rows) in 64 bits."""
    q, page = s["q"].double(), s["k"].shape[1]
    B, H, D = q.shape
    G = s["k"].shape[2]
    k, v = s["k"].clone(), s["v"].clone()
    out = [torch.zeros(B, H, D, dtype=torch.float64, device=q.device) for _ in range(3)]
    for b, n in enumerate(s["lengths"].tolist()):
        if n <= 0:
            continue
        at = s["table"][b, : -(-n // page)].long()
        if s["k_new"] is not None:
            k[at[-1], (n - 1) % page], v[at[-1], (n - 1) % page] = s["k_new"][b], s["v_new"][b]
        lo = max(0, n - window) if window else 0
        kb, vb = (t[at].flatten(0, 1)[lo:n].double().repeat_interleave(H // G, 1) for t in (k, v))
        x = torch.einsum("hd,jhd->hj", q[b], kb) * (scale or D ** -0.5)
        if cap:
            x = cap * torch.tanh(x / cap)
        if slopes is not None:
            x = x - slopes.double()[:, None] * torch.arange(n - 1 - lo, -1, -1, device=q.device)
        p = torch.softmax(x, -1)
        out[0][b], out[1][b], out[2][b] = torch.einsum("hj,jhd->hd", p, vb), torch.einsum("hj,jhd->hd", p, vb.abs()), vb.abs().sum(0)
    return *out, k, v


def check(s, window=None, cap=None, slopes=None, scale=None, roundings=2):
    want, mag, low, k, v = formula(s, window, cap, slopes, scale)
    got = ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], scale, window, softcap=cap, slopes=slopes, k_new=s["k_new"], v_new=s["v_new"])
    dtype = s["q"].dtype
    assert got.dtype == dtype and torch.isfinite(got).all()
    err = (got.double() - want).abs()
    if dtype == torch.float32:
        assert (err <= 64 * 2.0 ** -24 * mag).all()
    else:
        u = torch.finfo(dtype).eps / 2
        tiny = torch.finfo(dtype).smallest_normal * u
        assert (err <= (roundings + 0.25) * u * mag + tiny * (low + 1)).all(), ((err / mag.clamp_min(1e-30)).max().item() / u)
        if want.norm() > 0:
            assert (got.double() - want).norm() < roundings * u * want.norm()
    for a, b in ((s["k"], k), (s["v"], v)):                    # the new rows are there, and nothing else has changed
        assert torch.equal(a.view(torch.uint8) if a.dtype.itemsize == 1 else a.view(torch.int16 if a.dtype.itemsize == 2 else torch.int32),
                           b.view(torch.uint8) if b.dtype.itemsize == 1 else b.view(torch.int16 if b.dtype.itemsize == 2 else torch.int32))
    return got


def slope_table(H, device="cuda"):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=device)


# ---- on the CPU -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("window,cap,bias", [(None, None, False), (5, 3.0, True), (1, None, False), (100, 3.0, False)])
def test_eager_definition(window, cap, bias):
    s = make([0, 1, 7, 16, 17, 40], 6, 2, 10, page=8, dtype=torch.float32, device="cpu")
    got = check(s, window, cap, slope_table(6, "cpu") if bias else None)
    assert (got[0] == 0).all()
    s["k_new"] = s["v_new"] = None                             # the rows are in the cache by now
    assert torch.equal(check(s, window, cap, slope_table(6, "cpu") if bias else None), got)


def test_refusals():
    def bad(error=ValueError, **kw):
        s = make([5, 9], 4, 2, 8, page=8, dtype=torch.float32, device="cpu")
        opt = {x: kw.pop(x) for x in ("scale", "window", "softcap", "slopes") if x in kw}
        s.update({x: y(s[x]) if callable(y) else y for x, y in kw.items()})
        with pytest.raises(error):
            ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], k_new=s["k_new"], v_new=s["v_new"], **opt)
    bad(q=lambda t: t[None]), bad(q=lambda t: t[:, :3]), bad(q=lambda t: t[:, :, :4]), bad(q=lambda t: t.double())
    bad(v=lambda t: t[:, :4]), bad(v=lambda t: t.half()), bad(k=lambda t: t[:, :, :0], v=lambda t: t[:, :, :0])
    bad(k=lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)), bad(q=lambda t: t.requires_grad_(True))
    bad(table=lambda t: t.long()), bad(table=lambda t: t[:1]), bad(lengths=lambda t: t.long()), bad(lengths=lambda t: t[:1])
    bad(k_new=None), bad(v_new=None), bad(k_new=lambda t: t[:1]), bad(v_new=lambda t: t.half())
    bad(window=0), bad(scale=-1.0), bad(softcap=0.0), bad(slopes=torch.ones(3)), bad(slopes=torch.ones(4).double())
    bad(q=torch.zeros(2, 4, 600), k=torch.zeros(3, 8, 2, 600), v=torch.zeros(3, 8, 2, 600), k_new=None, v_new=None)
    # lengths and pages that are none: the CPU form sees them
    bad(lengths=torch.tensor([5, 99], dtype=torch.int32)), bad(lengths=torch.tensor([-1, 9], dtype=torch.int32))
    bad(table=torch.tensor([[0, 0], [7, 9]], dtype=torch.int32)), bad(table=torch.tensor([[-1, 0], [1, 2]], dtype=torch.int32))


def test_split_rule():
    """At least one part, none of fewer than 128 keys of a long request; one wave of CTAs, or two parts."""
    for B in (1, 2, 8, 64, 1000):
        for G in (1, 2, 8):
            for heads in (1, 8, 9, 33):
                for D in (64, 128):
                    for keys in (0, 1, 256, 257, 5000, 1 << 20):
                        n, first = PA.splits_of(B, G, heads, D, keys)
                        assert 1 <= n <= max(1, -(-keys // 128))
                        assert n <= 2 or n * B * G <= 4 * 148
                        assert not first or 1 < B <= 128


# ---- on the GPU -----------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [8, 64, 72, 128])
def test_lengths(dtype, D):
    """Empty requests, single keys, groups and pages that end inside, splits."""
    s = make([0, 1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 700, 1500], 8, 2, D, dtype=dtype)
    got = check(s)
    assert (got[0] == 0).all()
    check(s, cap=20.0)


@gpu
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (8, 8), (8, 1), (9, 1), (16, 1), (40, 2), (24, 3)])
@pytest.mark.parametrize("cap,bias", [(None, False), (30.0, True)])
def test_heads_and_scores(heads, cap, bias):
    s = make([300, 20, 1], *heads, 64, size=4.0)
    check(s, cap=cap, slopes=slope_table(heads[0]) if bias else None)


@gpu
@pytest.mark.parametrize("window", [1, 15, 16, 17, 64, 100, 5000])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_windows_and_pages(window, page):
    s = make([1, 90, 640, 1033], 4, 2, 128, page=page)
    check(s, window, slopes=slope_table(4))


@gpu
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
def test_any_number_of_splits(splits, monkeypatch):
    """The parts of a request, more CTAs than it has keys for among them, give the whole."""
    monkeypatch.setattr(PA, "splits_of", lambda *a: (splits, splits % 2))
    s = make([0, 5, 256, 257, 2000, 4097], 8, 2, 128, size=4.0)
    check(s, cap=50.0)
    check(s, 1000)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,page", [(7, 64), (64, 10), (128, 64), (192, 64), (300, 16), (512, 32)])
def test_general_kernel(dtype, D, page):
    """fp32, wide and odd heads, odd pages."""
    s = make([0, 1, 9, 64, 65, 333], 6, 2, D, page=page, dtype=dtype)
    vec = dtype != torch.float32 and D % 8 == 0 and D <= 128 and page % 16 == 0
    check(s, None, 20.0, slope_table(6), roundings=2 if vec else 1)
    check(s, 40, roundings=2 if vec else 1)


@gpu
def test_strides():
    """A pool that holds keys and values side by side, queries and new rows inside a projection, a table of a wider one; rows that are not aligned."""
    s = make([70, 130], 4, 2, 64)
    want = check(s)
    P, page, G, D = s["k"].shape
    pool = torch.stack([s["k"], s["v"]], dim=3)
    qkv = torch.cat([s["q"].reshape(2, -1), s["k_new"].reshape(2, -1), s["v_new"].reshape(2, -1)], 1)
    wide = torch.stack([s["table"], s["table"]], 2)
    got = ops.paged_attention(qkv[:, :256].view(2, 4, 64), pool[:, :, :, 0], pool[:, :, :, 1], wide[:, :, 0], s["lengths"], k_new=qkv[:, 256:384].view(2, 2, 64),
                              v_new=qkv[:, 384:].view(2, 2, 64))
    assert torch.equal(got, want)
    flat = torch.empty(s["q"].numel() + 1, dtype=s["q"].dtype, device="cuda")[1:].view_as(s["q"]).copy_(s["q"])
    off = ops.paged_attention(flat, s["k"], s["v"], s["table"], s["lengths"], k_new=s["k_new"], v_new=s["v_new"])
    assert ((off.double() - want.double()).norm() / want.double().norm()).item() < 4 * 2.0 ** -8


@gpu
def test_pages_and_lengths_that_are_none():
    """A page number outside the pool hides its keys, a length outside the table is clipped: the error word says so, and nothing is stored there."""
    from linear_moe_b200.ops import gemm
    for dtype in (torch.bfloat16, torch.float32):
        s = make([200, 200, 130], 4, 2, 64, dtype=dtype, stale=0.0)
        s["table"][0, 1], s["table"][1, 3] = s["k"].shape[0], -1       # in the middle; the page of the new token
        k0, v0 = s["k"].clone(), s["v"].clone()
        got = ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], k_new=s["k_new"], v_new=s["v_new"])
        with pytest.raises(RuntimeError, match="0x12000"):
            gemm.check_error()
        gemm.check_error()
        assert torch.isfinite(got).all()
        # request 0 without its second page, request 1 without its last
        for b, keep in ((0, list(range(64)) + list(range(128, 200))), (1, list(range(192)))):
            at = s["table"][b].long().clamp(0, s["k"].shape[0] - 1)
            kb, vb = (t[at].flatten(0, 1)[keep].double().repeat_interleave(2, 1) for t in (s["k"], s["v"]))
            p = torch.softmax(torch.einsum("hd,jhd->hj", s["q"][b].double(), kb) / 8, -1)
            w = torch.einsum("hj,jhd->hd", p, vb)
            assert ((got[b].double() - w).norm() / w.norm()).item() < 2 * 2.0 ** -8
        k0[s["table"][0, 3].long(), 199 % 64], v0[s["table"][0, 3].long(), 199 % 64] = s["k_new"][0], s["v_new"][0]
        k0[s["table"][2, 2].long(), 129 % 64], v0[s["table"][2, 2].long(), 129 % 64] = s["k_new"][2], s["v_new"][2]
        assert torch.equal(s["k"], k0) and torch.equal(s["v"], v0)
        s = make([100], 2, 1, 64, dtype=dtype, stale=0.0)
        s["table"][0] = torch.tensor([0, 1, 2], device="cuda")
        s["lengths"][0] = 10 ** 9
        got = ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"])
        with pytest.raises(RuntimeError, match="0x11000"):
            gemm.check_error()
        s["lengths"][0] = 192
        assert torch.equal(got, ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"]))
        s["lengths"][0] = -5
        assert (ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"]) == 0).all()
        with pytest.raises(RuntimeError, match="0x11000"):
            gemm.check_error()


@gpu
def test_captured_steps_grow():
    """A captured step goes on over page borders and splits as the lengths on the device grow; two graphs in turn, another stream."""
    s = make([60, 250, 1], 8, 2, 64, spare=20)
    for b in range(3):
        n = -(-int(s["lengths"][b]) // 64)
        s["table"][b, n:] = 0
    free = [p for p in range(s["k"].shape[0]) if p not in {int(s["table"][b, i]) for b in range(3) for i in range(-(-int(s["lengths"][b]) // 64))}]
    for b in range(3):
        n = -(-int(s["lengths"][b]) // 64)
        for i in range(n, s["table"].shape[1]):
            s["table"][b, i] = free.pop()
    k, v = s["k"].clone(), s["v"].clone()
    args = lambda: (s["q"], s["k"], s["v"], s["table"], s["lengths"])      # noqa: E731
    kw = dict(k_new=s["k_new"], v_new=s["v_new"], softcap=30.0)
    ops.paged_attention(*args(), **kw)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = ops.paged_attention(*args(), **kw)
        graphs.append((g, o))
    s["k"].copy_(k), s["v"].copy_(v)
    for step in range(9):
        g, o = graphs[step % 2]
        e = {x: y.clone() for x, y in s.items()}
        g.replay()
        want, mag, low, kk, vv = formula(e, cap=30.0)
        assert ((o.double() - want).abs() <= 2.25 * 2.0 ** -8 * mag + 1e-30).all()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = ops.paged_attention(*(e[x] for x in ("q", "k", "v", "table", "lengths")), k_new=e["k_new"], v_new=e["v_new"], softcap=30.0)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(o, other)
        s["lengths"] += 1
        for x in ("q", "k_new", "v_new"):
            s[x].normal_()


@gpu
def test_shared_pages_and_far_offsets():
    """Two requests on the same pages, and a pool whose offsets pass 2^31 elements."""
    P = (1 << 31) // (64 * 128) + 4                            # 4.3 GB a pool
    k, v = (torch.zeros(P, 64, 1, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    s = make([200, 200], 4, 1, 128)
    at = s["table"][0, :4].long()
    far = torch.arange(P - 4, P, device="cuda")
    k[far], v[far] = s["k"][at].nan_to_num(), s["v"][at].nan_to_num()
    k[far[3], 7], v[far[3], 7] = s["k_new"][0], s["v_new"][0]
    table = far.int().expand(2, 4).contiguous()
    got = ops.paged_attention(s["q"][:1].expand(2, 4, 128), k, v, table, s["lengths"])
    assert torch.equal(got[0], got[1])
    assert torch.equal(got[0], check(s)[0])


@gpu
def test_window_beyond_32_bits():
    """More keys than the cache can have: no window at all."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(*s, generator=gen, device="cuda").bfloat16() for s in ((2, 4, 64), (6, 64, 2, 64), (6, 64, 2, 64)))
    table, lengths = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device="cuda"), torch.tensor([150, 7], dtype=torch.int32, device="cuda")
    for x, y, z in ((q, k, v), (q.float(), k.float(), v.float())):
        assert torch.equal(ops.paged_attention(x, y, z, table, lengths, window=1 << 40), ops.paged_attention(x, y, z, table, lengths))


@gpu
@pytest.mark.parametrize("heads", [(8, 2), (16, 4), (32, 2)])
def test_only_the_result_is_rounded(heads):
    """bf16, few keys of similar weights: the weights' roundings would be as large as the result's, u / sqrt(3) x sqrt(0.54) = 0.42 u in root mean square (numbers spread evenly over a
    power of two), 0.6 u together.  Their remainders go into the products too, so the result's own are left."""
    (H, G), D, n = heads, 128, 300
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(*s, generator=gen, device="cuda").bfloat16() for s in ((4, H, D), (20, 64, G, D), (20, 64, G, D)))
    table, lengths = torch.arange(20, dtype=torch.int32, device="cuda").view(4, 5), torch.full((4,), n, dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, k, v, table, lengths).double()
    kk, vv = (t.view(4, 320, G, D)[:, :n].double().repeat_interleave(H // G, 2) for t in (k, v))
    want = torch.einsum("bhj,bjhd->bhd", torch.softmax(torch.einsum("bhd,bjhd->bhj", q.double(), kk) * D ** -0.5, -1), vv)
    assert ((got - want).norm() / want.norm()).item() < 0.5 * torch.finfo(torch.bfloat16).eps / 2
