"""Attention with capped scores, a bias by distance and a range of keys per query, against the formulas in 64 bits.

Bounds.  u = finfo(type).eps / 2 is the largest relative error of one rounding.  An output is a sum of p v whose weights are rounded once and which
is rounded itself: elementwise |error| <= 2 u sum p |v|.  dv likewise.  ds = p (dp - delta) (1 - tanh^2) is rounded once, and delta is taken from the rounded output
(2 u more of its terms), so dq and dk stay within 4 u of the sums of their terms' magnitudes.  A quarter of u on top covers the 32-bit part: scores of up to 60
to 2^-24 of their terms, 2e-7 of the cap in tanh, exp2 to 2^-22.
In fp16 a number below 2^-14 is rounded by up to 2^-25 whatever its size: half the distance 2^-24 of the subnormals.  Weights are rounded in units of a maximum that is at
most the row's sum, so a normalised weight is off by at most max(u p, 2^-25) and ds by max(u ds, 2^-25): the bounds get 2^-25 times the sums of the
magnitudes of the visible v, k, q and do.  (A key whose weights all lie below 2^-14 has a dv of which u times its terms is less than that.)
In bf16 the same holds for 2^-126, below which 32-bit numbers are flushed to zero (weights of far keys under a steep bias).
The bounds by magnitudes would let a wrong key among hundreds pass, so the relative error in the 2-norm is held to 2 u and 4 u as well: errors of single roundings have no common
sign and their squares add up to less."""
import math

import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.ops import scored_attn as SA
from linear_moe_b200.ref import ops as R

gpu = pytest.mark.gpu


def visible(Tq, Tk, causal, off, window, first, stop, device):
    i, j = torch.arange(Tq, device=device)[:, None] + off, torch.arange(Tk, device=device)[None]
    m = torch.ones(1, Tq, Tk, dtype=torch.bool, device=device)
    if causal:
        m = m & (j <= i)
        if window:
            m = m & (j > i - window)
    if first is not None:
        m = m & (j >= first[:, :, None])
    if stop is not None:
        m = m & (j < stop[:, :, None])
    return m[:, None], (i - j).abs().double()


def forward64(q, k, v, scale, cap, slopes, seen, dist):
    rep = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(rep, 2), v.repeat_interleave(rep, 2)
    x = torch.einsum("bihd,bjhd->bhij", q, k) * scale
    t = torch.tanh(x / cap) if cap else torch.zeros_like(x)
    x = cap * t if cap else x
    if slopes is not None:
        x = x - slopes.double()[:, None, None] * dist
    p = torch.nan_to_num(torch.softmax(x.masked_fill(~seen, -math.inf), -1))
    return torch.einsum("bhij,bjhd->bihd", p, v), p, t, k, v


def formulas(q, k, v, do, scale, cap, slopes, seen, dist):
    """(results, sums of their terms' magnitudes, sums of what the weights multiply) of o, dq, dk, dv."""
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    G = k.shape[2]
    o, p, t, kr, vr = forward64(q, k, v, scale, cap, slopes, seen, dist)
    own = lambda x: x.unflatten(2, (G, -1)).sum(3)            # noqa: E731  sums over the query heads of a key head
    dp, delta = torch.einsum("bihd,bjhd->bhij", do, vr), (do * o).sum(-1).transpose(1, 2)[..., None]
    ds = p * (dp - delta) * (1 - t * t) * scale
    s1 = seen.double().expand_as(p)
    res = [o, torch.einsum("bhij,bjhd->bihd", ds, kr), own(torch.einsum("bhij,bihd->bjhd", ds, q)), own(torch.einsum("bhij,bihd->bjhd", p, do))]
    mo = torch.einsum("bhij,bjhd->bihd", p, vr.abs())
    md = (do.abs() * mo).sum(-1).transpose(1, 2)[..., None]
    ms = p * (torch.einsum("bihd,bjhd->bhij", do.abs(), vr.abs()) + md) * (1 - t * t) * scale
    mag = [mo, torch.einsum("bhij,bjhd->bihd", ms, kr.abs()), own(torch.einsum("bhij,bihd->bjhd", ms, q.abs())),
           own(torch.einsum("bhij,bihd->bjhd", p, do.abs()))]
    low = [torch.einsum("bhij,bjhd->bihd", s1, vr.abs()), scale * torch.einsum("bhij,bjhd->bihd", s1, kr.abs()),
           own(scale * torch.einsum("bhij,bihd->bjhd", s1, q.abs())), own(torch.einsum("bhij,bihd->bjhd", s1, do.abs()))]
    return res, mag, low


def check(got, res, mag, low, dtype, names=("o", "dq", "dk", "dv")):
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    for name, g, w, m, z in zip(names, got, res, mag, low):
        n = 2 if name in ("o", "dv") else 4
        assert g.dtype == dtype and g.shape == w.shape
        assert torch.isfinite(g).all(), name
        over = ((g.double() - w).abs() - (n + 0.25) * u * m - tiny * (z + 1)).max().item() if g.numel() else 0.0
        assert over <= 0, (name, over)
        if w.norm() > 1e-2 * m.norm():                        # else a difference of equal terms: only the bound above says something
            rel = ((g.double() - w).norm() / w.norm()).item()
            assert rel < n * u, (name, rel / u)


def inputs(B, Tq, Tk, Hq, Hkv, D, dtype, device="cuda", size=1.5, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, device=device)          # noqa: E731
    return ((n(B, Tq, Hq, D) * size).to(dtype), n(B, Tk, Hkv, D).to(dtype), n(B, Tk, Hkv, D).to(dtype), n(B, Tq, Hq, D).to(dtype))


def run(q, k, v, do, scale=None, causal=True, off=0, window=None, **kw):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = ops.softmax_attention(q, k, v, scale, causal, off, window, **kw)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]


def compare(q, k, v, do, causal=True, off=0, window=None, cap=None, slopes=None, first=None, stop=None, scale=None):
    from linear_moe_b200.ops import gemm
    got = run(q, k, v, do, scale, causal, off, window, softcap=cap, slopes=slopes, key_first=first, key_stop=stop)
    gemm.check_error()
    seen, dist = visible(q.shape[1], k.shape[1], causal, off, window, first, stop, q.device)
    check(got, *formulas(q, k, v, do, scale or q.shape[3] ** -0.5, cap, slopes, seen, dist), q.dtype)
    return got


def packed(B, T, lens, device="cuda"):
    first = torch.zeros(B, T, dtype=torch.int32)
    for b in range(B):
        row, at = lens[b % len(lens)], 0
        while at < T:
            for n in row:
                first[b, at:at + n] = at
                at += n
                if at >= T:
                    break
    return first.to(device)


def slope_table(H, device="cuda"):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=device)


# ---- on the CPU -----------------------------------------------------------------------------------------------------------------
def test_formulas_against_differences():
    """The gradients that the kernels are held to, against differences of the forward formula."""
    torch.manual_seed(0)
    q, k, v = (torch.randn(1, n, h, 4, dtype=torch.float64, requires_grad=True) for n, h in ((5, 4), (6, 2), (6, 2)))
    first = torch.tensor([[0, 0, 2, 5, 2]], dtype=torch.int32)
    seen, dist = visible(5, 6, True, 1, None, first, None, "cpu")
    f = lambda q, k, v: forward64(q, k, v, 0.7, 2.0, slope_table(4, "cpu"), seen, dist)[0]       # noqa: E731
    assert torch.autograd.gradcheck(f, (q, k, v))
    do = torch.randn(1, 5, 4, 4, dtype=torch.float64)
    want = torch.autograd.grad(f(q, k, v), (q, k, v), do)
    for a, b in zip(formulas(q, k, v, do, 0.7, 2.0, slope_table(4, "cpu"), seen, dist)[0][1:], want):
        assert torch.allclose(a, b, atol=1e-12)


@pytest.mark.parametrize("cap,bias,causal", [(None, False, True), (3.0, False, True), (None, True, True), (3.0, True, False)])
def test_eager_definition(cap, bias, causal):
    """CPU tensors run the eager form: fp32 against the formulas in 64 bits, rows that see nothing among them."""
    q, k, v, do = inputs(2, 9, 11, 4, 2, 6, torch.float32, "cpu")
    first, stop = torch.randint(0, 6, (2, 9), dtype=torch.int32), torch.randint(4, 12, (2, 9), dtype=torch.int32)
    first[0, 3], stop[0, 3] = 7, 7
    sl = slope_table(4, "cpu") if bias else None
    got = run(q, k, v, do, None, causal, 2, None, softcap=cap, slopes=sl, key_first=first, key_stop=stop)
    seen, dist = visible(9, 11, causal, 2, None, first, stop, "cpu")
    res, mag, _ = formulas(q, k, v, do, 6 ** -0.5, cap, sl, seen, dist)
    for g, w, m in zip(got, res, mag):
        assert ((g.double() - w).abs() <= 64 * 2.0 ** -24 * m + 1e-30).all()
    assert got[0][0, 3].abs().max() == 0 and got[1][0, 3].abs().max() == 0


def test_range_builders():
    E = 9
    tok = torch.tensor([[1, 2, E, 3, E, E, 4], [E, 1, 1, 1, 1, 1, E]])
    assert ops.document_first(tok, E).tolist() == [[0, 0, 0, 3, 3, 5, 6], [0, 1, 1, 1, 1, 1, 1]]
    assert ops.document_first(tok, E).dtype == torch.int32
    assert ops.prefix_stop(5, [3, 0], [5, 2]).tolist() == [[3, 3, 3, 4, 5], [1, 2, 0, 0, 0]]
    assert ops.prefix_stop(3, [9]).tolist() == [[9, 9, 9]]
    assert ops.prefix_stop(3, [9], [2]).tolist() == [[2, 2, 0]]


def test_refusals():
    q, k, v, _ = inputs(2, 4, 4, 4, 2, 8, torch.float32, "cpu")
    f = torch.zeros(2, 4, dtype=torch.int32)
    sl = slope_table(4, "cpu")
    bad = [dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=math.inf), dict(softcap=math.nan), dict(slopes=sl[:3]), dict(slopes=sl.double()),
           dict(slopes=sl.clone().requires_grad_(True)), dict(key_first=f.long()), dict(key_first=f[:1]), dict(key_stop=f[:, :3]),
           dict(key_first=f, window=0), dict(key_first=f, window=3, causal=False), dict(key_first=f, scale=0.0), dict(key_first=f, scale=math.nan)]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.softmax_attention(q, k, v, **kw)
    for a, b, c in [(q[0], k, v), (q[:1], k, v), (q, k[:, :3], v), (q, k[..., :4], v), (q[:, :, :3], k, v), (q, k, v.double()), (q, k[:, :, :0], v[:, :, :0])]:
        with pytest.raises(ValueError):
            ops.softmax_attention(a, b, c, softcap=5.0)


def test_empty_tensors():
    for B, Tq, Tk in [(0, 3, 3), (2, 0, 3), (2, 3, 0)]:
        q, k, v, do = inputs(B, Tq, Tk, 2, 1, 8, torch.bfloat16, "cpu")
        got = run(q, k, v, do, softcap=5.0, key_first=torch.zeros(B, Tq, dtype=torch.int32))
        assert [g.shape for g in got] == [q.shape, q.shape, k.shape, v.shape] and all((g == 0).all() for g in got)


def test_strides_of_views():
    """What a tensor map gets: dimensions of one take a dense stride, others are refused (and copied) where they are broadcast or not aligned."""
    t = torch.zeros(1, 5, 2, 64, dtype=torch.bfloat16)
    assert list(SA._strides(t.as_strided((1, 5, 2, 64), (3, 128, 64, 1)))) == [640, 128, 64]
    assert SA._strides(torch.zeros(1, 5, 2, 64).bfloat16().expand(3, 5, 2, 64)) is None
    assert SA._strides(torch.zeros(2, 5, 2, 68).bfloat16()[..., :64]) is None
    assert SA._strides(torch.zeros(2, 5, 2, 64, 2).bfloat16()[..., 0]) is None
    laid = SA._laid_out(torch.ones(1, 5, 2, 64).bfloat16().expand(3, 5, 2, 64))
    assert list(SA._strides(laid)) == [640, 128, 64] and laid.shape == (3, 5, 2, 64) and (laid == 1).all()
    off = SA._laid_out(torch.zeros(641).bfloat16()[1:].view(1, 5, 2, 64))
    assert off.data_ptr() % 16 == 0


# ---- on the GPU -----------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [8, 64, 72, 128])
@pytest.mark.parametrize("T", [1, 127, 128, 129, 300])
def test_documents(dtype, D, T):
    """Packed documents of every length around the tiles, with caps."""
    q, k, v, do = inputs(2, T, T, 4, 2, D, dtype, size=4.0)
    compare(q, k, v, do, cap=20.0, first=packed(2, T, [[1, 2, 60, 65], [128, 7]]))


@gpu
@pytest.mark.parametrize("cap,bias", [(None, False), (None, True), (30.0, False), (30.0, True)])
@pytest.mark.parametrize("heads", [(1, 1), (6, 2), (8, 1), (3, 3)])
def test_scores_and_heads(cap, bias, heads):
    q, k, v, do = inputs(2, 257, 257, *heads, 64, torch.bfloat16, size=4.0)
    compare(q, k, v, do, cap=cap, slopes=slope_table(heads[0]) if bias else None, first=packed(2, 257, [[100, 30], [257]]))


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk,off,window", [(1, 513, 512, None), (130, 700, 570, None), (300, 300, 0, 1), (513, 513, 0, 129), (64, 1000, 200, 300),
                                              (200, 100, 0, None), (150, 400, -100, None)])
def test_offsets_and_windows(D, Tq, Tk, off, window):
    """Causal with an offset and a window, and queries in front of the first key or behind the last one."""
    q, k, v, do = inputs(1, Tq, Tk, 4, 2, D, torch.bfloat16)
    compare(q, k, v, do, off=off, window=window, cap=50.0)
    compare(q, k, v, do, off=off, window=window, slopes=slope_table(4))
    compare(q, k, v, do, off=off, window=window, stop=torch.full((1, Tq), Tk - 3, dtype=torch.int32, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefixes_and_padding(dtype):
    T = 391
    q, k, v, do = inputs(4, T, T, 4, 2, 64, dtype)
    stop = ops.prefix_stop(T, [0, 130, 256, 50], [T, 200, 257, 1], "cuda")
    got = compare(q, k, v, do, causal=False, stop=stop)
    for b, n in enumerate((T, 200, 257, 1)):                   # padded queries and keys take and give nothing
        assert all((t[b, n:] == 0).all() for t in got)
    compare(q, k, v, do, causal=False, stop=stop, slopes=slope_table(4))
    compare(q, k, v, do, causal=False, slopes=slope_table(4))


@gpu
def test_ranges_of_any_kind():
    """Ranges in no order, empty ones, whole tiles of empty ones, and numbers outside the keys."""
    T = 520
    q, k, v, do = inputs(3, T, T, 2, 1, 64, torch.bfloat16)
    gen = torch.Generator().manual_seed(1)
    first = torch.randint(-50, T + 50, (3, T), generator=gen, dtype=torch.int32)
    stop = first + torch.randint(-5, 400, (3, T), generator=gen, dtype=torch.int32)
    stop[1, 128:400] = 0
    first[2], stop[2] = 2 ** 31 - 1, -2 ** 31
    first, stop = first.cuda(), stop.cuda()
    got = compare(q, k, v, do, causal=False, first=first, stop=stop)
    assert all((t[2] == 0).all() for t in got)
    compare(q, k, v, do, causal=True, window=200, cap=10.0, first=first, stop=stop)
    # keys that no query sees get exact zeros
    none = torch.zeros(3, T, dtype=torch.int32, device="cuda")
    got = compare(q, k, v, do, causal=False, stop=none + 130)
    assert (got[2][:, 130:] == 0).all() and (got[3][:, 130:] == 0).all()


@gpu
@pytest.mark.parametrize("dtype,D,heads,cap,bias", [(torch.bfloat16, 128, (16, 4), 30.0, False), (torch.bfloat16, 64, (24, 12), None, True), (torch.float16, 128, (12, 2), 50.0, True),
                                                    (torch.bfloat16, 96, (20, 20), None, False)])
def test_more_tiles_than_ctas(dtype, D, heads, cap, bias):
    """Several hundred tiles of queries, which the CTAs work through: none to twelve key tiles each, in turns, so that every ring and phase meets every other one; key heads with shares of four, two and
    one CTAs."""
    B, T = 3, 1500
    q, k, v, do = inputs(B, T, T, *heads, D, dtype, size=3.0)
    first = packed(B, T, [[700, 3, 120, 40], [128, 256, 1, 127], [1500]])
    stop = torch.full((B, T), T, dtype=torch.int32, device="cuda")
    stop[0, 128:384] = 0                                       # whole tiles that see nothing
    stop[1, ::2] = 0
    stop[2, 1408:] = 700
    sl = slope_table(heads[0]) if bias else None
    a = compare(q, k, v, do, cap=cap, slopes=sl, first=first, stop=stop)
    for _ in range(3):
        b = run(q, k, v, do, softcap=cap, slopes=sl, key_first=first, key_stop=stop)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
def test_views_and_copies():
    """Views into a fused projection, broadcast batches, an unaligned base, heads in front of tokens; ranges that are views too."""
    B, T, H, G, D = 2, 200, 4, 2, 64
    torch.manual_seed(3)
    qkv = torch.randn(B, T, G, H // G + 2, D, device="cuda").bfloat16()
    q, k, v = qkv[:, :, :, :2].reshape(B, T, H, D), qkv[:, :, :, 2], qkv[:, :, :, 3]
    do = torch.randn(B, H, T, D, device="cuda").bfloat16().transpose(1, 2)
    first = packed(1, T, [[33, 80]]).expand(B, T)
    a = compare(q, k, v, do, cap=15.0, first=first)
    flat = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view_as(q).copy_(q)
    wide = torch.zeros(B, 2 * T, dtype=torch.int32, device="cuda")
    wide[:, ::2] = first
    b = compare(flat, k.contiguous(), v.transpose(1, 2).contiguous().transpose(1, 2), do.contiguous(), cap=15.0, first=wide[:, ::2])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    compare(q, k[:1].expand(B, T, G, D), v[:, :, :1].expand(B, T, G, D), do, cap=15.0, first=first)
    one = inputs(1, T, T, 2, 2, D, torch.bfloat16)
    compare(one[0].as_strided((1, T, 2, D), (3, 2 * D, D, 1)), *one[1:], cap=15.0)


@gpu
def test_same_bits_twice_and_in_a_graph():
    q, k, v, do = inputs(2, 333, 333, 4, 2, 128, torch.bfloat16)
    first = packed(2, 333, [[50, 130], [200]])
    kw = dict(softcap=30.0, key_first=first)
    want = run(q, k, v, do, **kw)
    assert all(torch.equal(a, b) for a, b in zip(want, run(q, k, v, do, **kw)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(q, k, v, do, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    hold = [t.clone() for t in (q, k, v, do)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*hold, **kw)
    for t in hold:
        t.zero_()
    graph.replay()
    assert all((t == 0).all() for t in out[:1])
    for t, s in zip(hold, (q, k, v, do)):
        t.copy_(s)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, out))


@gpu
def test_heads_the_kernels_do_not_take():
    """Wider heads and fp32 run the eager definition."""
    q, k, v, do = inputs(1, 70, 70, 2, 1, 192, torch.bfloat16)
    compare(q, k, v, do, cap=20.0)
    got = run(*(t.float() for t in (q, k, v, do)), softcap=20.0)
    seen, dist = visible(70, 70, True, 0, None, None, None, "cuda")
    for g, w in zip(got, formulas(q, k, v, do, 192 ** -0.5, 20.0, None, seen, dist)[0]):
        assert ((g.double() - w).norm() / w.norm()).item() < 1e-5


@gpu
def test_large_scores():
    """Scores far beyond the cap and beyond 2^10 without one."""
    q, k, v, do = inputs(1, 200, 200, 2, 2, 64, torch.bfloat16, size=100.0)
    got = run(q, k, v, do, softcap=5.0)
    seen, dist = visible(200, 200, True, 0, None, None, None, "cuda")
    pick = lambda x: [x[0], x[3]]                              # noqa: E731
    check(pick(got), *(pick(x) for x in formulas(q, k, v, do, 0.125, 5.0, None, seen, dist)), torch.bfloat16, ("o", "dv"))
    for t in run(q, k, v, do, slopes=slope_table(2)):
        assert torch.isfinite(t).all()


# ---- calls at the edges of what is allowed -------------------------------------------------------------------------------------------
def test_positions_that_do_not_fit():
    q, k, v, _ = inputs(1, 4, 4, 2, 1, 8, torch.float32, "cpu")
    for off in (1 << 30, -(1 << 30), 1 << 40):
        with pytest.raises(ValueError):
            ops.softmax_attention(q, k, v, q_offset=off, softcap=5.0)
    plain = ops.softmax_attention(q, k, v, softcap=5.0)
    assert torch.equal(ops.softmax_attention(q, k, v, window=1 << 40, softcap=5.0), plain)


@gpu
def test_window_beyond_32_bits():
    q, k, v, do = inputs(1, 200, 200, 2, 1, 64, torch.bfloat16)
    for a, b in zip(run(q, k, v, do, window=1 << 40, softcap=5.0), run(q, k, v, do, softcap=5.0)):
        assert torch.equal(a, b)


@gpu
def test_more_heads_than_the_kernels_take():
    compare(*inputs(1, 3, 3, 1024, 2, 8, torch.bfloat16), cap=20.0)


@gpu
def test_offsets_in_front_of_and_behind_the_keys():
    """No query sees a key; all see all of them."""
    q, k, v, do = inputs(2, 130, 140, 4, 2, 64, torch.bfloat16)
    for t in run(q, k, v, do, off=-200, slopes=slope_table(4)):
        assert (t == 0).all()
    compare(q, k, v, do, off=100000, slopes=slope_table(4))


@gpu
def test_gradient_of_a_sum():
    """The incoming gradient is one number, broadcast."""
    q, k, v, _ = inputs(1, 140, 140, 4, 2, 72, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(ops.softmax_attention(*leaves, softcap=20.0).sum(), leaves)
    want = run(q, k, v, torch.ones_like(q), softcap=20.0)[1:]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    (only,) = torch.autograd.grad(ops.softmax_attention(q.detach(), k, v.detach(), softcap=20.0).sum(), (k,))
    assert torch.equal(only, want[1])


@gpu
@pytest.mark.parametrize("D,Hkv", [(64, 1), (128, 2)])
def test_long_sequence(D, Hkv):
    """66000 queries, most of whose rows see a window in the middle of everything: pieces of the results against the formulas of the piece."""
    T, W = 66000, 100
    q, k, v, do = inputs(1, T, T, 2, Hkv, D, torch.bfloat16)
    sl = slope_table(2)
    got = run(q, k, v, do, window=W, slopes=sl)
    for t0 in (0, 32700, T - 512):
        cut = slice(t0, t0 + 512)
        seen, dist = visible(512, 512, True, 0, W, None, None, "cuda")
        parts = formulas(*(t[:, cut] for t in (q, k, v, do)), D ** -0.5, None, sl, seen, dist)
        lo, hi = (0 if t0 == 0 else W - 1), (512 if t0 + 512 == T else 512 - W + 1)          # keys whose queries all lie in the piece, and behind them queries whose keys do
        rows = lambda x: [x[0][:, lo:], x[1][:, lo:], x[2][:, lo:hi], x[3][:, lo:hi]]         # noqa: E731
        check(rows([g[:, cut] for g in got]), *(rows(x) for x in parts), torch.bfloat16)


@gpu
def test_two_graphs_at_once():
    """Two captured calls, replayed side by side on two streams: each has its own workspace."""
    jobs = []
    for seed in (1, 2):
        held = inputs(2, 400, 400, 8, 2, 128, torch.bfloat16, seed=seed)
        kw = dict(softcap=30.0, key_first=packed(2, 400, [[70, 150]]))
        want = run(*held, **kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(*held, **kw)
        jobs.append((graph, out, want, torch.cuda.Stream(), held, kw))              # (a graph reads the inputs that it was captured with)
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, _, _, stream, _, _ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _, _, _ in jobs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@gpu
@pytest.mark.parametrize("cap,bias", [(None, False), (None, True), (30.0, False), (50.0, False), (80.0, False), (50.0, True)])
def test_gradients_where_one_weight_is_large(cap, bias):
    """dq and dk are sums of  p (dp - do . o), a difference of nearly equal terms where one weight is close to 1.  All that should be left are two roundings in a row, of ds and of the
    result: rounding to u is off by u / sqrt(3) x sqrt(0.54) = 0.42 u in root mean square (numbers spread evenly over a power of two), twice that in squares is 0.59 u; the roundings of
    the weights in o, which the sum of many makes small, may add half as much in squares: sqrt(0.59^2 + 0.42^2) = 0.72 u.  An o that is off by the largest weight's rounding, or that
    is used as it was rounded, adds another 0.42 u or more to ds."""
    u = torch.finfo(torch.bfloat16).eps / 2
    q, k, v, do = inputs(1, 512, 512, 4, 2, 128, torch.bfloat16, size=4.0)
    sl = slope_table(4) if bias else None
    got = run(q, k, v, do, softcap=cap, slopes=sl, key_first=torch.zeros(1, 512, dtype=torch.int32, device="cuda"))
    seen, dist = visible(512, 512, True, 0, None, None, None, "cuda")
    res = formulas(q, k, v, do, 128 ** -0.5, cap, sl, seen, dist)[0]
    for name, g, w in zip(("dq", "dk"), got[1:3], res[1:3]):
        rel = ((g.double() - w).norm() / w.norm()).item()
        assert rel < 0.72 * u, (name, rel / u)


@gpu
@pytest.mark.parametrize("cap", [2.0, 4.0, 6.0, 8.0, 12.0, 200.0])
def test_scores_against_the_cap(cap):
    """Scores of 1.5 in root mean square, up to 7: below three quarters of the cap, up to one and a half times, and beyond, where tanh is evaluated in different ways."""
    compare(*inputs(1, 260, 260, 4, 2, 64, torch.bfloat16), cap=cap)
    compare(*inputs(1, 260, 260, 4, 2, 128, torch.float16), cap=cap)


def test_caps_and_scales_that_32_bits_do_not_hold():
    q, k, v, _ = inputs(1, 4, 4, 2, 1, 8, torch.float32, "cpu")
    for kw in (dict(softcap=1e-40), dict(softcap=1e39), dict(softcap=5.0, scale=1e-40), dict(softcap=5.0, scale=1e39)):
        with pytest.raises(ValueError):
            ops.softmax_attention(q, k, v, **kw)


@gpu
def test_ranges_at_the_ends_of_their_type():
    """Beside rows that see something, rows whose ranges end or begin at the smallest and the largest number."""
    q, k, v, do = inputs(1, 200, 300, 2, 1, 64, torch.bfloat16)
    big, small = 2 ** 31 - 1, -2 ** 31
    first = torch.tensor([[0, big, small, small, 100][i % 5] for i in range(200)], dtype=torch.int32, device="cuda")[None]
    stop = torch.tensor([[300, big, small, big, small][i % 5] for i in range(200)], dtype=torch.int32, device="cuda")[None]
    for causal in (False, True):
        compare(q, k, v, do, causal=causal, off=60, first=first, stop=stop)
    compare(q, k, v, do, off=-100, window=2 ** 31 - 1, first=first)
