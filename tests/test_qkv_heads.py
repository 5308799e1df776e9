"""Heads of a fused projection (norm, rotation, backward) against the formula in 64 bits.

Bounds.  u = finfo(type).eps / 2 is the largest relative error of one rounding; every number is rounded once.  What 32 bits cost on the way, with e = 2^-24 a rounding of their own: a sum of n terms, 32 lanes
of them side by side, is off by (n / 32 + 6) e of its terms' magnitudes, the norm's factor by half of that and three roundings; a rotation by three roundings of |y_a| + |y_b|.  fp16 numbers below 2^-14 are
rounded by up to 2^-25 whatever their size.  A weight's gradient is a sum over all tokens and heads: e times the longest chain of additions (a lane's items, eight warps, the blocks' parts) of its terms'
magnitudes, and each term is off by the roundings above."""
import math

import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.ops import gemm

gpu = pytest.mark.gpu
E = 2.0 ** -24


def make(B, T, G, r, D, R=None, norm=True, at=None, dtype=torch.float32, device="cpu", seed=0, w_dtype=None, at_type=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen)            # noqa: E731
    s = dict(qkv=(n(B, T, G, r + 2, D) * 1.3).to(dtype), wq=None, wk=None, cos=None, sin=None, at=None)
    if norm:
        s["wq"], s["wk"] = ((1 + 0.2 * n(D)).to(w_dtype or dtype) for _ in range(2))
    R = D if R is None else R
    if R:
        turn = torch.arange(at or T)[:, None].double() * 10000.0 ** (-torch.arange(0, R, 2).double() / R)
        s["cos"], s["sin"] = turn.cos().float(), turn.sin().float()
        if at:
            s["at"] = torch.randint(0, at, (B, T), generator=gen).to(at_type)
    s["grads"] = [n(B, T, h, D).to(dtype) for h in (G * r, G, G)]
    return {k: [x.to(device) for x in v] if isinstance(v, list) else v if v is None else v.to(device) for k, v in s.items()}


def pair(x, R, interleaved):
    """The other number of every pair (nothing behind the first R)."""
    y = torch.zeros_like(x)
    if interleaved:
        y[..., 0:R:2], y[..., 1:R:2] = x[..., 1:R:2], x[..., 0:R:2]
    else:
        y[..., : R // 2], y[..., R // 2:R] = x[..., R // 2:R], x[..., : R // 2]
    return y


def formula(s, eps, interleaved):
    """Outputs and gradients in 64 bits (autograd on the formula), and what bounds their errors."""
    d = lambda t: None if t is None else t.detach().double()            # noqa: E731
    B, T, G, S, D = s["qkv"].shape
    x = d(s["qkv"]).requires_grad_()
    ws = [None if w is None else d(w).requires_grad_() for w in (s["wq"], s["wk"])]
    cos, sin, R = d(s["cos"]), d(s["sin"]), 0
    if cos is not None:
        R = 2 * cos.shape[1]
        at = s["at"].long() if s["at"] is not None else torch.arange(T, device=x.device).expand(B, T)
        c, n = (t[at][:, :, None] for t in (cos, sin))
        c, n = ((t.repeat_interleave(2, -1) if interleaved else torch.cat([t, t], -1)) for t in (c, n))
        sign = torch.ones(R, device=x.device, dtype=torch.float64)
        sign[(slice(0, R, 2) if interleaved else slice(0, R // 2))] = -1
    outs, room = [], []
    chain = D / 64 + 10
    for i, (h, w) in enumerate(((x[..., : S - 2, :].reshape(B, T, -1, D), ws[0]), (x[..., S - 2, :], ws[1]))):
        y = h if w is None else h * w / (h.square().mean(-1, keepdim=True) + eps).sqrt()
        z = y
        if cos is not None:
            z = torch.cat([y[..., :R] * c + sign * n * pair(y, R, interleaved)[..., :R], y[..., R:]], -1)
        outs.append(z)
        room.append(chain * E * (y.abs() + pair(y.abs(), R, interleaved)).detach())
    outs.append(x[..., S - 1, :])
    room.append(torch.zeros_like(outs[2]).detach())
    leaves = [x] + [w for w in ws if w is not None]
    grads = torch.autograd.grad(outs, leaves, [g.double() for g in s["grads"]])
    droom = torch.zeros_like(x).detach()
    wroom = []
    for i, (h, w) in enumerate(((x[..., : S - 2, :].reshape(B, T, -1, D), ws[0]), (x[..., S - 2, :], ws[1]))):
        h, g = h.detach(), s["grads"][i].double().abs()
        g = g + pair(g, R, interleaved)
        if w is None:
            bound = 4 * E * g
        else:
            inv = 1 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
            xh, gw = h.abs() * inv, g * w.detach().abs()
            bound = (D / 32 + 16) * E * inv * (gw + xh * (gw * xh).mean(-1, keepdim=True))
            wroom.append((g * xh).sum((0, 1, 2)))
        (droom[..., : S - 2, :] if i == 0 else droom[..., S - 2, :]).copy_(bound.view(B, T, G, S - 2, D) if i == 0 else bound)
    items = B * T * G * S
    longest = items / (8 * max(1, min(-(-items // 8), 8 * 148))) + 8 + 8 * 148 / 16 + 16
    return [o.detach() for o in outs], room, grads, [droom] + [(longest + D / 32 + 16) * E * t for t in wroom]


def close(got, want, room, what):
    u = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bad = (got.double() - want).abs() - (u * (want.abs() + room) + room + tiny)
    assert got.isfinite().all() and bad.max() <= 0, (what, float(bad.max()))


def check(s, eps=1e-6, interleaved=False):
    leaves = [s[k].requires_grad_() for k in ("qkv", "wq", "wk") if s[k] is not None]
    outs = ops.qkv_heads(s["qkv"], s["wq"], s["wk"], eps, s["cos"], s["sin"], positions=s["at"], interleaved=interleaved)
    grads = torch.autograd.grad(outs, leaves, s["grads"])
    want, room, wgrads, groom = formula(s, eps, interleaved)
    for got, w, r, n in zip(outs, want, room, "qkv"):
        close(got, w, r, n)
    for got, w, r, n in zip(grads, wgrads, groom, ("dqkv", "dwq", "dwk")):
        close(got, w, r, n)
    return outs, grads


SHAPES = [(1, 1, 1, 1, 2), (2, 7, 2, 3, 6), (1, 3, 1, 1, 40), (2, 65, 2, 2, 64), (3, 33, 4, 3, 96), (1, 50, 8, 4, 128), (2, 5, 1, 7, 80), (1, 9, 2, 2, 256), (1, 4, 2, 1, 513), (1, 3, 1, 2, 1024)]


@pytest.mark.parametrize("shape", SHAPES[:5])
@pytest.mark.parametrize("interleaved", [False, True])
def test_the_eager_form(shape, interleaved):
    check(make(*shape, R=shape[4] // 2 * 2), interleaved=interleaved)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, interleaved, dtype):
    check(make(*shape, R=shape[4] // 2 * 2, dtype=dtype, device="cuda"), interleaved=interleaved)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(64, 0), (64, 2), (64, 6), (64, 16), (96, 32), (96, 48), (128, 16), (128, 64), (128, 126), (256, 64)])
def test_a_part_of_the_head_turns(D, R, interleaved, dtype):
    check(make(2, 19, 2, 3, D, R=R, dtype=dtype, device="cuda", at=77 if R else None, at_type=torch.int32), interleaved=interleaved)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_without_norms(dtype):
    check(make(2, 31, 2, 2, 64, norm=False, dtype=dtype, device="cuda"))
    s = make(2, 31, 2, 2, 64, dtype=dtype, device="cuda")
    s["wk"] = None
    check(s)
    s = make(2, 31, 2, 2, 64, R=0, dtype=dtype, device="cuda")
    s["wq"] = None
    check(s)


@gpu
def test_weights_of_another_type():
    check(make(2, 31, 2, 2, 128, dtype=torch.bfloat16, w_dtype=torch.float32, device="cuda"))
    check(make(2, 31, 2, 2, 64, dtype=torch.float32, w_dtype=torch.bfloat16, device="cuda"))
    check(make(2, 31, 2, 2, 64, dtype=torch.float16, w_dtype=torch.bfloat16, device="cuda"))


@gpu
@pytest.mark.parametrize("rows", [(1, 4099), (4, 1500)])
def test_many_rows(rows):
    """More heads than the blocks of a launch, so that blocks go on to the next ones."""
    check(make(*rows, 4, 3, 128, dtype=torch.bfloat16, device="cuda"))


@gpu
def test_sizes_of_the_numbers():
    """Rows of zeros, tiny and huge ones: epsilon, and squares that 32 bits still hold."""
    for size, eps in ((0.0, 1e-6), (1e-4, 1e-6), (1e4, 1e-6), (1e-3, 0.0), (1e15, 1e-6)):
        s = make(1, 5, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
        s["qkv"] = s["qkv"] * size
        check(s, eps)


@gpu
@pytest.mark.parametrize("D", [64, 80])
def test_strides(D):
    s = make(3, 9, 2, 2, D, dtype=torch.bfloat16, device="cuda")
    want, grads = check(dict(s))
    wide = torch.full((3, 9, 2 * 4 * D + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    views = [wide[..., 8:8 + 8 * D].unflatten(-1, (2, 4, D)), wide[..., 3:3 + 8 * D].unflatten(-1, (2, 4, D)), torch.empty(9, 3, 2, 4, D, dtype=torch.bfloat16, device="cuda").transpose(0, 1),
             torch.empty(3, 9, 4, 2, D, dtype=torch.bfloat16, device="cuda").transpose(2, 3)]
    for view in views:
        view.copy_(s["qkv"].detach())
        leaf = view.detach().requires_grad_()
        got = ops.qkv_heads(leaf, s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])
        (dx,) = torch.autograd.grad(got, leaf, [g.transpose(1, 2).contiguous().transpose(1, 2) for g in s["grads"]])
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(dx, grads[0])


@gpu
@pytest.mark.parametrize("used", [(0,), (1,), (2,), (0, 2)])
def test_outputs_that_nothing_uses(used):
    s = make(2, 17, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    leaves = [s[k].requires_grad_() for k in ("qkv", "wq", "wk")]
    outs = ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])
    got = torch.autograd.grad([outs[i] for i in used], leaves, [s["grads"][i] for i in used])
    zero = [g if i in used else torch.zeros_like(g) for i, g in enumerate(s["grads"])]
    outs = ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])
    want = torch.autograd.grad(outs, leaves, zero)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@gpu
def test_a_weight_of_queries_and_keys():
    """One tensor in both places gets both gradients; frozen ones get none."""
    s = make(2, 17, 2, 2, 64, dtype=torch.float32, device="cuda")
    args = (1e-6, s["cos"], s["sin"])
    two = [s["wq"].clone().requires_grad_() for _ in range(2)]
    torch.autograd.backward(ops.qkv_heads(s["qkv"], *two, *args), s["grads"])
    one = s["wq"].clone().requires_grad_()
    torch.autograd.backward(ops.qkv_heads(s["qkv"], one, one, *args), s["grads"])
    assert torch.equal(one.grad, two[0].grad + two[1].grad) and s["qkv"].grad is None
    x, w = s["qkv"].clone().requires_grad_(), s["wk"].clone().requires_grad_()
    torch.autograd.backward(ops.qkv_heads(x, s["wq"], w, *args), s["grads"])
    assert x.grad is not None and w.grad is not None and s["wq"].grad is None


@gpu
def test_differences():
    """The loss's slope along a direction, from the formula in 64 bits at two points: off by h^2 / 6 of its third derivative, far below what 32 bits leave of the gradient."""
    s = make(2, 11, 2, 2, 64, device="cuda", at=50)
    leaves = [s[k].requires_grad_() for k in ("qkv", "wq", "wk")]
    grads = torch.autograd.grad(ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"], positions=s["at"]), leaves, s["grads"])
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i, k in enumerate(("qkv", "wq", "wk")):
        way = torch.randn(s[k].shape, generator=gen, device="cuda", dtype=torch.float64)
        h, loss = 1e-4, []
        for sign in (1, -1):
            t = dict(s, **{k: s[k].detach().double() + sign * h * way})
            loss.append(sum((o * g.double()).sum() for o, g in zip(formula(t, 1e-6, False)[0], s["grads"])))
        slope, got = (loss[0] - loss[1]) / (2 * h), (grads[i].double() * way).sum()
        # roundings of the gradient's numbers, each 100 e of a few units at most, without a common sign; and 1e-8 for the difference
        assert abs(slope - got) <= 100 * E * float((grads[i].double().abs() + 1).square().mul(way.square()).sum().sqrt()) * 4 + 1e-6 * abs(slope)


@gpu
def test_the_same_every_time_and_on_another_stream():
    s = make(2, 700, 4, 2, 64, dtype=torch.bfloat16, device="cuda")
    a = check(s)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        b = check(s)
    st.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((*a[0], *a[1]), (*b[0], *b[1])))


@gpu
def test_captured():
    """A step's positions grow on the device; the replayed call goes on from them."""
    s = make(3, 1, 2, 2, 64, dtype=torch.bfloat16, device="cuda", at=90)
    call = lambda: ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"], positions=s["at"])            # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        s["at"].copy_((s["at"] + 1) % 90)
        s["qkv"].copy_(s["qkv"] * 1.1)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(out, call()))


def test_refusals():
    s = make(2, 5, 2, 2, 8)
    good = dict(qkv=s["qkv"], q_weight=s["wq"], k_weight=s["wk"], eps=1e-6, cos=s["cos"], sin=s["sin"])
    ops.qkv_heads(**good)
    for bad in (dict(qkv=s["qkv"][0]), dict(qkv=s["qkv"][..., :2, :]), dict(qkv=s["qkv"].double()), dict(q_weight=s["wq"][:4]), dict(k_weight=s["wk"].double()), dict(q_weight=s["wq"].bfloat16()),
                dict(eps=-1.0), dict(eps=float("nan")), dict(sin=None), dict(cos=None, sin=None, positions=torch.zeros(2, 5, dtype=torch.int64)), dict(cos=s["cos"].double(), sin=s["sin"].double()),
                dict(cos=s["cos"].repeat(1, 2), sin=s["sin"].repeat(1, 2)), dict(cos=s["cos"][:4], sin=s["sin"][:4]), dict(cos=s["cos"].clone().requires_grad_()),
                dict(positions=torch.zeros(2, 4, dtype=torch.int64)), dict(positions=torch.zeros(2, 5)), dict(positions=torch.full((2, 5), 5)), dict(positions=torch.full((2, 5), -1)),
                dict(qkv=torch.zeros(1, 1, 1, 3, 1025), q_weight=None, k_weight=None), dict(qkv=torch.zeros(1, 1, 1, 3, 0), q_weight=None, k_weight=None)):
        with pytest.raises(ValueError):
            ops.qkv_heads(**{**good, **bad})


def test_nothing():
    for B, T in ((0, 3), (2, 0)):
        s = make(B, T, 2, 2, 8)
        assert [t.shape for t in ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])] == [(B, T, 4, 8), (B, T, 2, 8), (B, T, 2, 8)]


@gpu
def test_nothing_and_positions_outside_on_the_gpu():
    for B, T in ((0, 3), (2, 0)):
        s = make(B, T, 2, 2, 8, device="cuda")
        x = s["qkv"].requires_grad_()
        outs = ops.qkv_heads(x, s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])
        assert [t.shape for t in outs] == [(B, T, 4, 8), (B, T, 2, 8), (B, T, 2, 8)]
        assert torch.autograd.grad(outs, x, s["grads"])[0].shape == x.shape
    for D in (64, 6):
        s = make(1, 2, 2, 2, D, device="cuda", at=9)
        gemm.check_error()
        for at, near in ((9, 8), (-1, 0), (1 << 40, 8)):
            s["at"][0, 1] = at
            got = ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"], positions=s["at"])
            with pytest.raises(RuntimeError, match="a position outside the tables"):
                gemm.check_error()
            s["at"][0, 1] = near
            assert all(torch.equal(x, y) for x, y in zip(got, ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"], positions=s["at"])))
    assert math.isfinite(float(got[0].float().sum()))


def test_divisions():
    """n / d as the kernel does it: a product's upper half, a sum that stays below 2^32, a shift."""
    from linear_moe_b200.ops.qkv_heads import _divisor
    gen = torch.Generator().manual_seed(0)
    for d in [1, 2, 3, 5, 7, 8, 31, 32, 33, 48, 1000, 4097, 16384, 65535, (1 << 20) + 1, (1 << 30) - 1, 1 << 30, (1 << 31) - 1] + torch.randint(1, 1 << 31, (200,), generator=gen).tolist():
        m, s = _divisor(d)
        assert m < 1 << 32
        top = (1 << 31) - 1
        for n in {0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, top, top // d * d, max(top // d * d - 1, 0)} | set(torch.randint(0, top, (20,), generator=gen).tolist()):
            if n <= top:
                assert ((m * n >> 32) + n) >> s == n // d, (n, d)


@gpu
def test_captured_training():
    """Forward and backward in one graph: replayed on other numbers they give what the eager pass gives."""
    s = make(2, 33, 2, 3, 64, dtype=torch.bfloat16, device="cuda")
    leaves = [s[k].requires_grad_() for k in ("qkv", "wq", "wk")]

    def step():
        outs = ops.qkv_heads(*leaves, 1e-6, s["cos"], s["sin"])
        return (*outs, *torch.autograd.grad(outs, leaves, s["grads"]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(2):
        other = make(2, 33, 2, 3, 64, dtype=torch.bfloat16, device="cuda", seed=i + 1)
        with torch.no_grad():
            for leaf, k in zip(leaves, ("qkv", "wq", "wk")):
                leaf.copy_(other[k])
            for g, o in zip(s["grads"], other["grads"]):
                g.copy_(o)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_error_texts():
    assert "a position outside the tables" in gemm.error_text(0x41000)
    for code, text in ((0x42000, "a length outside the page table"), (0x43000, "a page number outside the pool"), (0x44021, "a bounded wait expired")):
        assert "4 bits a number: " + text in gemm.error_text(code)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", ["qkv", "wq"])
def test_forward_mode(which, grad, device):
    """Tangents come through (the eager form) or are refused: they are not dropped."""
    import torch.autograd.forward_ad as fw
    s = make(1, 5, 2, 2, 64, device=device)
    with torch.set_grad_enabled(grad), fw.dual_level():
        plain = ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])            # a level alone changes nothing
        assert all(fw.unpack_dual(t).tangent is None for t in plain)
        s[which] = fw.make_dual(s[which], torch.ones_like(s[which]))
        if device == "cuda":
            with pytest.raises(RuntimeError):
                ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])
        else:
            assert fw.unpack_dual(ops.qkv_heads(s["qkv"], s["wq"], s["wk"], 1e-6, s["cos"], s["sin"])[0]).tangent is not None


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("B,T", [(0, 3), (2, 0)])
def test_gradients_of_nothing(B, T, device):
    """No tokens: the weights' gradients are zeros."""
    s = make(B, T, 2, 2, 64, device=device, at=7)
    leaves = [s[k].requires_grad_() for k in ("qkv", "wq", "wk")]
    outs = ops.qkv_heads(*leaves, 1e-6, s["cos"], s["sin"], positions=s["at"])
    grads = torch.autograd.grad(outs, leaves, s["grads"])
    assert [g.shape for g in grads] == [t.shape for t in leaves] and not grads[1].any() and not grads[2].any()

@gpu
@pytest.mark.parametrize("D", [64, 6])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 0.0])
def test_outputs_that_nothing_uses_bring_no_nan(bad, D):
    """What nothing asks of has a gradient of zero, whatever lies there: NaN, infinities, and zeros without an epsilon, whose norm has no slope."""
    s = make(2, 17, 2, 2, D, dtype=torch.bfloat16, device="cuda")
    s["qkv"][0, 3, 1, 2] = bad                                # a key
    leaves = [s[k].requires_grad_() for k in ("qkv", "wq", "wk")]
    q, _, v = ops.qkv_heads(*leaves, 0.0, s["cos"], s["sin"])
    dx, dwq, dwk = torch.autograd.grad((q, v), leaves, (s["grads"][0], s["grads"][2]))
    assert dx.isfinite().all() and dwq.isfinite().all() and not dwk.any() and not dx[:, :, :, 2].any()
