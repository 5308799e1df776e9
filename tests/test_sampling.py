"""Sampling from given random numbers, against the definition in whole numbers of more bits.

The token is a function of the logits and the random number, whatever the order of sums, but where a border (p of the whole, min_p of the largest weight, the draw) lies within what a weight's rounding leaves open:
2^-45 of the largest weight a token, so V 2^-45 for a sum.  The oracle computes the weights in 64 bits (exp to 2^-52) and says how near the borders are; random draws are not that near one (probability V 2^-45 over the
weight of a token, 1e-7), and constructed ones lie half a token off.  The log-probability is rounded to 32 bits: 2^-24 of it, and V 2^-45 of the sum and 2^-45 of the largest weight, relative to the token's own."""
import math

import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.ops import sampling as S

gpu = pytest.mark.gpu
INF = float("inf")


def oracle(x, u, t=1.0, k=0, p=1.0, least=0.0):
    """(token, log-probability, number of kept tokens) of one row of finite and infinite numbers."""
    x = x.double()
    x = torch.where(x.isnan(), -INF, x)
    z, order = torch.sort(x, descending=True, stable=True)
    if float(z[0]) == -INF:
        return 0, -INF, 0
    w = torch.where(z == z[0], 1.0, ((z - z[0]) / (t if t > 0 else 1.0)).exp())
    if not t > 0:
        k = 1
    keep = w >= least
    if k > 0:
        keep[k:] = False
    if p < 1:
        upto = w.cumsum(0)
        keep[1:] &= upto[:-1] < p * upto[-1]
    keep[0] = True
    kept = torch.zeros_like(w)
    kept[order] = torch.where(keep, w, 0.0)
    upto = kept.cumsum(0)
    i = int((upto <= u * upto[-1]).sum())
    return i, math.log(float(kept[i] / upto[-1])), int((kept > 0).sum())


def check(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    token, logp = ops.sample_tokens(x, u, temperature, top_k, top_p, min_p)
    assert token.dtype == torch.int64 and logp.dtype == torch.float32 and token.shape == logp.shape == u.shape
    settings = [s.tolist() if torch.is_tensor(s) else torch.tensor(s, dtype=torch.float32).expand(x.shape[0]).tolist() for s in (u, temperature, top_k, top_p, min_p)]
    for b, (d, t, k, p, least) in enumerate(zip(*settings)):
        want, lp, _ = oracle(x[b], d, t, int(k), p, least)
        assert int(token[b]) == want, (b, int(token[b]), want)
        if lp == -INF:
            assert float(logp[b]) == -INF
        else:
            assert abs(float(logp[b]) - lp) <= 2.0 ** -23 * abs(lp) + 2.0 ** -44 * math.exp(min(-lp, 30)) + x.shape[1] * 2.0 ** -44
    return token, logp


def rows(B, V, dtype=torch.float32, seed=0, device="cpu", spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=gen) * spread
    x.scatter_add_(1, torch.randint(0, V, (B, 20), generator=gen), torch.empty(B, 20).exponential_(0.25, generator=gen))
    return x.to(dtype).to(device), torch.rand(B, generator=gen).to(device)


SETTINGS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=2), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.1, temperature=1.7), dict(min_p=0.05), dict(top_k=40, top_p=0.95, min_p=0.02, temperature=0.8),
            dict(top_p=0.999), dict(temperature=0.0), dict(top_k=10 ** 6, top_p=2.0), dict(temperature=30.0, top_p=0.7), dict(min_p=1.0), dict(top_p=0.0), dict(temperature=0.01, top_k=5),
            dict(temperature=1e6, top_p=0.5), dict(temperature=1e-6, top_p=0.5), dict(temperature=INF, top_k=30)]


@pytest.mark.parametrize("kw", SETTINGS)
def test_the_eager_form(kw):
    for V in (1, 2, 77, 1000):
        check(*rows(5, V), **kw)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", SETTINGS)
def test_settings(kw, dtype):
    for B, V in ((3, 1), (4, 2), (3, 33), (5, 1000), (2, 4099), (3, 32000)):
        check(*rows(B, V, dtype, device="cuda", seed=V), **kw)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(1, 50257), (3, 128256), (9, 65537), (2, 151936), (1, 300001), (1, 1 << 19), (40, 20000), (200, 3001)])
def test_sizes(B, V, dtype):
    for kw in (dict(), dict(top_k=300, temperature=0.7), dict(top_p=0.92), dict(top_k=1000, top_p=0.97, min_p=0.001)):
        check(*rows(B, V, dtype, device="cuda", seed=B), **kw)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_settings_of_each_request(dtype):
    gen = torch.Generator().manual_seed(5)
    B, V = 24, 5003
    x, u = rows(B, V, dtype, device="cuda")
    t, p, least = (torch.rand(B, generator=gen).cuda() for _ in range(3))
    k = torch.randint(-1, 400, (B,), generator=gen, dtype=torch.int32).cuda()
    t[3], p[4], p[5], least[6], k[7], k[8] = 0.0, 1.0, 0.0, 1.0, 0, 1
    check(x, u, t + (t > 0) * 0.3, k, p, least * 0.1)
    check(x, u, 0.9, k, 1.0, least * 0.1)
    check(x, u, t, 7, p)
    strided = torch.stack([t, p], 1).cuda()
    check(x, u, strided[:, 0], k.repeat_interleave(2)[::2], strided[:, 1])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits(dtype):
    """Cuts inside of equal logits, by number and by weight, in every part of a row; draws half a token off the borders."""
    for V in (7, 600, 40000, 140001):
        x = torch.full((6, V), 1.5, dtype=dtype, device="cuda")
        n = torch.tensor([1, 2, V // 3 + 1, V // 2 + 1, V - 1, V], device="cuda")
        for first in (0, 1, 5):
            x[:, :first], x[:, first * 2 + 1:first * 2 + 2] = -3.0, 2.5
            for place in (0.0, 0.3, 0.77, 1.0):
                k = n.int()
                m = torch.tensor([oracle(x[b], 0.0, 1.0, int(k[b]))[2] for b in range(6)], dtype=torch.float64)
                u = ((place * (m - 1)).floor() + 0.5) / m
                check(x, u.float().cuda(), top_k=k)
            # weights: half a token above the n-th
            p = ((n.double() - 0.5) / V).float()
            check(x, torch.full((6,), 0.61, device="cuda"), top_p=p)
            check(x, torch.full((6,), 0.99, device="cuda"), top_p=p, top_k=(n // 2 + 1).int())


@gpu
def test_near_numbers():
    """Neighbouring 32-bit numbers, zeros of both signs, ends of the type: the cut falls between the right two."""
    near = (torch.arange(3000) * 7 % 3000).int() + torch.tensor(8.0).view(torch.int32)
    x = near.view(torch.float32)[None].repeat(4, 1).cuda()
    check(x, torch.tensor([0.0, 0.4, 0.9, 0.9999], device="cuda"), top_k=torch.tensor([1, 7, 1500, 2999], dtype=torch.int32, device="cuda"))
    check(x, torch.tensor([0.0, 0.4, 0.9, 0.9999], device="cuda"), 1e-4, top_k=torch.tensor([1, 7, 1500, 2999], dtype=torch.int32, device="cuda"))
    check(x, torch.tensor([0.0, 0.4, 0.9, 0.9999], device="cuda"), 1e-3, top_p=torch.tensor([0.1, 0.5, 0.77, 0.993], device="cuda"))
    z = torch.tensor([[0.0, -0.0, 0.0, -0.0, 1e-45, -1e-45, 0.0]]).repeat(7, 1).cuda()
    u = torch.full((7,), 0.999, device="cuda")
    token, _ = ops.sample_tokens(z, u, 1.0, torch.arange(1, 8, dtype=torch.int32, device="cuda"))
    assert token.tolist() == [4, 4, 4, 4, 4, 6, 6]                # 4 first, then 0, 1, 2, 3, 6, and 5 last
    assert ops.sample_tokens(z, u, 1.0, torch.arange(1, 8, dtype=torch.int32, device="cuda"))[0].tolist() == S._eager(z, u, 1.0, torch.arange(1, 8, dtype=torch.int32, device="cuda"), 1.0, 0.0)[0].tolist()
    big = torch.tensor([[3.0e38, -3.0e38, 3.0e38, 1.0], [-3e38, -3.1e38, -3e38, -INF], [1e30, 1.0001e30, 0.0, 1e30]], device="cuda")
    for kw in (dict(), dict(top_k=2), dict(top_p=0.4), dict(top_k=3, top_p=0.9), dict(temperature=1e37, top_k=3), dict(temperature=1e26, top_p=0.7)):
        for d in (0.0, 0.3, 0.8):
            check(big, torch.full((3,), d, device="cuda"), **kw)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_nan_and_infinities(device):
    nan = float("nan")
    x = torch.tensor([[1.0, nan, 2.0, -INF], [INF, 1.0, INF, nan], [-INF] * 4, [nan] * 4, [nan, -INF, 3.0, nan], [-INF, -5.0, -INF, -5.0]], device=device)
    for kw in (dict(), dict(top_k=1), dict(top_k=3), dict(top_p=0.6), dict(temperature=0.0), dict(temperature=INF), dict(min_p=0.5), dict(top_k=2, top_p=0.9, temperature=0.1)):
        for u in (0.0, 0.45, 0.9):
            check(x, torch.full((6,), u, device=device), **kw)
    y = x.repeat(1, 2000)
    for kw in (dict(), dict(top_k=3), dict(top_p=0.6)):
        token, logp = ops.sample_tokens(y, torch.full((6,), 0.3, device=device), **kw)
        assert token[2:4].tolist() == [0, 0] and logp[2:4].tolist() == [-INF, -INF] and y[1, token[1]] == INF and y[4, token[4]] == 3 and y[5, token[5]] == -5


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_draws_at_the_ends(device):
    x = torch.tensor([[-4.0, 1.0, 0.5, -INF, -2.0]], device=device).repeat(6, 1)
    u = torch.tensor([0.0, -1.0, 1.0, 2.0, float("nan"), 1 - 2.0 ** -24], device=device)
    assert ops.sample_tokens(x, u)[0].tolist() == [0, 0, 4, 4, 0, 4]
    assert ops.sample_tokens(x, u, top_k=2)[0].tolist() == [1, 1, 2, 2, 1, 2]


@gpu
def test_the_shares_of_the_draws():
    """Draws spread evenly over [0, 1) fall to the tokens by their weights, to one draw."""
    V, N = 50, 4096
    x = torch.randn(V, generator=torch.Generator().manual_seed(0)).cuda()
    token, _ = ops.sample_tokens(x.expand(N, V), (torch.arange(N, device="cuda") + 0.5) / N, 0.9)
    assert ((torch.bincount(token, minlength=V) - N * torch.softmax(x.double() / 0.9, 0)).abs() <= 1).all()


@gpu
def test_strides_streams_and_graphs():
    x, u = rows(5, 4001, device="cuda")
    kw = dict(temperature=0.8, top_k=100, top_p=0.9, min_p=0.01)
    want = check(x, u, **kw)
    wide = torch.full((5, 4100), float("nan"), device="cuda")
    for view in (wide[:, 3:4004], wide[:, 8:4009], torch.empty(4001, 5, device="cuda").t(), torch.empty(10, 4001, device="cuda")[::2]):
        view.copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(ops.sample_tokens(view, u, **kw), want))
    assert all(torch.equal(a, b) for a, b in zip(ops.sample_tokens(x[:1].expand(5, -1), u, **kw), ops.sample_tokens(x[:1].repeat(5, 1), u, **kw)))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.sample_tokens(x, u, **kw)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_tokens(x, u, **kw)
    for i in range(3):
        u.copy_(rows(5, 4001, seed=i + 1)[1])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, ops.sample_tokens(x, u, **kw)))


def test_refusals():
    x, u = rows(3, 10)
    for args, kw in (((x[0], u), {}), ((x.double(), u), {}), ((x[:, :0], u), {}), ((x, u[:2]), {}), ((x, u.double()), {}), ((x, u), dict(temperature=-1.0)), ((x, u), dict(temperature=float("nan"))),
                     ((x, u), dict(top_k=-1)), ((x, u), dict(top_k=1.5)), ((x, u), dict(top_p=-0.1)), ((x, u), dict(min_p=1.1)), ((x, u), dict(min_p=-0.1)), ((x, u), dict(temperature=u.double())),
                     ((x, u), dict(top_k=torch.ones(3))), ((x, u), dict(top_k=torch.ones(3, dtype=torch.int64))), ((x, u), dict(top_p=u[:2])), ((x, u), dict(min_p=u[:, None]))):
        with pytest.raises(ValueError):
            ops.sample_tokens(*args, **kw)
    assert ops.sample_tokens(x[:0], u[:0])[0].shape == (0,)


@pytest.mark.parametrize("V", [1, 77, 4096, 65536, 65537, 128256, 1 << 19])
def test_shares(V):
    parts, length = S._shares(V)
    assert parts in (1, 2, 4, 8) and parts * length >= V and length <= S.PART and length % 128 == 0


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_settings_outside_their_ranges(device):
    """Tensors are not looked at on the host: NaN cuts nothing off (a temperature of NaN takes the largest), numbers beyond the ends are the ends."""
    x, u = rows(6, 300, device=device)
    nan = float("nan")
    one = lambda v, dtype=torch.float32: torch.full((6,), v, dtype=dtype, device=device)            # noqa: E731
    plain, best = ops.sample_tokens(x, u), ops.sample_tokens(x, u, 0.0)
    for kw, want in ((dict(top_p=one(nan)), plain), (dict(min_p=one(nan)), plain), (dict(min_p=one(-1.0)), plain), (dict(top_p=one(7.0)), plain), (dict(top_k=one(-3, torch.int32)), plain),
                     (dict(top_k=one((1 << 31) - 1, torch.int32)), plain), (dict(temperature=one(nan)), best), (dict(temperature=one(-1.0)), best), (dict(top_p=one(-0.5)), best), (dict(min_p=one(3.0)), best)):
        got = ops.sample_tokens(x, u, **kw)
        assert torch.equal(got[0], want[0]) and torch.allclose(got[1], want[1], atol=1e-6), kw


@gpu
def test_many_rows_again_and_again():
    """The CTAs of a row go through the levels of a search at their own pace; the answer is the same every time."""
    for dtype, kw in ((torch.float32, dict(top_p=0.95)), (torch.float32, dict(top_k=500, temperature=1.4)), (torch.bfloat16, dict(top_p=0.7, top_k=3000, temperature=2.0))):
        x, u = rows(160, 40000, dtype, device="cuda", seed=3)
        want = ops.sample_tokens(x, u, **kw)
        got = [ops.sample_tokens(x, u, **kw) for _ in range(150)]
        assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
        eager = S._eager(x, u, kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0), 0.0)
        assert torch.equal(want[0], eager[0])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_nothing_is_cut_off_of_long_flat_rows(device):
    """The whole of 300001 equal weights is above 2^62 units of 2^-44."""
    x = torch.zeros(4, 300001, device=device)
    u = torch.tensor([0.1, 0.87, 0.95, 0.999], device=device)
    for kw in (dict(), dict(min_p=0.5), dict(top_k=290000), dict(top_p=torch.full((4,), 1.0, device=device))):
        check(x, u, **kw)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("V", [(1 << 19) - 1, 1 << 19, (1 << 19) + 1, 1 << 20, 1100000, 1 << 21])
def test_sums_of_long_rows(V, device):
    """Equal weights, whose sum is 2^63 units at 2^19 and 2^20 logits, and weights that a high temperature makes nearly so; draws half a token off the borders (of equal weights)."""
    flat = torch.zeros(5, V, device=device)
    u = ((torch.tensor([0.0, 0.3, 0.5, 0.9, 1.0], dtype=torch.float64) * (V - 1)).floor() + 0.5) / V
    u = u.float().clamp_max(1 - 2.0 ** -24).to(device)
    u[1] = 0.300048828125                                # a draw of few bits: the product is exact
    for kw in (dict(), dict(top_p=0.9), dict(top_k=V // 3), dict(top_k=V - 1, top_p=0.999), dict(min_p=0.5)):
        check(flat, u, **kw)
    x, u = rows(2, V, device=device, seed=V % 1000)
    for kw in (dict(temperature=30.0), dict(temperature=5.0), dict(temperature=30.0, top_p=0.8, top_k=V // 2), dict(temperature=INF)):
        check(x, u, **kw)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_draws_far_outside(device):
    """A draw times the sum may leave 63 bits: from one on it is the last kept token."""
    x = torch.tensor([[-4.0, 1.0, 0.5, -INF, -2.0]], device=device).repeat(5, 1)
    u = torch.tensor([1e6, 3e38, INF, -3e38, -INF], device=device)
    assert ops.sample_tokens(x, u)[0].tolist() == [4, 4, 4, 0, 0]
    assert ops.sample_tokens(x, u, top_k=2)[0].tolist() == [2, 2, 2, 1, 1]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_plus_infinity_and_an_endless_temperature(device):
    """Tokens at plus infinity share the whole weight whatever the temperature, and what top_p leaves of them is counted by weight."""
    u = torch.tensor([0.1, 0.3, 0.6, 0.9], device=device)
    for other in (2.0, -INF):
        x = torch.tensor([[1.0, INF, other, INF, -INF, INF, INF, float("nan")]], device=device).repeat(4, 1)
        for t in (INF, 1e30, 1.0, 0.001):
            for top_p, want in ((1.0, [1, 3, 5, 6]), (0.9, [1, 3, 5, 6]), (0.7, [1, 1, 3, 5]), (0.4, [1, 1, 3, 3])):
                token, logp = ops.sample_tokens(x, u, t, 0, top_p)
                assert token.tolist() == want and torch.allclose(logp.exp(), torch.full((4,), 1 / len(set(want)), device=device)), (other, t, top_p)


@gpu
def test_rows_of_different_lengths_from_two_threads():
    """What a launch may have of shared memory belongs to the kernel, not to the call: a call of short rows must not take it from one of long rows in another thread."""
    import threading
    errors = []

    def work(V):
        try:
            x, u = rows(1, V, device="cuda", seed=V)
            with torch.cuda.stream(torch.cuda.Stream()):
                torch.cuda.synchronize()
                want = ops.sample_tokens(x, u, top_p=0.9)
                for _ in range(40):
                    got = [ops.sample_tokens(x, u, top_p=0.9) for _ in range(50)]
                    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
        except BaseException as e:      # noqa: B036
            errors.append(e)
    threads = [threading.Thread(target=work, args=(V,)) for V in (300001, 1000, 131072, 2000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
