"""A paged cache of 4 bits a number: what it holds, bit for bit, and one-token attention over it against the formula in 64 bits.

Bounds.  What is stored is defined step by step in 32 bits, so pools are equal byte for byte; a number comes back within half a size, and the size is at most (range + 2^-7 |low|) / 15 (1 + 2^-7): ``low`` and ``size``
are each rounded away from the group by one bf16 step, 2^-7 of them at most.
Attention: u = finfo(type).eps / 2, one rounding of the output.  On the tensor cores codes go in as they are and queries exactly (but for 2^-36 of the head's largest number), so a score's sum of products, which the
tensor cores round to 2^-23 of its largest part per step of 16, is off by D / 16 2^-23 of scale sum |q| (15 size + |low|), and as much again for the sum over the groups; tanh by 1e-6 of the score.  A weight times a
value's size is rounded to 2^-12 of it for bf16 outputs and to 2^-22 for fp16 ones, of 15 sizes at most; it goes in as fp16 numbers, whose smallest is 2^-32 of the largest size that a warp has met (rounded up to a
power of two, and weights may be counted from a maximum 2^8 below the largest score: half of 2^-31 times 15 a key).  In 32 bits throughout: N + 8 roundings of scale sum |q| |k|, and a chain of additions as long as a
warp's keys.  A weight is off by twice what its score is, and 2^-20 for the exponentials.  fp16 numbers below 2^-14
are rounded by up to 2^-25."""
import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.ops import gemm
from linear_moe_b200.ref import int4_cache as R

gpu = pytest.mark.gpu
BF, HALF, F = torch.bfloat16, torch.float16, torch.float32


def tables(lens, page, gen, spare=3):
    need = [-(-max(x, 0) // page) for x in lens]
    P, width = sum(need) + spare, max(need + [1]) + 1
    order = torch.randperm(P, generator=gen).tolist()
    table = torch.randint(-9, P + 9, (len(lens), width), generator=gen, dtype=torch.int32)       # entries behind the length: anything
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table, P


def make(lens, H, G, D, page=64, dtype=BF, device="cuda", size=1.5, seed=0, stale=True, values=None):
    """Pools of random rows; what lies behind a request's last row, and on the pages of nobody, is NaN or infinite where it is not a code."""
    gen = torch.Generator().manual_seed(seed)
    table, P = tables(lens, page, gen)
    pools = []
    for _ in range(2):
        pool = ops.int4_pages(P, G, D, page)
        if stale:
            pool.fill_(255)                                  # scales of NaN
        pools.append(pool)
    lengths = torch.tensor(lens, dtype=torch.int32)
    most = max(max(lens), 1)
    rows = [torch.zeros(len(lens), most, G, D) for _ in range(2)]
    for b, n in enumerate(lens):
        for r in rows:
            r[b, most - n:] = torch.randn(n, G, D, generator=gen) if values is None else values(gen, n, G, D)
    ops.store_rows_int4(rows[0].to(dtype), rows[1].to(dtype), *pools, table, lengths)
    s = dict(q=(torch.randn(len(lens), H, D, generator=gen) * size).to(dtype), k=pools[0], v=pools[1], table=table, lengths=lengths)
    return {k: t.to(device) for k, t in s.items()}


def formula(s, window=None, cap=None, slopes=None, scale=None, tensor=True):
    """The output in 64 bits, and its room but for the output's own rounding."""
    q = s["q"].double()
    B, H, D = q.shape
    G, page = s["k"].shape[1], 8 * s["k"].shape[2] // (5 * D)
    scale = D ** -0.5 if scale is None else scale
    out, room = torch.zeros_like(q), torch.zeros_like(q)
    for b, n in enumerate(s["lengths"].tolist()):
        keys = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        if len(keys) == 0:
            continue
        at = s["table"][b].long()[keys // page]
        k, v = (R.read(s[x], at, keys % page, D).double().repeat_interleave(H // G, 1) for x in "kv")
        x = torch.einsum("hd,jhd->hj", q[b], k) * scale
        if tensor:
            codes, scales = R._parts(s["k"], D)
            sc = scales[at, :, keys % page].contiguous().view(BF).double().unflatten(-1, (2, -1)).abs()
            reach = (15 * sc[:, :, 1] + sc[:, :, 0]).repeat_interleave(32, -1).repeat_interleave(H // G, 1)
            off = 2 * (D / 16) * 2 ** -23 * scale * torch.einsum("hd,jhd->hj", q[b].abs(), reach)
        else:
            off = (D / 32 + 8) * 2 ** -24 * scale * torch.einsum("hd,jhd->hj", q[b].abs(), k.abs()) + 4 * 2 ** -24 * x.abs()
        if cap:
            x = cap * torch.tanh(x / cap)
            off = off + 1e-6 * x.abs()
        if slopes is not None:
            far = slopes.double()[:, None] * (n - 1 - keys).double()
            x, off = x - far, off + 4 * 2 ** -24 * (far + x.abs())
        p = torch.softmax(x, -1)
        # a weight far below the largest one may be off by more than its share: its score's error counts by the weight
        rel = (p * off).sum(-1, keepdim=True) + off + 2 ** -20 + (2.0 ** (-13 if s["q"].dtype == BF else -22) if tensor else (n / 8 + 64) * 2 ** -24)      # doubled below
        out[b] = torch.einsum("hj,jhd->hd", p, v)
        if tensor:                                           # lows and codes are added up by themselves
            sv = R._parts(s["v"], D)[1][at, :, keys % page].contiguous().view(BF).double().unflatten(-1, (2, -1)).abs()
            v = (sv[:, :, 0] + 15 * sv[:, :, 1]).repeat_interleave(32, -1).repeat_interleave(H // G, 1)
        room[b] = 2 * torch.einsum("hj,jhd->hd", p * rel, v.abs())
        if tensor:
            room[b] += len(keys) * 15 * 2.0 ** -32 * sv[:, :, 1].max()
    return out, room


def attend(s, window=None, cap=None, slopes=None, scale=None):
    return ops.paged_attention_int4(s["q"], s["k"], s["v"], s["table"], s["lengths"], scale, window, softcap=cap, slopes=slopes)


def on_tensor_cores(s):
    return s["q"].is_cuda and s["q"].dtype != F and s["q"].shape[2] <= 128


def check(s, **kw):
    got = attend(s, **kw)
    want, room = formula(s, tensor=on_tensor_cores(s), **kw)
    u = torch.finfo(got.dtype).eps / 2
    bad = (got.double() - want).abs() - (u * (want.abs() + room) + room + (2.0 ** -25 if got.dtype == HALF else 0.0))
    assert got.isfinite().all() and bad.max() <= 0, float(bad.max())
    gemm.check_error()
    return got


# ---- rows -------------------------------------------------------------------------------------------------------------------------
def groups():
    """Groups where the codes can go wrong: equal numbers, zeros of both signs, ties, one number far out, subnormal ranges, the ends of the types, NaN and infinities."""
    gen = torch.Generator().manual_seed(1)
    g = [torch.zeros(32), -torch.zeros(32), torch.full((32,), 1.7), torch.full((32,), -3e-39), torch.arange(32.0) / 2, torch.arange(32.0).neg() * 1e-40, torch.randn(32, generator=gen) * 1e30,
         torch.randn(32, generator=gen) * 1e-38, torch.cat([torch.randn(31, generator=gen), torch.tensor([1e6])]), torch.tensor([-65504.0, 65504.0] * 16), torch.randn(32, generator=gen) + 1000,
         torch.tensor([3.38e38] * 31 + [3.3e38]), torch.tensor([3.38e38, -3.38e38] * 16), torch.full((32,), -3.4028e38), torch.full((32,), float("nan")), torch.full((32,), float("inf"))]
    for bad in ("nan", "inf", "-inf"):
        x = torch.randn(32, generator=gen)
        x[17] = float(bad)
        g.append(x)
    g += [torch.randn(32, generator=gen) * 10.0 ** i for i in range(-6, 7)]
    for i in range(20):                                     # quotients at and next to the borders between two codes
        size = 2.0 ** (i - 10)
        x = torch.randint(0, 30, (32,), generator=gen).float() / 2 * size
        x[3], x[20] = 0.0, 14.96875 * size              # a size that is a power of two
        x[i] = x[i].nextafter(torch.tensor(100.0 if i % 2 else -100.0)) if float(x[i]) > 0 else x[i]
        g.append(x - (i % 3) * 4 * size)
    return torch.stack(g)


def test_what_comes_back():
    """Within half a size of what went in, sizes as small as the definition says."""
    x = groups()
    code, low, size = R.encode(x)
    low, size = low.double(), size.double()
    good = low[:, 0].isfinite()
    assert good.tolist() == [bool(g.isfinite().all()) and float(g.min()) > -3.39e38 and float(g.max().double() - g.min().double()) < 3.4e38 for g in x]
    y = (low[..., None] + size[..., None] * code.double()).flatten(1)
    x = x.double()
    off, span = (y - x).abs().amax(1), x.amax(1) - x.amin(1)
    limit = (span + x.amin(1).abs() * 2 ** -7) / 15 * (1 + 2 ** -7) + 2e-40
    assert (off[good] <= size[good, 0] / 2 * (1 + 2 ** -14) + 1e-45).all() and (size[good, 0] <= limit[good]).all()
    assert y[~good].isnan().all()


def same(x, y):
    return torch.equal(x.nan_to_num(nan=12345.0), y.nan_to_num(nan=12345.0))


CASES = [([1], 1, 32, 16), ([5, 0, 130], 2, 64, 64), ([64, 63, 65], 3, 96, 64), ([200, 17, 33], 4, 128, 16), ([40, 3], 2, 160, 32), ([70], 1, 256, 48), ([100, 90], 2, 224, 64)]


@pytest.mark.parametrize("lens,G,D,page", CASES)
def test_rows_of_the_eager_form(lens, G, D, page):
    rows_in_and_out(lens, G, D, page, F, "cpu")


@gpu
@pytest.mark.parametrize("dtype", [F, BF, HALF])
@pytest.mark.parametrize("lens,G,D,page", CASES)
def test_rows(lens, G, D, page, dtype):
    rows_in_and_out(lens, G, D, page, dtype, "cuda")


def rows_in_and_out(lens, G, D, page, dtype, device):
    gen = torch.Generator().manual_seed(3)
    table, P = tables(lens, page, gen)
    pools = [torch.randint(0, 256, (P, G, page * 5 * D // 8), generator=gen, dtype=torch.uint8) for _ in range(2)]
    first = [p.clone() for p in pools]
    here, where = [p.to(device) for p in pools], table.to(device)
    T, B = max(max(lens) // 2, 1), len(lens)
    g = groups().to(dtype).flatten()
    new = [g[torch.randint(0, g.numel() // 32, (B * T * G * D // 32, 1), generator=gen) * 32 + torch.arange(32)].view(B, T, G, D) for _ in range(2)]
    lengths = torch.tensor(lens, dtype=torch.int32)
    ops.store_rows_int4(new[0].to(device), new[1].to(device), *here, where, lengths.to(device))
    R.store_rows(*new, *pools, table, lengths)
    written = torch.zeros(P, G, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        keys = torch.arange(max(0, n - T), n)
        written[table[b].long()[keys // page], :, keys % page] = True
    for x, y, z in zip(here, pools, first):
        # NaN scales have one form; every byte that no row was stored in is as it was
        assert torch.equal(x.cpu(), y)
        for part, old in zip(R._parts(y, D), R._parts(z, D)):
            assert torch.equal(part.flatten(3)[~written], old.flatten(3)[~written])
    n = max(max(lens), 1) + 3
    got = ops.read_rows_int4(*here, where, lengths.to(device), n, D, dtype)
    want = R.read_rows(*pools, table, lengths, n, D, dtype)
    for x, y in zip(got, want):
        assert x.shape == (B, n, G, D) and x.dtype == dtype and same(x.cpu(), y)
        for b, length in enumerate(lens):
            assert (x[b, length:] == 0).all()
    # half of them
    for x, y in zip(ops.read_rows_int4(*here, where, lengths.to(device), n // 2, D, F), R.read_rows(*pools, table, lengths, n // 2, D, F)):
        assert same(x.cpu(), y)


@gpu
def test_rows_of_any_strides():
    lens, G, D = [40, 9], 2, 96
    gen = torch.Generator().manual_seed(4)
    table, P = tables(lens, 64, gen)
    x = torch.randn(2, 40, G, D, generator=gen).to(BF)
    lengths = torch.tensor(lens, dtype=torch.int32)
    want = [ops.int4_pages(P, G, D) for _ in range(2)]
    R.store_rows(x, x.neg(), *want, table, lengths)
    wide = torch.full((2, 40, G * D + 40), float("nan"), dtype=BF, device="cuda")
    for view in (wide[..., 8:8 + G * D].unflatten(-1, (G, D)), wide[..., 5:5 + G * D].unflatten(-1, (G, D)), torch.empty(2, G, 40, D, dtype=BF, device="cuda").transpose(1, 2),
                 torch.empty(2, 40, D, G, dtype=BF, device="cuda").transpose(2, 3), torch.empty(40, 2, G, D, dtype=BF, device="cuda").transpose(0, 1)):
        view.copy_(x)
        pools = [ops.int4_pages(P, G, D, device="cuda") for _ in range(2)]
        table2 = torch.full((2, 2 * table.shape[1]), -7, dtype=torch.int32, device="cuda")[:, ::2]
        table2.copy_(table)
        lengths2 = torch.zeros(2, 3, dtype=torch.int32, device="cuda")[:, 1]
        lengths2.copy_(lengths)
        ops.store_rows_int4(view, view.neg() if view.is_contiguous() else torch.empty_strided(view.shape, view.stride(), dtype=BF, device="cuda").copy_(-x.cuda()), *pools, table2, lengths2)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(pools, want))
        assert all(torch.equal(a.cpu(), b) for a, b in zip(ops.read_rows_int4(*pools, table2, lengths2, 41, D, BF), R.read_rows(*want, table, lengths, 41, D, BF)))


# ---- attention --------------------------------------------------------------------------------------------------------------------
def test_the_eager_form():
    s = make([1, 0, 77, 64], 4, 2, 64, dtype=F, device="cpu")
    check(s)
    check(s, window=5, cap=3.0, slopes=ops.alibi_slopes(4), scale=0.3)


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, F])
@pytest.mark.parametrize("H,G,D", [(1, 1, 32), (4, 2, 64), (16, 2, 64), (9, 3, 96), (32, 8, 128), (24, 2, 128), (40, 2, 128), (5, 1, 128), (6, 2, 160), (4, 4, 256)])
def test_heads(H, G, D, dtype):
    check(make([1, 15, 16, 17, 64, 65, 300, 0], H, G, D, dtype=dtype))


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_pages(D, page, dtype):
    check(make([1, 47, 48, 49, 700], 8, 2, D, page=page, dtype=dtype))


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, F])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=16), dict(window=33), dict(window=1000), dict(cap=2.0), dict(cap=50.0), dict(slopes=True), dict(scale=0.02), dict(scale=1.0, cap=20.0, slopes=True, window=70)])
def test_scores(kw, dtype):
    s = make([1, 16, 77, 300, 513], 8, 2, 64, dtype=dtype, size=3.0)
    check(s, **{**kw, **({"slopes": ops.alibi_slopes(8).cuda()} if kw.get("slopes") else {})})
    s = make([1, 16, 77, 300, 513], 12, 1, 128, dtype=dtype, size=3.0)
    check(s, **{**kw, **({"slopes": ops.alibi_slopes(12).cuda()} if kw.get("slopes") else {})})


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("lens,H,G,D", [([5000], 16, 4, 128), ([20000, 3], 8, 1, 64), ([3000, 2900, 17, 0], 8, 2, 96), ([40000], 4, 1, 128), ([2048, 2000], 64, 8, 128)])
def test_shared_out_keys(lens, H, G, D, dtype):
    """Requests that several CTAs, a cluster's or more, share."""
    s = make(lens, H, G, D, dtype=dtype)
    check(s)
    check(s, window=1500, cap=30.0)


@gpu
@pytest.mark.parametrize("B", [70, 150])
def test_many_requests(B):
    gen = torch.Generator().manual_seed(B)
    check(make(torch.randint(0, 400, (B,), generator=gen).tolist(), 16, 8, 64))


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, F])
def test_sizes_of_the_numbers(dtype):
    """Values whose groups differ by many powers of two, keys with a mean far from zero, tiny and large ones."""
    def values(gen, n, G, D):
        return torch.randn(n, G, D, generator=gen) * 10.0 ** torch.randint(-4, 3, (n, G, 1), generator=gen)
    check(make([300, 20], 8, 2, 64, dtype=dtype, values=values, size=0.2))
    check(make([300, 20], 8, 2, 128, dtype=dtype, values=lambda gen, n, G, D: torch.randn(n, G, D, generator=gen) + 9, size=0.5))
    check(make([300, 20], 8, 2, 128, dtype=dtype, values=lambda gen, n, G, D: torch.randn(n, G, D, generator=gen) * 1e-6, size=2.0))


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, F])
@pytest.mark.parametrize("where", ["q", "k", "v"])
def test_nan(where, dtype):
    """NaN in a visible key's group gives NaN to the heads that see it, in a value's group to the numbers of that group, in a query to its head; hidden ones nothing."""
    def values(gen, n, G, D):
        return torch.randn(n, G, D, generator=gen)
    s = make([100, 40], 8, 2, 64, dtype=dtype, values=values)
    want = attend(s)
    if where == "q":
        s["q"][0, 3, 5] = float("nan")
        got = attend(s)
        assert got[0, 3].isnan().all()
        got[0, 3] = want[0, 3]
    else:
        pool = s[where]
        _, scales = R._parts(pool, 64)
        at = s["table"][0, 1].long()
        scales[at, 1, 30].view(BF)[1] = float("nan")            # key 94, head 1: the second group's low
        got = attend(s)
        if where == "k":
            assert got[0, 4:].isnan().all()
        else:
            assert got[0, 4:, 32:].isnan().all() and got[0, 4:, :32].isfinite().all()
        hidden = attend(s, window=5)
        assert hidden.isfinite().all()
        got[0, 4:] = want[0, 4:]
    assert torch.equal(got, want)


@gpu
def test_bad_tables_and_lengths():
    """Reported, and nothing out of range is touched: the kernels check every page and length."""
    for dtype, D in ((BF, 64), (F, 64), (BF, 160)):
        s = make([100, 40], 4, 2, D, dtype=dtype)
        gemm.check_error()
        want = check(s)
        for bad in (-1, s["k"].shape[0], 1 << 30):
            t = dict(s, table=s["table"].clone())
            t["table"][0, 1] = bad
            got = attend(t)
            with pytest.raises(RuntimeError, match="4 bits a number: a page number outside the pool"):
                gemm.check_error()
            assert torch.equal(got[1], want[1])
            short = dict(s, lengths=torch.tensor([64, 40], dtype=torch.int32, device="cuda"))
            assert torch.allclose(got[0].float(), attend(short)[0].float(), atol=0.05)          # the page's keys are hidden
            rows = ops.read_rows_int4(t["k"], t["v"], t["table"], t["lengths"], 100, D, dtype)
            with pytest.raises(RuntimeError, match="a page number outside the pool"):
                gemm.check_error()
            assert (rows[0][0, 64:] == 0).all()
            pools = [t["k"].clone(), t["v"].clone()]
            ops.store_rows_int4(torch.ones(2, 1, 2, D, dtype=dtype, device="cuda"), torch.ones(2, 1, 2, D, dtype=dtype, device="cuda"), *pools, t["table"], t["lengths"])
            with pytest.raises(RuntimeError, match="a page number outside the pool"):
                gemm.check_error()
        for bad in (-3, s["table"].shape[1] * 64 + 1):
            t = dict(s, lengths=torch.tensor([bad, 40], dtype=torch.int32, device="cuda"))
            if bad > 0:
                t["table"] = s["table"].clamp(0, s["k"].shape[0] - 1)
            got = attend(t)
            with pytest.raises(RuntimeError, match="4 bits a number: a length outside the page table"):
                gemm.check_error()
            assert torch.equal(got[1], want[1])
            pools = [t["k"].clone(), t["v"].clone()]
            ops.store_rows_int4(torch.ones(2, 1, 2, D, dtype=dtype, device="cuda"), torch.ones(2, 1, 2, D, dtype=dtype, device="cuda"), *pools, t["table"], t["lengths"])
            with pytest.raises(RuntimeError, match="a length outside the page table"):
                gemm.check_error()
        gemm.check_error()


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, F])
def test_strides_streams_and_graphs(dtype):
    s = make([300, 77, 2050], 8, 2, 128, dtype=dtype)
    want = attend(s)
    wide = torch.full((3, 8, 136), float("nan"), dtype=dtype, device="cuda")
    for view in (wide[..., 8:], wide[..., 3:131], torch.empty(8, 3, 128, dtype=dtype, device="cuda").transpose(0, 1), torch.empty(3, 128, 8, dtype=dtype, device="cuda").transpose(1, 2)):
        view.copy_(s["q"])
        assert torch.equal(attend(dict(s, q=view)), want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        assert torch.equal(attend(s), want)
    st.synchronize()
    # a captured step: the new token's row is stored, attention sees it, the lengths grow on the device
    s = make([300, 77, 2030], 8, 2, 128, dtype=dtype)
    new = [torch.randn(3, 1, 2, 128, device="cuda").to(dtype) for _ in range(2)]

    def step(t):
        ops.store_rows_int4(*new, t["k"], t["v"], t["table"], t["lengths"])
        return attend(t)
    other = {k: t.clone() for k, t in s.items()}
    step({k: t.clone() for k, t in s.items()})
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(s)
    with torch.cuda.graph(graph2):
        out2 = step(s)
    for i in range(4):
        for t in (s, other):
            t["lengths"] += 1
        for x in new:
            x.copy_(x * 1.1)
        (graph if i % 2 else graph2).replay()
        want = step(other)
        assert torch.equal(out if i % 2 else out2, want) and torch.equal(s["k"], other["k"]) and torch.equal(s["v"], other["v"])
    gemm.check_error()


def test_refusals():
    s = make([20, 9], 4, 2, 64, dtype=F, device="cpu")
    new = torch.zeros(2, 1, 2, 64)
    at = (s["k"], s["v"], s["table"], s["lengths"])

    def swap(i, t):
        return [t if j == i else x for j, x in enumerate(at)]
    bad_pools = [swap(0, s["k"].to(torch.int8)), swap(0, s["k"][:, :, :-20]), swap(1, s["v"][:2]), swap(0, s["k"][:, :1]), swap(0, s["k"].transpose(0, 1)), swap(2, s["table"].long()), swap(2, s["table"][:1]),
                 swap(3, s["lengths"].long()), swap(3, s["lengths"][:1]), swap(3, torch.tensor([20, -1], dtype=torch.int32)), swap(3, torch.tensor([20, 900], dtype=torch.int32)),
                 swap(2, torch.full_like(s["table"], 99))]
    for bad in bad_pools:
        with pytest.raises(ValueError):
            ops.store_rows_int4(new, new, *bad)
        with pytest.raises(ValueError):
            ops.read_rows_int4(*bad, 20, 64, F)
        with pytest.raises(ValueError):
            ops.paged_attention_int4(s["q"], *bad)
    for args in ((new[0], new[0]), (new, new[:, :, :1]), (new, new.half()), (new.double(), new.double()), (new[:, :, :1], new[:, :, :1]), (new[..., :48], new[..., :48])):
        with pytest.raises(ValueError):
            ops.store_rows_int4(*args, *at)
    for args in ((20, 96, F), (20, 64, torch.float64), (-1, 64, F), (20, 40, F)):
        with pytest.raises(ValueError):
            ops.read_rows_int4(*at, *args)
    for q, kw in ((s["q"][0], {}), (s["q"][:, :3], {}), (s["q"].double(), {}), (s["q"], dict(window=0)), (s["q"], dict(softcap=-1.0)), (s["q"], dict(scale=-1.0)), (s["q"], dict(slopes=torch.ones(3))),
                  (s["q"].clone().requires_grad_(), {})):
        with pytest.raises(ValueError):
            ops.paged_attention_int4(q, *at, **kw)
    for args in ((3, 2, 33), (3, 2, 288), (3, 2, 64, 24), (3, 2, 0)):
        with pytest.raises(ValueError):
            ops.int4_pages(*args)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_nothing(device):
    pools = [ops.int4_pages(0, 2, 64, device=device) for _ in range(2)]
    table, lengths = torch.zeros(2, 0, dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int32, device=device)
    new = torch.ones(2, 3, 2, 64, device=device)
    ops.store_rows_int4(new, new, *pools, table, lengths)
    ops.store_rows_int4(new[:, :0], new[:, :0], *pools, table, lengths)
    assert (ops.read_rows_int4(*pools, table, lengths, 4, 64, BF)[1] == 0).all() and ops.read_rows_int4(*pools, table, lengths, 0, 64, BF)[0].shape == (2, 0, 2, 64)
    for dtype in (BF, F):
        assert (ops.paged_attention_int4(torch.ones(2, 4, 64, dtype=dtype, device=device), *pools, table, lengths) == 0).all()
        assert ops.paged_attention_int4(torch.ones(0, 4, 64, dtype=dtype, device=device), *pools, table[:0], lengths[:0]).shape == (0, 4, 64)
    gemm.check_error()


@gpu
def test_pages_copied_with_the_others():
    s = make([70, 20], 4, 2, 64)
    ops.copy_pages_([s["k"], s["v"]], s["table"][0, :2].tolist(), [int(p) for p in range(s["k"].shape[0]) if p not in s["table"][0, :2].tolist() + s["table"][1, :1].tolist()][:2])
    free = [int(p) for p in range(s["k"].shape[0]) if p not in s["table"][0, :2].tolist() + s["table"][1, :1].tolist()][:2]
    want = attend(s)
    s["table"][0, :2] = torch.tensor(free, dtype=torch.int32)
    assert torch.equal(attend(s), want)


def test_sizes_that_the_kernels_do_not_count():
    """Refused by shape alone: long tables and pages, many heads."""
    lengths = torch.zeros(1, dtype=torch.int32)
    pool = ops.int4_pages(1, 1, 32)
    with pytest.raises(ValueError, match="longer tables"):
        ops.read_rows_int4(pool, pool, torch.zeros(1, dtype=torch.int32).expand(1, (1 << 31) // 64), lengths, 1, 32, F)
    with pytest.raises(ValueError):
        ops.int4_pages(1, 1, 32, 65552)
    wide = torch.zeros(0, 32768, 320, dtype=torch.uint8)
    with pytest.raises(ValueError, match="heads are more"):
        ops.read_rows_int4(wide, wide, torch.zeros(1, 0, dtype=torch.int32), lengths, 1, 32, F)


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("H,G,D", [(2, 2, 128), (4, 2, 32), (9, 3, 96), (16, 4, 128), (8, 2, 64), (10, 2, 64), (16, 2, 128), (12, 1, 96), (20, 1, 128)])
def test_weights_times_sizes_of_22_bits(H, G, D, dtype):
    """The output is the 64-bit value rounded once, to the neighbour that 22 bits of a weight times its value's size leave open.  With queries as small as here scores are off by less than 2^-24, so what is left
    of a weight's room is 2^-20 for its exponential and 2^-22; rounding is monotone, so the output lies between the rounded ends of that room (a number goes to 32 bits on its way to 16: 2^-24 more)."""
    for lens in ([1, 2, 3, 5, 9, 17, 33, 70], [1500, 4], [20000]):
        s = make(lens, H, G, D, dtype=dtype, size=1e-3)
        for kw in (dict(), dict(window=6)):
            got = attend(s, **kw)
            want, room = formula(dict(s, q=s["q"].float()), tensor=True, **kw)
            room = room + 2.0 ** -24 * want.abs()
            low, high = (want - room).to(dtype), (want + room).to(dtype)
            wrong = (got < low) | (got > high)
            assert not wrong.any(), (lens, kw, int(wrong.sum()), wrong.numel())
    gemm.check_error()


def test_sizes_are_not_negative():
    """Of zeros either sign has a size of +0: as bits the other one is larger than every size."""
    x = torch.cat([-torch.zeros(1, 32), torch.zeros(1, 32), torch.tensor([[-0.0, 0.0] * 16]), torch.full((1, 32), -2.0)])
    code, low, size = R.encode(x)
    assert (size.view(torch.int16) >= 0).all() and not size.any() and not code.any() and low.flatten().tolist() == [0.0, 0.0, 0.0, -2.0]


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, F])
@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (16, 2, 128), (3, 1, 96), (1, 1, 32)])
def test_values_of_negative_zeros(H, G, D, dtype):
    """A key whose value is nothing but -0.0 leaves the others as they are."""
    def values(gen, n, G, D):
        x = torch.randn(n, G, D, generator=gen)
        x[n // 2] = -0.0
        x[n // 3, :, :32] = -0.0
        return x
    s = make([40, 9, 1, 700], H, G, D, dtype=dtype, values=values)
    pools = [torch.full_like(s[k], 255) for k in "kv"]                # (the rows once more, by the kernel)
    rows = ops.read_rows_int4(s["k"], s["v"], s["table"], s["lengths"], 700, D, F)
    back = [torch.cat([torch.zeros(700 - n, G, D, device="cuda"), r[i, :n]]) for r in rows for i, n in enumerate([40, 9, 1, 700])]
    back = [torch.where(r == 0, -0.0, r) for r in back]
    ops.store_rows_int4(torch.stack(back[:4]), torch.stack(back[4:]), *pools, s["table"], s["lengths"])
    for k, v in ((s["k"], s["v"]), pools):
        check(dict(s, k=k, v=v))
        check(dict(s, k=k, v=v), window=20)


@gpu
@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (8, 1, 64), (6, 2, 96), (2, 1, 32)])
@pytest.mark.parametrize("size", [1e35, 1e30, 1e-30, 1e-35])
def test_values_far_from_one(size, H, G, D):
    """Values whose sizes are powers of two from -118 to 118: scaled for the products and back without leaving 32 bits, also where the largest score so far lags behind (scores of up to 5).  Sums below 2^-126 are zeros: of a
    warp's rounded, rest and low sums, four warps, up to eight parts, before the division by a sum of weights of one at least, and of the output: 97 times 2^-126 at most."""
    floor = 97 * 2.0 ** -126

    def check(s, **kw):
        got = attend(s, **kw).double()
        want, room = formula(s, **kw)
        assert got.isfinite().all() and ((got - want).abs() <= 2.0 ** -8 * (want.abs() + room) + room + floor).all()
        gemm.check_error()
    for lens, scores in (([300, 20, 1], 1.5), ([200, 33], 4.0)):
        s = make(lens, H, G, D, size=scores)
        s["v"] = make(lens, H, G, D, values=lambda gen, n, G, D: torch.randn(n, G, D, generator=gen) * size)["v"]      # (the same pages)
        check(s)
        check(s, cap=3.0, window=70)
    # sizes that grow and shrink by many powers of two on the way
    s["v"] = make(lens, H, G, D, values=lambda gen, n, G, D: torch.randn(n, G, D, generator=gen) * size * 2.0 ** torch.randint(-20, 3, (n, 1, 1), generator=gen))["v"]
    check(s)


@gpu
@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (8, 1, 64)])
def test_values_near_the_largest_number(H, G, D):
    """One or two keys' values of up to 1.6 10^38, whose sum 32 bits still hold."""
    s = make([1, 2, 2], H, G, D)
    s["v"] = make([1, 2, 2], H, G, D, values=lambda gen, n, G, D: torch.rand(n, G, D, generator=gen) * 3.2e38 - 1.6e38)["v"]
    check(s)


@gpu
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (8, 1, 64), (6, 2, 96)])
@pytest.mark.parametrize("power", [110, 117, 120, 125, -90, -110])
def test_queries_far_from_one(power, H, G, D, dtype):
    """Queries of 2^110 to 2^127 and of 2^-90 to 2^-112 with keys that bring the scores back to a few: the same bounds, which grow with scale, query and key alike."""
    keys = -power // 2
    for lens in ([300, 20, 1], [200, 33]):
        s = make(lens, H, G, D, dtype=dtype)
        s["k"] = make(lens, H, G, D, values=lambda gen, n, G, D: torch.randn(n, G, D, generator=gen) * 2.0 ** keys)["k"]      # (the same pages)
        s["q"] = (s["q"].double().clamp(-3.9, 3.9) * 2.0 ** power).to(dtype)
        scale = D ** -0.5 * 2.0 ** (-power - keys)
        check(s, scale=scale)
        check(s, scale=scale, cap=3.0, window=70)
        check(s, scale=scale, slopes=ops.alibi_slopes(H).cuda())
