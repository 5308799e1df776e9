"""One-token attention with NaN in what a head sees: the head gives NaN, whichever kernel and however many CTAs have its keys; hidden NaN changes nothing.

The definition decides where NaN is: a query's or a key's NaN makes all weights of the heads that see it NaN, a value's one number of their results.  Bounds of the rest: as in
test_paged_attention.py."""
import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.ops import paged_attn as PA
from test_paged_attention import formula, make, slope_table

gpu = pytest.mark.gpu
# (type, head size, page, parts of a request: None for the rule's own)
KERNELS = [("cpu", torch.float32, 24, 16, None),
           *[pytest.param("cuda", t, d, 64, s, marks=gpu) for t, d in ((torch.bfloat16, 128), (torch.float16, 64)) for s in (1, 3, 8, 64, None)],
           *[pytest.param("cuda", t, d, p, None, marks=gpu) for t, d, p in ((torch.float32, 64, 64), (torch.bfloat16, 192, 64), (torch.float16, 64, 10), (torch.float32, 300, 16))]]


def cut(monkeypatch, parts):
    """Requests in so many parts; plans of other tests' calls of the same layout are put aside."""
    if parts is not None:
        monkeypatch.setattr(PA, "_PLANS", {})
        monkeypatch.setattr(PA, "splits_of", lambda *a: (parts, 0))


def check(s, where, window=None, cap=None, slopes=None):
    """`where` [B, H, D]: the results that have to be NaN."""
    want, mag, low, _, _ = formula(s, window, cap, slopes)
    assert torch.equal(want.isnan(), where)
    got = ops.paged_attention(s["q"], s["k"].clone(), s["v"].clone(), s["table"], s["lengths"], None, window, softcap=cap, slopes=slopes, k_new=s["k_new"], v_new=s["v_new"])
    assert torch.equal(got.isnan(), where)
    dtype, fin = s["q"].dtype, ~where
    err = (got.double() - want).abs()[fin]
    if dtype == torch.float32:
        assert (err <= 64 * 2.0 ** -24 * mag[fin]).all()
    else:
        u = torch.finfo(dtype).eps / 2
        assert (err <= 2.25 * u * mag[fin] + torch.finfo(dtype).smallest_normal * u * (low.expand_as(mag)[fin] + 1)).all()


@pytest.mark.parametrize("device,dtype,D,page,parts", KERNELS)
@pytest.mark.parametrize("options", [dict(), dict(cap=20.0, bias=True)])
def test_visible_nan(device, dtype, D, page, parts, options, monkeypatch):
    cut(monkeypatch, parts)
    H, G = 6, 2
    kw = dict(cap=options.get("cap"), slopes=slope_table(H, device) if options.get("bias") else None)

    def fresh():
        return make([700, 3, 40], H, G, D, page=page, dtype=dtype, device=device)

    def row(s, b, key):
        return int(s["table"][b, key // page]), key % page
    nothing = torch.zeros(3, H, D, dtype=torch.bool, device=device)
    check(fresh(), nothing, **kw)
    # a query head
    for b, h in ((0, 1), (1, 5), (2, 0)):
        s, where = fresh(), nothing.clone()
        s["q"][b, h, D // 3] = torch.nan
        where[b, h] = True
        check(s, where, **kw)
    # a key and a value: the first one, ahead of and behind others of the same warp, the last in the cache, the new one
    for b, key in ((0, 0), (0, 5), (0, 130), (0, 333), (0, 698), (1, 1), (2, 17)):
        s, where = fresh(), nothing.clone()
        s["k"][(*row(s, b, key), 1, 2)] = torch.nan
        where[b, H // G:] = True
        check(s, where, **kw)
        s, where = fresh(), nothing.clone()
        s["v"][(*row(s, b, key), 0, 3)] = torch.nan
        where[b, :H // G, 3] = True
        check(s, where, **kw)
    for b in range(3):
        s, where = fresh(), nothing.clone()
        s["k_new"][b, 0, D - 1] = torch.nan
        s["v_new"][b, 1, 0] = torch.nan
        where[b, :H // G] = True
        where[b, H // G:, 0] = True
        check(s, where, **kw)


@pytest.mark.parametrize("device,dtype,D,page,parts", KERNELS)
def test_hidden_nan(device, dtype, D, page, parts, monkeypatch):
    """Keys in front of the window, and (as everywhere in these tests) rows behind the last key and pages of nobody."""
    cut(monkeypatch, parts)
    window = 45
    s = make([700, 3, 60], 6, 2, D, page=page, dtype=dtype, device=device)
    for b, n in ((0, 700), (2, 60)):
        for key in range(n - window):
            s["k"][int(s["table"][b, key // page]), key % page] = torch.nan
            s["v"][int(s["table"][b, key // page]), key % page] = torch.nan
    check(s, torch.zeros(3, 6, D, dtype=torch.bool, device=device), window)
