"""A beam's selection where a part of a row is many chunks of 4096 logits, and where rows that are equal begin at different places of a 16-byte vector.

Bounds.  A thread's sum of exponentials takes, per chunk, 16 terms, each within 2.4 2^-23 of the largest one (CUDA's bound of 2 + 1.2 |t| steps for e^t), six additions, and a factor
e^-t for what was summed so far.  That factor's error, (2 + 1.2 t) 2^-23, counts with the share u / (1 + u), u = S e^-t, that S has of the new sum; with S of at most 16 terms a chunk, 2^9 here,
it is below 6 2^-23.  Joining threads and parts adds two more factors and ten additions.  With c chunks the sum is within (2.4 + 9 c + 2 6 + 5) 2^-23, as is its logarithm, and a score is within that and
2^-24 |score| of the one in 64 bits.  Candidates of one beam are compared by their logits alone, so their order is exact; those of different beams may change places within the bound."""
import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.ops import beam as BM
from test_beam import want

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def check(logits, scores, n, chunks):
    V = logits.shape[2]
    s, b, t = ops.beam_select(logits, scores, n)
    ws = want(logits, scores, n)[0]
    tol = (19.4 + 9 * chunks) * 2.0 ** -23 + 2.0 ** -24 * ws.abs()
    fin = torch.isfinite(ws)
    assert torch.equal(s[~fin].double(), ws[~fin]) and ((s.double() - ws).abs() <= tol)[fin].all()
    assert (s[:, :-1] >= s[:, 1:]).all()
    x = logits.double().nan_to_num(nan=-torch.inf, posinf=torch.inf, neginf=-torch.inf)
    top = x.amax(-1, keepdim=True)
    lp = x - top - (x - top).exp().sum(-1, keepdim=True).log()
    for i in range(len(s)):
        own = scores[i, b[i]].double() + lp[i, b[i], t[i]]               # what was chosen has the score that is given for it
        ok = torch.isfinite(own)
        assert torch.equal(ok, fin[i]) and ((own - s[i].double()).abs() <= tol[i])[ok].all()
        place = (b[i] * V + t[i]).tolist()
        assert len(set(place)) == n
        for beam in set(b[i][ok].tolist()):                               # a beam's own: the best of its logits, in order, ties to the lowest token
            got = t[i][ok & (b[i] == beam)]
            order = torch.sort(x[i, beam], descending=True, stable=True)
            assert torch.equal(got, order.indices[:len(got)])


def chunks_of(N, K, V):
    """Chunks of a part on a GPU of 148 SMs."""
    parts = max(1, min(-(-V // BM.CHUNK), 4 * 148 // (N * K)))
    return -(-(-(-V // parts)) // BM.CHUNK)


SHAPES = [(16, 8, 40000), (1, 128, 40000), (2, 64, 33001), (37, 8, 12290)]


def inputs(N, K, V, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn(N, K, V, generator=gen, device="cuda") * 3).to(dtype)
    return logits, -5 - 4 * torch.randn(N, K, generator=gen, device="cuda").abs()


def test_these_shapes_have_several_chunks():
    for shape in SHAPES:
        assert chunks_of(*shape) > 1


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,V", SHAPES)
def test_several_chunks(N, K, V, dtype):
    c = chunks_of(N, K, V)
    logits, scores = inputs(N, K, V, dtype)
    for n in (1, 16, 128):
        check(logits, scores, n, c)
    # rows that begin at every place of a vector
    wide = inputs(N, K, V + 7, dtype, 1)[0]
    for skew in range(1, 8):
        check(wide[:, :, skew:V + skew], scores, 16, c)
    # the best ones last; ties all over the row; a first chunk of nothing, of one value, of more equal ones than are held
    check(logits.sort(dim=-1).values, scores, 16, c)
    check(logits.sort(dim=-1, descending=True).values, scores, 128, c)
    check(logits.round(), scores, 128, c)
    x = logits.clone()
    x[:, :, :BM.CHUNK] = -torch.inf
    check(x, scores, 16, c)
    x[:, :, :BM.CHUNK] = torch.nan
    check(x, scores, 16, c)
    x[:, :, :BM.CHUNK] = 9.0
    check(x, scores, 16, c)
    x[:, :, :BM.CHUNK] = -40.0
    check(x, scores, 128, c)
    x[:, :, BM.CHUNK:] = 3.0
    check(x, scores, 128, c)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [4099, 8191, 20001, 50257])
def test_equal_rows_at_any_place(device, dtype, V):
    """Beams with the same logits and scores: ties go to the lowest beam, though their rows (of an odd number of logits) begin at different places of a vector."""
    for seed in range(4 if device == "cuda" else 1):
        gen = torch.Generator().manual_seed(seed)
        row = (torch.randn(V, generator=gen) * 3).to(dtype)
        if dtype != torch.float32:
            row[torch.randperm(V, generator=gen)[:40]] = (torch.arange(40) / 8 + 14).to(dtype)
        logits = row.to(device).expand(2, 9, V).contiguous()
        scores = torch.tensor([-1.7, -0.3], device=device)[:, None].expand(2, 9).contiguous()
        s, b, t = ops.beam_select(logits, scores, 36)
        lp = torch.log_softmax(row.double(), -1)                          # of the one row that they all are (sums of its copies need not have the same bits)
        total = (scores.cpu().double()[:, 0, None] + lp)[:, None].expand(2, 9, V).flatten(1)
        at = torch.sort(total, dim=-1, descending=True, stable=True).indices[:, :36].to(device)
        assert torch.equal(b, at // V) and torch.equal(t, at % V)
        assert (s.view(2, -1, 9) == s.view(2, -1, 9)[:, :, :1]).all()


def test_places_stay_below_32_bits():
    """The last number that a part's chunks (and the one asked for ahead) count up to, at the largest searches that the kernels take."""
    for N, K in ((1, 1), (1, 3), (1, 128), (4, 2), (500, 128), (60000, 1)):
        V = BM.PLACES // K
        assert BM._held(N, K, V, 1) and not BM._held(N, K, V + K, 1)
        for V in (V, V - 1, V - BM.CHUNK, 5):
            parts, length = BM._shares(N, K, V, 4 * 148)
            assert parts * length >= V and length % 8 == 0
            assert (parts - 1) * length + -(-length // BM.CHUNK) * BM.CHUNK < 1 << 31
    assert not BM._held(0, 1, 10, 1) and not BM._held(1, 129, 10, 1) and not BM._held(1, 1, 1000, 129) and not BM._held(65536, 1, 10, 1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [301, 4099, 20001])
def test_equal_rows_of_a_wide_search(device, V):
    """The same with more beams than the kernels hold."""
    for seed in range(4):
        row = torch.randn(V, generator=torch.Generator().manual_seed(seed)) * 3
        s, b, t = ops.beam_select(row.to(device).expand(1, 131, V).contiguous(), torch.full((1, 131), -0.7, device=device), 262)
        best = torch.sort(row, descending=True, stable=True).indices[:2]
        assert b[0].tolist() == 2 * list(range(131)) and t[0].tolist() == [int(x) for x in best for _ in range(131)]
