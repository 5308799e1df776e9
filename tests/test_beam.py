"""A beam search's selection and the reordering of its states.

Selection against a stable sort of the scores in 64 bits.  Beams and tokens have to be equal.  The logits' sum is taken from 32-bit exponentials, each within (2 + 1.2 |t|) 2^-23 of
e^t by CUDA's bound, so within 2.4 2^-23 of the largest term, and of nine 32-bit additions, 2^-24 each: 7 2^-23 of the sum at most, 2^-20 in its logarithm.  A score is within
2^-20 + 2^-24 |score| of the one in 64 bits, and the tests' candidates from different beams lie further apart than that or are equal in every bit."""
import pytest
import torch

from linear_moe_b200 import ops
from linear_moe_b200.ops import beam as BM

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def want(logits, scores, n):
    x = logits.double()
    x = torch.where(torch.isnan(x), -torch.inf, x)
    top = x.amax(-1, keepdim=True)
    x = x - torch.where(top == -torch.inf, 0.0, top)          # before the logarithm joins: logits of the type's lowest value would swallow it
    lp = torch.where(top == -torch.inf, -torch.inf, x - x.exp().sum(-1, keepdim=True).log())
    total = (scores.double()[..., None] + lp).flatten(1)
    best, at = torch.sort(total, dim=-1, descending=True, stable=True)
    return best[:, :n], at[:, :n] // logits.shape[2], at[:, :n] % logits.shape[2]


def check(logits, scores, n):
    s, b, t = ops.beam_select(logits, scores, n)
    ws, wb, wt = want(logits, scores, n)
    assert s.dtype == torch.float32 and b.dtype == t.dtype == torch.int64 and s.shape == b.shape == t.shape == ws.shape
    assert torch.equal(b, wb) and torch.equal(t, wt)
    fin = torch.isfinite(ws)
    assert torch.equal(s[~fin].double(), ws[~fin])
    assert ((s.double() - ws)[fin].abs() <= 2.0 ** -20 + 2.0 ** -24 * ws[fin].abs()).all()


def inputs(N, K, V, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(N, K, V, generator=gen) * 3).to(dtype)
    scores = -5 - 4 * torch.randn(N, K, generator=gen).abs()
    return logits.to(device), scores.to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,V,n", [(1, 1, 1, 1), (1, 4, 1000, 8), (3, 5, 8193, 10), (2, 1, 24577, 2), (2, 8, 8185, 128), (1, 128, 130, 128), (2, 3, 50, 150), (1, 2, 8186, 4),
                                     (1, 3, 16400, 6), (2, 2, 300, 100)])
def test_selection(device, dtype, N, K, V, n):
    """Around a part's 8192 numbers, rows that begin off the 16-byte boundaries, more candidates than a part has tokens, all of them."""
    check(*inputs(N, K, V, dtype, device), n)


@pytest.mark.parametrize("device", DEVICES)
def test_equal_logits(device):
    """Ties go to the lowest place: few values, one value, whole parts of it; equal beams."""
    logits, scores = inputs(2, 3, 9001, torch.float32, device)
    check(logits.round(), scores, 12)
    check((logits > 3).float(), torch.zeros_like(scores), 128)
    same = torch.zeros(1, 4, 20000, device=device)
    s, b, t = ops.beam_select(same, torch.zeros(1, 4, device=device), 30)
    assert (b == 0).all() and t[0].tolist() == list(range(30))
    s, b, t = ops.beam_select(same, torch.tensor([[0.0, 1.0, 1.0, 0.5]], device=device), 30)
    assert (b == 1).all() and t[0].tolist() == list(range(30))


@pytest.mark.parametrize("device", DEVICES)
def test_masked_logits(device):
    """Minus infinity, the type's lowest value, NaN, beams of nothing, beams that are dead."""
    logits, scores = inputs(2, 4, 5000, torch.float32, device)
    logits[0, :, 100:] = -torch.inf
    logits[1, 0] = torch.finfo(torch.float32).min
    logits[1, 1, 7:900] = torch.nan
    logits[0, 2] = -torch.inf
    logits[1, 3] = torch.nan
    check(logits, scores, 16)
    scores[1, 2] = -torch.inf
    check(logits, scores, 16)
    only = torch.full((1, 2, 4100), -torch.inf, device=device)
    only[0, 1, 4099] = 2.0
    check(only, torch.zeros(1, 2, device=device), 6)
    check(torch.full((1, 2, 9000), -torch.inf, device=device), torch.zeros(1, 2, device=device), 6)


@pytest.mark.parametrize("device", DEVICES)
def test_views(device):
    logits, scores = inputs(2, 3, 2 * 501 + 1, torch.bfloat16, device)
    check(logits[:, :, ::2], scores, 6)
    check(logits[:, :, 1:502], scores, 6)
    check(logits.transpose(0, 1), scores.t(), 4)
    check(logits[:1].expand(4, 3, 1003), scores[:1].expand(4, 3), 6)


def test_selection_refusals():
    logits, scores = inputs(2, 3, 10, torch.float32, "cpu")
    for a, b, n in [(logits[0], scores[0], 2), (logits, scores[:1], 2), (logits.double(), scores, 2), (logits, scores.double(), 2), (logits, scores, 0), (logits, scores, 31)]:
        with pytest.raises(ValueError):
            ops.beam_select(a, b, n)
    s, b, t = ops.beam_select(logits[:0], scores[:0], 2)
    assert s.shape == b.shape == t.shape == (0, 2)


@gpu
def test_wide_search():
    """More candidates than the kernels hold."""
    check(*inputs(1, 130, 300, torch.float32, "cuda"), 260)


@gpu
def test_selection_in_a_graph():
    logits, scores = inputs(3, 4, 20000, torch.float32, "cuda")
    first = ops.beam_select(logits, scores, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.beam_select(logits, scores, 8)
    for seed in (1, 2):
        logits.copy_(inputs(3, 4, 20000, torch.float32, "cuda", seed)[0])
        graph.replay()
        for a, b in zip(got, ops.beam_select(logits, scores, 8)):
            assert torch.equal(a, b)
    assert not torch.equal(first[2], got[2])


@pytest.mark.parametrize("device", DEVICES)
def test_reorder(device):
    """Rows of every size and type, strided ones, empty ones; more tensors than one launch takes; the same row twice."""
    gen = torch.Generator().manual_seed(0)
    parents = torch.tensor([3, 3, 0, 5, 1, 1, 2], device=device)
    states = [torch.randn(6, 2, 33, 65, generator=gen).to(device), torch.randn(6, 7, generator=gen).half().to(device), torch.randint(0, 99, (6,), generator=gen).to(device),
              torch.randint(0, 99, (6, 13), generator=gen, dtype=torch.uint8).to(device), torch.randn(5, 6, 300, generator=gen).bfloat16().to(device).transpose(0, 1),
              torch.zeros(6, 0, device=device), torch.randn(6, 100001, generator=gen).to(device)]
    states += [torch.randn(6, i + 1, generator=gen).to(device) for i in range(70)]
    got = ops.reorder_states(states, parents)
    for a, b in zip(got, states):
        assert torch.equal(a, b[parents]) and a.is_contiguous()
    assert ops.reorder_states([], parents) == []
    assert ops.reorder_states(states[:1], parents[:0])[0].shape == (0, 2, 33, 65)


def test_reorder_refusals():
    t = torch.zeros(4, 2)
    for states, parents in [([t], torch.zeros(2, dtype=torch.int32)), ([t], torch.zeros(2, 2, dtype=torch.int64)), ([torch.tensor(1.0)], torch.zeros(2, dtype=torch.int64))]:
        with pytest.raises(ValueError):
            ops.reorder_states(states, parents)
    with pytest.raises(IndexError):
        ops.reorder_states([t], torch.tensor([4]))
    for src, dst in [([0], [0]), ([0, 1], [2, 2]), ([0], [4]), ([-1], [2]), ([0, 1], [2]), ([0, 1], [1, 2])]:
        with pytest.raises(ValueError):
            ops.copy_pages_([t], src, dst)
    with pytest.raises(ValueError):
        ops.copy_pages_([t.t()], [0], [1])


@gpu
def test_parents_that_are_none():
    from linear_moe_b200.ops import gemm
    t = torch.arange(12.0, device="cuda").view(4, 3)
    got = ops.reorder_states([t], torch.tensor([1, 4, -1, 3], device="cuda"))[0]
    with pytest.raises(RuntimeError, match="0x13000"):
        gemm.check_error()
    assert torch.equal(got[0], t[1]) and torch.equal(got[3], t[3])


@pytest.mark.parametrize("device", DEVICES)
def test_copy_pages(device):
    pools = [torch.randn(9, 64, 2, 8, device=device).bfloat16(), torch.randn(9, 3, device=device)]
    old = [p.clone() for p in pools]
    ops.copy_pages_(pools, [1, 1, 8], [0, 5, 2])
    for p, o in zip(pools, old):
        o[[0, 5, 2]] = o[[1, 1, 8]]
        assert torch.equal(p, o)
    ops.copy_pages_(pools, [], [])


def test_pools_on_two_devices():
    with pytest.raises(ValueError):
        ops.copy_pages_([torch.zeros(4, 2), torch.zeros(4, 2, device="meta")], [0], [1])


@gpu
def test_state_without_rows():
    """Every parent is one too many."""
    from linear_moe_b200.ops import gemm
    assert ops.reorder_states([torch.zeros(0, 3, device="cuda")], torch.tensor([0, 1], device="cuda"))[0].shape == (2, 3)
    with pytest.raises(RuntimeError, match="0x13000"):
        gemm.check_error()
