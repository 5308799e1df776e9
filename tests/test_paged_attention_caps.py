"""One-token attention with caps far above its scores, on the tensor cores: cap tanh(x / cap) is x nearly, to the bounds of test_paged_attention.py.

tanh has a relative error of 9e-7, whatever the cap, so scores of up to 40 are off by 4e-5 (5e-5 in units of log 2) and weights by as much, below the quarter of u (fp16: 1.2e-4) that those
bounds leave for the 32-bit part."""
import pytest
import torch

from test_paged_attention import check, make, slope_table

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(8, 2), (16, 1)])
@pytest.mark.parametrize("cap", [0.01, 1.0, 6.0, 100.0, 1e3, 1e4, 1e5, 1e6, 9e6])
def test_caps(dtype, heads, cap):
    s = make([1, 20, 300, 1500], *heads, 64, dtype=dtype, size=4.0)
    check(s, cap=cap)
    check(s, cap=cap, slopes=slope_table(heads[0]))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_and_step_agree(dtype):
    """The last row of a prompt and one token from pages have the same capped scores."""
    from linear_moe_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = (torch.randn(1, 256, h, 128, generator=gen, device="cuda").to(dtype) for h in (8, 2, 2))
    q = q * 4
    table, lengths = torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.tensor([256], dtype=torch.int32, device="cuda")
    for cap in (50.0, 1e5, 9e6):
        a = ops.softmax_attention(q, k, v, softcap=cap)[:, -1]
        b = ops.paged_attention(q[:, -1], k.view(4, 64, 2, 128), v.view(4, 64, 2, 128), table, lengths, softcap=cap)
        # each within its weights' and its own rounding (2 u) and a quarter
        assert ((a.double() - b.double()).norm() / a.double().norm()).item() < 4.5 * torch.finfo(dtype).eps / 2
