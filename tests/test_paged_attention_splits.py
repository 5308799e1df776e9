"""One-token attention with a request's keys in any number of parts: one CTA, a cluster, parts that a second launch joins.  Bounds: as in test_paged_attention.py."""
import pytest
import torch

from linear_moe_b200.ops import paged_attn as PA
from test_paged_attention import check, make, slope_table


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 72)])
@pytest.mark.parametrize("splits", [1, 2, 3, 5, 7, 8, 16, 31, 64])
def test_parts(splits, dtype, D, monkeypatch):
    """More parts than a request has keys for among them; the longest requests first or not."""
    for longest_first in (0, 1):
        monkeypatch.setattr(PA, "_PLANS", {})
        monkeypatch.setattr(PA, "splits_of", lambda *a: (splits, longest_first))
        s = make([0, 5, 256, 257, 2000, 4097], 8, 2, D, dtype=dtype, size=4.0)
        check(s, cap=50.0)
        check(s, 1000, slopes=slope_table(8))
        s = make([1, 300, 1100], 32, 2, D, dtype=dtype)
        check(s)
