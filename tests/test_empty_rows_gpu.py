"""GPU: query rows that see no key, in work large enough for the persistent pairs of query blocks (fewer blocks are divided by keys)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("how", ["bottom-right", "bool", "add"])
def test_rows_without_keys_beside_rows_with_some(dtype, D, how):
    from tinytorch_b200 import op
    B, H, L, S = 64, 16, 200, 60
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(B, H, n, D, generator=g, device="cuda").to(dtype) for n in (L, S, S))
    if how == "bottom-right":
        o, lse = op.sdpAttentionFwd(q, k, v, isCausal="bottom-right")
        empty = torch.arange(L, device="cuda") < L - S
    else:
        empty = torch.arange(L, device="cuda") % 3 == 1
        sees = ~empty[:, None].expand(L, S)
        mask = sees if how == "bool" else torch.zeros(L, S, device="cuda").masked_fill(~sees, -math.inf).to(dtype)
        o, lse = op.sdpAttentionFwd(q, k, v, attnMask=mask)
    assert not o[:, :, empty].any() and bool((lse[:, :, empty] == -math.inf).all())
    assert bool(torch.isfinite(lse[:, :, ~empty]).all()) and bool(o[:, :, ~empty].any(-1).all())
