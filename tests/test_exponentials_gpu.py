"""GPU: the 16-bit kernels take some exponentials on the FMA pipe (forward, D = 64: the keys 1, 17, 33, ... of a tile; backward: every eighth
query); they are huge and 0 where the others are."""
import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


SHAPES = [(24, 16, 200, 600), (2, 16, 300, 600), (1, 2, 40, 1500)]  # pairs of query blocks, single blocks, divided over a cluster


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("nats", [60, 95, 130, 177, 190, 250, 267, 300, 350, 1000])
def test_one_score_far_above_the_tiles_before(dtype, D, shape, nats):
    """A row's reference is the maximum of its first tile, and a later key is far above it (2^87 ... 2^1443): O is that key's value."""
    from tinytorch_b200 import op
    B, H, L, S = shape
    q, k = torch.zeros(B, H, L, D, device="cuda", dtype=dtype), torch.zeros(B, H, S, D, device="cuda", dtype=dtype)
    v = randn((B, H, S, D), dtype, 1)
    q[..., 0] = 1
    for at in (128 * 2 + 17, 128 * 3 + 49, 128 * 4 + 1, 128 * 3 + 50):
        y = k.clone()
        y[:, :, at, 0] = nats
        o, lse = op.sdpAttentionFwd(q, y, v, scale=1.0)
        # One probability is 1, the others vanish.  On the FMA pipe that 1 is off by up to 7.5e-5, which rounds to 1 in P but not in the
        # sum that the result, rounded once, is divided by.
        want, slop = v[:, :, at:at + 1].double().expand_as(o), 7.6e-5 if D == 64 else 0.0
        assert bool(((o.double() - want).abs() <= (slop + ref.HALF[dtype]) * want.abs() * (1 + 2.0 ** -12) + ref.TINY[dtype]).all())
        # (to the base 2 and back: the roundings of two products and of log2 e, 2^-23 each at the most)
        size = float(y[0, 0, at, 0])
        assert bool(((lse - size).abs() <= 2.0 ** -21 * size + slop).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_hidden_pairs_give_nothing_to_gradients(dtype, D):
    """A boolean mask hides keys in every column: their dK and dV are 0 to the bit, whatever the values and gradients are."""
    from tinytorch_b200 import function
    B, H, L, S = 2, 8, 150, 200
    q, k, v = (randn((B, H, n, D), dtype, i).requires_grad_() for i, n in enumerate((L, S, S)))
    hidden = torch.arange(S, device="cuda") % 3 == 1
    mask = (~hidden).expand(L, S).clone()
    mask[:, :4] = True  # (not one that comes down to a length)
    mask[0, 2] = False
    hidden = ~mask.any(0)
    big = 60000.0 if dtype == torch.float16 else 3e38
    dq, dk, dv = torch.autograd.grad(function.sdpAttention(q, k, v, attnMask=mask), (q, k, v), randn((B, H, L, D), dtype, 9))
    assert not dk[:, :, hidden].any() and not dv[:, :, hidden].any()
    scaled = torch.autograd.grad(function.sdpAttention(q, k, v, attnMask=mask), v, torch.full((B, H, L, D), big, dtype=dtype, device="cuda"))[0]
    assert not scaled[:, :, hidden].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("causal", [False, True])
def test_hidden_values_give_nothing(D, shape, causal):
    """The largest values of bf16 behind hidden keys of every column, of a mask or beyond the triangle, leave not a bit."""
    from tinytorch_b200 import op
    B, H, L, S = shape
    q, k, v = (randn((B, H, n, D), torch.bfloat16, i) for i, n in enumerate((L, S, S)))
    if causal:
        kw, rows, hidden = dict(isCausal=True), slice(0, 30), torch.arange(S, device="cuda") >= 30
    else:
        hidden = torch.arange(S, device="cuda") % 3 == 1
        mask = (~hidden).expand(L, S).clone()
        mask[0, 2] = False  # (not one that comes down to a length)
        kw, rows = dict(attnMask=mask), slice(0, L)
    want = op.sdpAttentionFwd(q, k, v.masked_fill(hidden[:, None], 0.0), **kw)
    got = op.sdpAttentionFwd(q, k, v.masked_fill(hidden[:, None], 3e38), **kw)
    assert torch.equal(got[0][:, :, rows], want[0][:, :, rows]) and torch.equal(got[1], want[1])
