"""GPU: NaN and infinities in operands of attention come out where the 64-bit form has them, in every division of the work: none is
taken for a row without keys."""
import math

import pytest
import torch

import lm_reference as ref
import not_finite as nf

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SHAPES = {
    "pairs": (24, 16, 4, 200, 190),      # B, Hq, Hkv, L, S: persistent pairs of query blocks
    "keys": (2, 16, 4, 300, 290),        # single blocks, divided by keys
    "cluster": (1, 2, 1, 40, 1500),      # ... over the CTAs of a cluster
}


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def run(shape, D, dtype, how, poisoned, at, value, where):
    from tinytorch_b200 import op
    B, Hq, Hkv, L, S = SHAPES[shape]
    x = {n: randn((B, h, r, D), dtype, i) for i, (n, h, r) in enumerate((("q", Hq, L), ("k", Hkv, S), ("v", Hkv, S)))}
    # q's channel has one sign, so that an infinite k gives all rows of a head scores of one sign
    x["q"][..., 5] = x["q"][..., 5].abs() + 0.1
    x[poisoned] = nf.poison(x[poisoned], (B - 1, 0, at), value, where)
    q, k, v = x.values()
    kw, added = {}, None
    if how in ("bool", "add"):
        sees = (torch.arange(L, device="cuda")[:, None] * 7 + torch.arange(S, device="cuda") * 3) % 5 > 0
        sees[:, 1] = True
        sees[L // 3] = False  # (a row that sees nothing)
        if how == "bool":
            kw["attnMask"] = sees
        else:
            # a row that sees nothing keeps no -inf beside a NaN: NaN - inf is NaN
            added = torch.zeros(L, S, device="cuda").masked_fill(~sees, -1e4).to(dtype)
            added[L // 3] = 0
            kw["attnMask"], sees = added, torch.ones_like(sees)
    else:
        sees = ref.visible(L, S, how, "cuda")
        kw["isCausal"] = how
    o, lse = op.sdpAttentionFwd(q, k, v, **kw)
    group, b = Hq // Hkv, B - 1
    kk, vv = (t[b].double().repeat_interleave(group, 0) for t in (k, v))
    want = nf.attention(q[b].double(), kk, vv, 1 / math.sqrt(D), sees, None if added is None else added.double())
    if poisoned == "v":  # (who does not see it may meet it in a tile, as 0 times what it holds)
        met = ~o[b, :group].isfinite()
        assert bool((met if where == "all" else met[..., 5:6])[:, sees[:, at]].all())
        assert not o[b, :, ~sees.any(1)].any() and not lse[b].isnan().any()
        return
    assert want[0].isnan().any() or value == -math.inf or not sees[:, at].any()
    nf.agree(o[b], lse[b], want[0], want[1], want[2], vv, dtype)
    if B > 1:
        assert bool(o[:b].isfinite().all()) and not lse[:b].isnan().any()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("how", [False, True, "bottom-right", "bool", "add"])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(dt, D, how, shape):
    """A row of q, a key of the first and one of a later tile, a value."""
    S = SHAPES[shape][4]
    for value, where in nf.POISON:
        run(shape, D, DTYPES[dt], how, "q", 31, value, where)
        for at in (17, 22, S - 20 - S % 16):  # (17: a column whose exponentials D = 64 takes on the FMA pipe)
            run(shape, D, DTYPES[dt], how, "k", at, value, where)
            run(shape, D, DTYPES[dt], how, "v", at, value, where)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True, "bottom-right"])
@pytest.mark.parametrize("lens", [(9, 30, 17, 5) * 20, (60, 33, 64) * 12, (300, 1, 129, 40)], ids=["32", "64", "long"])
def test_packed(dt, D, causal, lens):
    """Short sequences whose heads share tiles, and long ones; the other sequences stay finite."""
    from tinytorch_b200 import op
    Hq, Hkv, dtype = 8, 2, DTYPES[dt]
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    T, n = int(cu[-1]), 2
    first, end = int(cu[n]), int(cu[n + 1])
    for name, at in (("q", end - 2), ("k", first + 1), ("k", first + 4)):
        for value, where in nf.POISON:
            x = {m: randn((T, h, D), dtype, i) for i, (m, h) in enumerate((("q", Hq), ("k", Hkv), ("v", Hkv)))}
            x["q"][..., 5] = x["q"][..., 5].abs() + 0.1
            x[name] = nf.poison(x[name], (at, 0), value, where)
            q, k, v = x.values()
            o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, causal)
            rows = slice(first, end)
            kk, vv = (t[rows].double().transpose(0, 1).repeat_interleave(Hq // Hkv, 0) for t in (k, v))
            want = nf.attention(q[rows].double().transpose(0, 1), kk, vv, 1 / math.sqrt(D), ref.visible(end - first, end - first, causal, "cuda"))
            nf.agree(o[rows].transpose(0, 1), lse[:, rows], want[0], want[1], want[2], vv, dtype)
            other = torch.ones(T, dtype=torch.bool, device="cuda")
            other[rows] = False
            assert bool(o[other].isfinite().all()) and bool(lse[:, other].isfinite().all())


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("how", [True, "bottom-right", "bool"])
def test_gradients_of_a_row_that_is_not_finite(dt, D, how):
    """Where the formula's gradients are NaN, the kernels' are."""
    from tinytorch_b200 import function
    B, H, L, S = 24, 16, 200, 190
    dtype = DTYPES[dt]
    q, k, v = (randn((B, H, n, D), dtype, i) for i, n in enumerate((L, S, S)))
    k = nf.poison(k, (B - 1, 3, 22), math.nan, "all")
    sees = torch.ones(L, S, dtype=torch.bool, device="cuda").tril(5) if how == "bool" else ref.visible(L, S, how, "cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = function.sdpAttention(*leaves, **(dict(attnMask=sees) if how == "bool" else dict(isCausal=how)))
    dq, dk, dv = torch.autograd.grad(o, leaves, randn(o.shape, dtype, 9))
    rows = sees[:, 22]            # they see the key: all their probabilities are NaN
    keys = sees[rows].any(0)      # the keys that they see
    assert bool(dq[-1, 3, rows].isnan().all()) and bool(dk[-1, 3, keys].isnan().all()) and bool(dv[-1, 3, keys].isnan().all())
    other = torch.ones(B, H, dtype=torch.bool, device="cuda")
    other[-1, 3] = False
    assert all(bool(g[other].isfinite().all()) for g in (dq, dk, dv))
