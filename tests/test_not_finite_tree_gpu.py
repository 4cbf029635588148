"""GPU: NaN and infinities among the valid rows of a cache, drafts and queries of a tree come out where the 64-bit form has them, wherever the
line of tiles is cut."""
import math

import pytest
import torch

import not_finite as nf

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# q heads, kv heads, drafts, capacity, lengths; the second sequence holds what is not finite
CASES = {
    "one walk in pieces, 4 copies": (8, 2, 5, 6000, (10, 5900)),
    "2 copies": (8, 2, 16, 6000, (3000, 5900)),
    "1 copy": (16, 2, 16, 6000, (3000, 5900)),
    "whole walks": (8, 2, 5, 300, (290, 280) + (300,) * 200),
    "whole walks, 1 copy": (16, 2, 16, 300, (290, 280) + (300,) * 200),
    "short": (2, 2, 9, 90, (90, 70)),
}


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", CASES)
def test_trees(dt, D, case):
    from tinytorch_b200 import op
    Hq, Hkv, T, cap, lens = CASES[case]
    dtype, B, n, group = DTYPES[dt], len(lens), lens[1], Hq // Hkv
    x = {m: randn((B, h, r, D), dtype, i) for i, (m, h, r) in enumerate((("q", Hq, T), ("kd", Hkv, T), ("vd", Hkv, T), ("kc", Hkv, cap), ("vc", Hkv, cap)))}
    x["q"][..., 5] = x["q"][..., 5].abs() + 0.1
    kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    chain = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    for name, at in (("q", T - 1), ("kc", 3), ("kc", n - 1), ("kc", n // 2), ("vc", n // 2), ("vc", 0), ("kd", 1)):
        for value, where in nf.POISON:
            y = dict(x)
            y[name] = nf.poison(x[name], (1, 0, at), value, where)
            o, lse = op.sdpAttentionTree(y["q"], y["kd"], y["vd"], y["kc"], y["vc"], kv_lens, chain, needLse=True)
            k, v = (torch.cat((c[1, :, :n], d[1]), 1).double().repeat_interleave(group, 0) for c, d in ((y["kc"], y["kd"]), (y["vc"], y["vd"])))
            sees = torch.cat((torch.ones(T, n, dtype=torch.bool, device="cuda"), chain), 1)
            want = nf.attention(y["q"][1].double(), k, v, 1 / math.sqrt(D), sees)
            if name == "vc":  # (a probability that is rounded to 0 times an infinity is NaN)
                assert torch.equal(o[1].isfinite(), want[0].isfinite()) and not want[0].isfinite().all()
                if value != value:
                    assert torch.equal(o[1].isnan(), want[0].isnan())
                assert bool(lse[1].isfinite().all())
            else:
                assert want[0].isnan().any() or value == -math.inf
                nf.agree(o[1], lse[1], want[0], want[1], want[2], v, dtype)
            other = [b for b in range(B) if b != 1]
            assert bool(o[other].isfinite().all()) and bool(lse[other].isfinite().all())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_without_keys_beside_one_that_is_not_finite(dt, D):
    """Drafts that see nothing give O = 0 and LSE = -inf, also where a query of theirs is NaN: it meets no key."""
    from tinytorch_b200 import op
    dtype, B, Hq, Hkv, T = DTYPES[dt], 3, 8, 2, 7
    q = randn((B, Hq, T, D), dtype, 1)
    q[1, :, 2] = math.nan
    kd, vd, kc, vc = (randn((B, Hkv, n, D), dtype, i) for i, n in ((2, T), (3, T), (4, 100), (5, 100)))
    lens = torch.tensor([50, 0, 0], dtype=torch.int32, device="cuda")
    mask = torch.eye(T, dtype=torch.bool, device="cuda").repeat(B, 1, 1)
    mask[1, 2] = mask[2, 4] = False
    o, lse = op.sdpAttentionTree(q, kd, vd, kc, vc, lens, mask, needLse=True)
    for b, t in ((1, 2), (2, 4)):
        assert not o[b, :, t].any() and bool((lse[b, :, t] == -math.inf).all())
    mask[1, 2, 2] = True
    o, lse = op.sdpAttentionTree(q, kd, vd, kc, vc, lens, mask, needLse=True)
    assert bool(o[1, :, 2].isnan().all()) and bool(lse[1, :, 2].isnan().all())
    assert int(o.isnan().sum()) == Hq * D and int(lse.isnan().sum()) == Hq
