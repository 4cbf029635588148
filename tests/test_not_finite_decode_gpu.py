"""GPU: NaN and infinities in a decode step's query and in the valid rows of its cache come out where the 64-bit form has them, however the cache is divided."""
import math

import pytest
import torch

import not_finite as nf

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (4, 4), (16, 2), (3, 1)])
@pytest.mark.parametrize("cap,lens", [(5000, (60, 4901)), (200, (200, 150) + (30,) * 150), (64, (1, 40))], ids=["divided", "whole", "short"])
@pytest.mark.parametrize("append", [False, True])
def test_decode(dt, D, Hq, Hkv, cap, lens, append):
    from tinytorch_b200 import op
    dtype, B, group, n = DTYPES[dt], len(lens), Hq // Hkv, lens[1]
    x = {m: randn((B, h, r, D), dtype, i) for i, (m, h, r) in enumerate((("q", Hq, 1), ("k", Hkv, cap), ("v", Hkv, cap), ("kn", Hkv, 1), ("vn", Hkv, 1)))}
    x["q"][..., 5] = x["q"][..., 5].abs() + 0.1
    kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for name, at in (("q", 0), ("k", 3), ("k", n - 1), ("k", n // 2), ("v", n // 2), ("v", 0)) + ((("kn", 0), ("vn", 0)) if append else ()):
        for value, where in nf.POISON:
            y = {m: t.clone() for m, t in x.items()}
            y[name] = nf.poison(x[name], (1, 0, at), value, where)
            k, v = y["k"][1, :, :n], y["v"][1, :, :n]
            if append:
                k, v = torch.cat((k, y["kn"][1]), 1), torch.cat((v, y["vn"][1]), 1)
                o, lse, _ = op.sdpAttentionDecodeAppend(y["q"], y["kn"], y["vn"], y["k"], y["v"], kv_lens.clamp(max=cap - 1) if n < cap else kv_lens, needLse=True)
            else:
                o, lse = op.sdpAttentionDecode(y["q"], y["k"], y["v"], kv_lens, needLse=True)
            k, v = (t.double().repeat_interleave(group, 0) for t in (k, v))
            want = nf.attention(y["q"][1].double(), k, v, 1 / math.sqrt(D), torch.ones(1, k.shape[1], dtype=torch.bool, device="cuda"))
            if name in ("v", "vn"):
                assert torch.equal(o[1].isfinite(), want[0].isfinite()) and not want[0].isfinite().all()
                assert bool(lse[1].isfinite().all())
            else:
                assert want[0].isnan().any() or value == -math.inf
                nf.agree(o[1], lse[1][:, None], want[0], want[1], want[2], v, dtype)
            other = [b for b in range(B) if b != 1]
            assert bool(o[other].isfinite().all()) and bool(lse[other].isfinite().all())
