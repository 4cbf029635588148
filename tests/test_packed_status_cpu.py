"""CPU: a status word of another kind is refused by both passes over packed sequences (fake CUDA tensors, as in test_lm_arguments_cpu.py)."""
import os

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from conftest import ROOT
from tinytorch_b200 import function, op


@pytest.mark.parametrize("status", [dict(dtype=torch.int64), dict(n=0), dict(device="cpu"), dict(dtype=torch.float32)])
def test_status_is_checked(status):
    if not os.path.exists(os.path.join(ROOT, "tinytorch_b200", "lib", "_native.so")):
        from tinytorch_b200.build import build, build_native
        build()
        build_native()
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16, device="cuda"):
            return torch.empty(shape, dtype=dtype, device=device)
        word = t(status.get("n", 1), dtype=status.get("dtype", torch.int32), device=status.get("device", "cuda"))
        q, k, cu = t(40, 8, 64), t(40, 2, 64), t(3, dtype=torch.int32)
        with pytest.raises(ValueError, match="status"):
            function.sdpAttentionPacked(q, k, k, cu, status=word)
        with pytest.raises(ValueError, match="status"):
            op.sdpAttentionPackedBwd(q, q, k, k, q, t(8, 40, dtype=torch.float32), cu, status=word)
