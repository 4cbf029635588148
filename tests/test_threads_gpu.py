"""GPU: calls from threads that have made no CUDA call before."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["forward", "decode", "linear"])
def test_first_call_of_a_thread(which):
    from tinytorch_b200 import fused, op
    q, k, v = (torch.randn(2, h, 300, 128, device="cuda").to(torch.bfloat16) for h in (8, 2, 2))
    q1, x, w = q[:, :, :1].contiguous(), torch.randn(64, 512, device="cuda").to(torch.bfloat16), torch.randn(256, 512, device="cuda").to(torch.bfloat16)
    call = {"forward": lambda: op.sdpAttentionFwd(q, k, v, isCausal=True)[0], "decode": lambda: op.sdpAttentionDecode(q1, k, v)[0],
            "linear": lambda: fused.linear(x, w)}[which]
    want = call()  # (and the blocks that the second call's results and scratch come from are in the allocator's cache)
    torch.cuda.synchronize()
    out = []

    def run():
        try:
            out.append(call())
        except Exception as e:  # (shown below, in the test's thread)
            out.append(e)
    t = threading.Thread(target=run)
    again = call()
    del again
    t.start()
    t.join()
    assert isinstance(out[0], torch.Tensor), out[0]
    torch.cuda.synchronize()
    assert torch.equal(out[0], want)
