"""GPU: the differentiable call over packed sequences says, in both of its passes, that offsets do not fit the rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BAD = [(0, 50, 40, 90), (-1, 20, 40, 90), (0, 20, 40, 91)]  # they fall, begin before the rows, end behind them


def operands(rows=90):
    g = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(rows, h, 64, generator=g, device="cuda").bfloat16().requires_grad_() for h in (8, 2, 2)]


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("offsets", [(0, 20, 40, 90), *BAD])
def test_status_of_both_passes(offsets, python):
    """python: the autograd function that a trace and torch's transforms get."""
    from tinytorch_b200 import function, op
    x = operands()
    cu = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = 16 if offsets in BAD else 0
    if python:
        o = function.FuncSDPAttentionPacked.apply(*x, cu, None, True, op.default_scale(64), status)
    else:
        o = function.sdpAttentionPacked(*x, cu, isCausal=True, status=status)
    assert int(status) == want and bool(o.any()) == (want == 0)
    status.zero_()  # (as a training step does when it has looked at it)
    grads = torch.autograd.grad(o, x, torch.ones_like(o))
    assert int(status) == want and all(bool(g.any()) == (want == 0) for g in grads)


def test_status_of_the_backward_operator():
    from tinytorch_b200 import op
    x = [t.detach() for t in operands()]
    good, bad = (torch.tensor(c, dtype=torch.int32, device="cuda") for c in ((0, 20, 40, 90), BAD[0]))
    o, lse = op.sdpAttentionPackedFwd(*x, good, True)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    first = op.sdpAttentionPackedBwd(o, *x, o, lse, good, True, status=status)
    assert int(status) == 0 and torch.equal(first[1], op.sdpAttentionPackedBwd(o, *x, o, lse, good, True)[1])
    assert not any(g.any() for g in op.sdpAttentionPackedBwd(o, *x, o, lse, bad, True, status=status)) and int(status) == 16


def test_status_of_a_replayed_step():
    """Forward and backward in a graph: the word is the caller's, looked at and cleared between replays."""
    from tinytorch_b200 import function
    x = operands()
    cu, status = torch.tensor((0, 20, 40, 90), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")

    def step():
        # (not the caller's tensor: a backward keeps its offsets from being changed between the passes)
        return torch.autograd.grad(function.sdpAttentionPacked(*x, cu.clone(), isCausal=True, status=status).float().square().sum(), x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for offsets, want in (((0, 20, 40, 90), 0), (BAD[0], 16), ((0, 1, 1, 30), 0)):
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        status.zero_()
        graph.replay()
        assert int(status) == want and all(bool(g.any()) == (want == 0) for g in out)
