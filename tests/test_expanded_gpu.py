"""GPU: operands and gradients of which several dimensions share memory give what their dense copies give."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def positions(n, top, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, top, (n,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_gradient_of_one_row(dtype, D):
    """The loss is a product with the sum over all rows: the gradient of O is one row, expanded; and at an odd offset of a larger one."""
    from tinytorch_b200 import function
    x = [randn((2, h, 70, D), dtype, h) for h in (8, 4, 4)]
    row, odd = randn((D,), dtype, 9), randn((2 * 8 * 70 * D + 1,), dtype, 10)[1:].view(2, 8, 70, D)

    def grads(g):
        leaves = [y.clone().requires_grad_() for y in x]
        return torch.autograd.grad(function.sdpAttention(*leaves, isCausal=True), leaves, g)
    for g in (row.expand(2, 8, 70, D), row.view(1, 1, 1, D).expand(2, 1, 70, D).expand(2, 8, 70, D), x[0][:, :, :1].expand(2, 8, 70, D), odd):
        # (70 keys are one tile: every element of dQ has one term, so the order of sums does not show)
        assert all(torch.equal(a, b) for a, b in zip(grads(g), grads(g.contiguous().clone())))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("packed", [False, True])
def test_norm_and_rotation(dtype, packed):
    """q and k of any strides but the last: one row, rows of one memory, an odd offset."""
    from tinytorch_b200 import fused, op
    D, S = 64, 30
    shapes = [(S, h, D) if packed else (2, h, S, D) for h in (6, 2)]
    w, (cos, sin), pos = [randn((D,), dtype, i) for i in (1, 2)], op.ropeTables(90, D), positions(S, 90, 3)

    def odd(shape, seed):
        n = torch.Size(shape).numel()
        return randn((n + 1,), dtype, seed)[1:].view(shape)

    def run(q, k):
        leaves = [y.detach().requires_grad_() for y in (q, k, *w)]
        out = fused.qkNormRope(*leaves, cos, sin, pos)
        return (*out, *torch.autograd.grad(out, leaves, [randn(y.shape, dtype, 20 + i) for i, y in enumerate(out)]))
    row = randn((D,), dtype, 4)
    for q, k in (([row.expand(s) for s in shapes]), ([randn(s, dtype, 5).narrow(0 if packed else 2, 0, 1).expand(s) for s in shapes]),
                 ([odd(s, 6) for s in shapes]), (row.expand(shapes[0]), randn(shapes[1], dtype, 7))):
        got, want = run(q, k), run(q.contiguous().clone(), k.contiguous().clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_query_for_all_heads_and_sequences(dtype):
    """A single row is no row that is shared: every stride may be 0."""
    from tinytorch_b200 import op
    B, Hq, Hkv, cap, D = 3, 8, 2, 200, 64
    q = randn((D,), dtype, 1).expand(B, Hq, 1, D)
    kd, vd = (randn((D,), dtype, i).expand(B, Hkv, 1, D) for i in (2, 3))
    kc, vc = (randn((B, Hkv, cap, D), dtype, i) for i in (4, 5))
    lens = torch.tensor([200, 17, 130], dtype=torch.int32, device="cuda")
    dense = [x.contiguous().clone() for x in (q, kd, vd)]
    assert torch.equal(op.sdpAttentionDecode(q, kc, vc, lens)[0], op.sdpAttentionDecode(dense[0], kc, vc, lens)[0])
    assert torch.equal(op.sdpAttentionTree(q, kd, vd, kc, vc, lens)[0], op.sdpAttentionTree(*dense, kc, vc, lens)[0])
    assert torch.equal(op.sdpAttentionFwd(q, kc, vc, kvLens=lens)[0], op.sdpAttentionFwd(dense[0], kc, vc, kvLens=lens)[0])
    caches = [[x.clone() for x in (kc, vc)] for _ in range(2)]
    path, counts, room = torch.zeros(B, 1, dtype=torch.int32, device="cuda"), torch.ones(B, dtype=torch.int32, device="cuda"), lens.clamp(max=cap - 1)
    for (k, v), (a, b) in zip(caches, ((kd, vd), dense[1:])):
        op.cacheAccept(a, b, k, v, room, path, counts)
    assert all(torch.equal(a, b) for a, b in zip(*caches))
    assert torch.equal(caches[0][0][0, :, cap - 1], kd[0, :, 0])
