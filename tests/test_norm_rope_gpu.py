"""GPU: the norm of queries and keys with the rotation, and its gradients, against a 64-bit form."""
import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def randn(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def positions(shape, top, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, top, shape, generator=g, device="cuda", dtype=torch.int32)


def check(q, k, qw, kw, cos, sin, pos, eps=1e-6, interleaved=False, sections=None, seed=50):
    """Forward, and gradients through autograd for outputs' gradients of the inputs' layout."""
    from tinytorch_b200 import fused
    leaves = [None if x is None else x.detach().requires_grad_() for x in (q, k, qw, kw)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = fused.qkNormRope(*leaves, cos, sin, pos, eps=eps, interleaved=interleaved, sections=sections, status=status)
    gs = [randn(x.shape, x.dtype, seed + i) for i, x in enumerate((q, k))]
    want = [x for x in leaves if x is not None]
    grads = dict(zip(map(id, want), torch.autograd.grad(out, want, gs)))
    cs = None if cos is None else ref.angles(cos, sin, pos, sections, q.dim())
    for i, (x, w, name) in enumerate(((q, qw, "q"), (k, kw, "k"))):
        w64 = None if w is None else w.double()
        ref.norm_rope_check(out[i], x.double(), w64, cs, eps, interleaved, x.dtype, name)
        ref.norm_rope_grads_check(grads[id(leaves[i])], None if w is None else grads[id(leaves[2 + i])], gs[i].double(), x.double(), w64, cs, eps,
                                  interleaved, x.dtype, name)
    return out, int(status)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 1, 1), (1, 32, 8), (3, 5, 5), (17, 28, 4), (300, 8, 1), (2000, 6, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_packed_rows(dt, D, T, Hq, Hkv, interleaved):
    from tinytorch_b200 import op
    dtype = DTYPES[dt]
    qkv = randn((T, Hq + 2 * Hkv, D), dtype, 1)
    cos, sin = op.ropeTables(500, D)
    check(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], 1 + 0.3 * randn((D,), dtype, 2), 1 + 0.3 * randn((D,), dtype, 3), cos, sin, positions((T,), 500, 4),
          interleaved=interleaved)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("by_token", [True, False])
@pytest.mark.parametrize("axes,sections", [(1, None), (2, (0.25, 0.75)), (3, (0.25, 0.375, 0.375)), (3, (0.3, 0.4, 0.3)), (4, (0.0, 0.5, 0.25, 0.25)), (1, (1.0,))])
def test_batches_and_axes(dt, D, by_token, axes, sections):
    """[B, H, S, D] in both orders; sections that are and are not whole vectors of pairs."""
    from tinytorch_b200 import op
    dtype, B, S, Hq, Hkv = DTYPES[dt], 2, 37, 6, 2
    if sections:
        n = [int(s * D / 2) for s in sections]
        n[-1] += D // 2 - sum(n)
        sections = n
    shape = lambda H: (B, S, H, D) if by_token else (B, H, S, D)
    q, k = (randn(shape(H), dtype, H).transpose(1, 2) if by_token else randn(shape(H), dtype, H) for H in (Hq, Hkv))
    cos, sin = op.ropeTables(100, D)
    for batched in (True, False):
        pos = positions(((axes,) if sections else ()) + ((B,) if batched else ()) + (S,), 100, 5)
        out, status = check(q, k, randn((D,), dtype, 6), randn((D,), dtype, 7), cos, sin, pos, sections=sections)
        assert status == 0 and out[0].stride() == q.stride() and out[1].stride() == k.stride()


@pytest.mark.parametrize("which", ["norm", "rotation", "q only", "nothing"])
def test_parts_of_it(which):
    from tinytorch_b200 import op
    q, k = randn((40, 4, 64), torch.float16, 1), randn((40, 2, 64), torch.float16, 2)
    w = randn((64,), torch.float16, 3)
    cos, sin = op.ropeTables(100, 64)
    rope = (cos, sin, positions((40,), 100, 4)) if which in ("rotation", "q only") else (None, None, None)
    out, _ = check(q, k, w if which in ("norm", "q only") else None, w if which == "norm" else None, *rope)
    if which == "nothing":
        assert torch.equal(out[0], q) and torch.equal(out[1], k)


def test_positions_outside_the_tables():
    from tinytorch_b200 import op
    q, k = randn((6, 4, 128), torch.bfloat16, 1), randn((6, 2, 128), torch.bfloat16, 2)
    w = randn((128,), torch.bfloat16, 3)
    cos, sin = op.ropeTables(10, 128)
    pos = torch.tensor([0, 9, 10, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    _, status = check(q, k, w, w, cos, sin, pos)
    assert status == 8
    _, status = check(q, k, w, w, cos, sin, torch.stack([pos, pos.clamp(0, 9)]), sections=(20, 44))
    assert status == 8
    assert check(q, k, w, w, cos, sin, pos.clamp(0, 9))[1] == 0


@pytest.mark.parametrize("std,eps", [(1e-4, 1e-6), (1e-4, 0.0), (200.0, 1e-5), (0.0, 1e-6)])
def test_sizes_of_values(std, eps):
    from tinytorch_b200 import op
    for dtype in (torch.bfloat16, torch.float32):
        q, k = randn((50, 5, 64), dtype, 1, std), randn((50, 3, 64), dtype, 2, std)
        w = randn((64,), dtype, 3)
        cos, sin = op.ropeTables(100, 64)
        check(q, k, w, w, cos, sin, positions((50,), 100, 4), eps=eps)


def test_infinities_stay_in_their_row():
    from tinytorch_b200 import fused, op
    q, k = randn((9, 4, 64), torch.bfloat16, 1), randn((9, 2, 64), torch.bfloat16, 2)
    w, (cos, sin), pos = randn((64,), torch.bfloat16, 3), op.ropeTables(20, 64), positions((9,), 20, 4)
    clean = fused.qkNormRope(q, k, w, w, cos, sin, pos)
    q2 = q.clone()
    q2[4, 1, 7] = float("inf")
    dirty = fused.qkNormRope(q2, k, w, w, cos, sin, pos)
    same = torch.ones(9, 4, dtype=torch.bool, device="cuda")
    same[4, 1] = False
    assert torch.equal(clean[0][same], dirty[0][same]) and torch.equal(clean[1], dirty[1]) and dirty[0][4, 1].isnan().any()


def test_no_rows():
    from tinytorch_b200 import fused, op
    w = randn((64,), torch.bfloat16, 1).requires_grad_()
    cos, sin = op.ropeTables(20, 64)
    for q, k, pos in ((randn((0, 4, 64), torch.bfloat16, 1), randn((0, 2, 64), torch.bfloat16, 2), positions((0,), 9, 3)),
                      (randn((2, 4, 0, 64), torch.bfloat16, 1), randn((2, 2, 0, 64), torch.bfloat16, 2), positions((2, 0), 9, 3))):
        out = fused.qkNormRope(q, k, w, w, cos, sin, pos)
        assert out[0].shape == q.shape and out[1].shape == k.shape
        assert not torch.autograd.grad(out, w, [x.detach() for x in out])[0].any()


def test_one_output_used_and_odd_gradients():
    """Only k' goes on; gradients at an odd offset, or of one value expanded."""
    from tinytorch_b200 import fused, op
    q, k = (randn((30, h, 64), torch.float16, h).requires_grad_() for h in (4, 2))
    w, (cos, sin), pos = randn((64,), torch.float16, 3).requires_grad_(), op.ropeTables(50, 64), positions((30,), 50, 4)
    cs = ref.angles(cos, sin, pos, None, 3)

    def grads(g):
        return torch.autograd.grad(fused.qkNormRope(q, k, w, w, cos, sin, pos)[1], (q, k, w), g)
    odd = randn((30 * 2 * 64 + 1,), torch.float16, 8)[1:].view(30, 2, 64)
    for g in (odd, torch.ones((), dtype=torch.float16, device="cuda").expand(30, 2, 64), randn((30, 2, 128), torch.float16, 9)[..., ::2]):
        dq, dk, dw = grads(g)
        assert not dq.any()
        ref.norm_rope_grads_check(dk, dw, g.double(), k.detach().double(), w.detach().double(), cs, 1e-6, False, torch.float16, "k")


def test_gradients_against_differences():
    from tinytorch_b200 import fused, op
    x = [randn((20, h, 64), torch.float32, 10 + h) for h in (3, 2)] + [randn((64,), torch.float32, 20 + i) for i in range(2)]
    cos, sin = op.ropeTables(90, 64)
    pos = positions((20,), 90, 4)
    g = [randn(t.shape, torch.float32, 30 + i) for i, t in enumerate(x[:2])]
    leaves = [t.clone().requires_grad_() for t in x]
    grads = torch.autograd.grad(fused.qkNormRope(*leaves, cos, sin, pos, eps=1e-5), leaves, g)
    cs = ref.angles(cos, sin, pos, None, 3)

    def loss(q, k, qw, kw):
        return sum((ref.norm_rope(a, w, cs, 1e-5, False) * t.double()).sum() for a, w, t in ((q, qw, g[0]), (k, kw, g[1]))).item()
    x = [t.double() for t in x]
    for i in range(4):
        d = randn(x[i].shape, torch.float64, 40 + i)
        plus, minus = ([t + s * 1e-5 * d if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        want = (loss(*plus) - loss(*minus)) / 2e-5
        got = (grads[i].double() * d).sum().item()
        # 64 steps of 2^-24 of every term, and the difference's own error, (1e-5)^2 of a third derivative of the loss
        assert abs(got - want) <= 64 * 2.0 ** -24 * (grads[i].double() * d).abs().sum().item() + 1e-6 * abs(want) + 1e-6


def test_sums_repeat_and_graphs_follow():
    """The weights' gradients are the same to the bit every time, from another stream and from a captured graph with other positions."""
    from tinytorch_b200 import fused, op
    q, k = (randn((3000, h, 128), torch.bfloat16, h).requires_grad_() for h in (8, 2))
    w = [randn((128,), torch.bfloat16, 3 + i).requires_grad_() for i in range(2)]
    cos, sin = op.ropeTables(800, 128)
    pos = positions((3000,), 800, 4)
    gs = [randn(x.shape, torch.bfloat16, 9) for x in (q, k)]

    def step(pos):
        out = fused.qkNormRope(q, k, *w, cos, sin, pos)
        grads = torch.autograd.grad(out, (q, k, *w), gs)
        return (*(x.detach() for x in out), *grads)  # (torch captures no backward of leaves whose eager graph is still held)
    first = step(pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(pos)
        held = torch.zeros_like(pos)
        step(held)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            replayed = step(held)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    held.copy_(pos)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, replayed))


def test_python_function_has_the_same_results():
    from tinytorch_b200 import fused, op
    q, k = (randn((30, h, 64), torch.bfloat16, h).requires_grad_() for h in (4, 2))
    w = [randn((64,), torch.bfloat16, 3 + i).requires_grad_() for i in range(2)]
    cos, sin = op.ropeTables(80, 64)
    pos = positions((2, 30), 80, 4)
    gs = [randn(x.shape, torch.bfloat16, 9) for x in (q, k)]
    a = fused.qkNormRope(q, k, *w, cos, sin, pos, sections=(12, 20))
    b = fused.FuncQkNormRope.apply(q, k, *w, cos, sin, pos, 1e-6, False, (12, 20), None)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(a, (q, k, *w), gs), torch.autograd.grad(b, (q, k, *w), gs)))


@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 128)])
def test_operands_that_end_where_their_memory_does(dt, D):
    from tinytorch_b200 import fused, op

    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, gq, gk, wq, wk = (torch.randn(*s, generator=g, device="cuda").to(dt) for s in ((37, 5, D), (37, 2, D), (37, 5, D), (37, 2, D), (D,), (D,)))
    cos, sin = op.ropeTables(100, D)
    pos = torch.arange(37, dtype=torch.int32, device="cuda") + 63  # the last row of the tables among them

    def run(q, k, wq, wk, cos, sin, pos, gq, gk):
        leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk)]
        out = fused.qkNormRope(*leaves, cos, sin, pos)
        return [*out, *torch.autograd.grad(out, leaves, (gq, gk))]

    want = run(q, k, wq, wk, cos, sin, pos, gq, gk)
    got = run(*(ref.at_the_end(x) for x in (q, k, wq, wk, cos, sin, pos, gq, gk)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_far_away():
    """More than 2^31 elements: the last rows are those of a call of their own."""
    from tinytorch_b200 import fused, op

    T, D = 540_000, 128
    q, k = torch.zeros(T, 32, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, 2, D, dtype=torch.bfloat16, device="cuda")
    assert q.numel() > 2 ** 31
    q[-9:], k[-9:] = randn((9, 32, D), torch.bfloat16, 1), randn((9, 2, D), torch.bfloat16, 2)
    w = randn((D,), torch.bfloat16, 3)
    cos, sin = op.ropeTables(64, D)
    pos = positions((T,), 64, 4)

    def run(q, k, pos):
        leaves = [q.detach().requires_grad_(), k.detach().requires_grad_(), w.clone().requires_grad_(), w.clone().requires_grad_()]
        out = fused.qkNormRope(*leaves, cos, sin, pos)
        return [x.detach() for x in out], torch.autograd.grad(out, leaves, (q.detach(), k.detach()))

    out, grads = run(q, k, pos)
    want, back = run(q[-9:].clone(), k[-9:].clone(), pos[-9:])
    assert all(torch.equal(x[-9:], y) for x, y in zip(out + list(grads[:2]), want + list(back[:2])))
    # (the other rows' outputs and their gradients are zeros: so are their shares of the weights' gradients)
    assert not out[0][:-9].any() and not grads[0][:-9].any()
    for x, y in zip(grads[2:], back[2:]):
        assert (x.float() - y.float()).abs().max() <= 2 ** -7 * y.float().abs().max()
