"""GPU: attention over packed sequences against a 64-bit form, a sequence at a time."""
import math

import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def offsets(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()


def make(rows, H, D, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, H, D, generator=g, device="cuda") * std).to(dtype)


def check(got, q, k, v, lens, causal, lens_k=None, scale=None, g=None, tail=0):
    """got: o, lse, and with g: dq, dk, dv"""
    o, lse = got[:2]
    D, group, dt = q.shape[2], q.shape[1] // k.shape[1], q.dtype
    scale = 1 / math.sqrt(D) if scale is None else scale
    a = b = 0
    for n, m in zip(lens, lens_k or lens):
        sees = ref.visible(n, m, causal, q.device)
        for h in range(k.shape[1]):
            hs = slice(h * group, (h + 1) * group)
            qh, kh, vh = q[a:a + n, hs].double().transpose(0, 1), k[b:b + m, h].double(), v[b:b + m, h].double()
            wo, wl, p = ref.attention(qh, kh, vh, scale, sees)
            what = "rows %d..%d head %d" % (a, a + n, h)
            ref.within(o[a:a + n, hs].transpose(0, 1), wo, ref.attention_bound(p, vh, wo, dt), what + " o")
            if lse is not None:
                gl = lse[hs, a:a + n]
                assert torch.equal(gl == -math.inf, wl == -math.inf)
                some = wl > -math.inf
                assert n == 0 or not some.any() or (gl.double() - wl)[some].abs().max() <= ref.SLOP
            if g is not None:
                gh = g[a:a + n, hs].double().transpose(0, 1)
                wq, wk, wv = ref.attention_grads(qh, kh, vh, wo, gh, p, scale, dt)
                ref.within(got[2][a:a + n, hs].transpose(0, 1), *wq, what + " dq")
                ref.within(got[3][b:b + m, h], *wk, what + " dk")
                ref.within(got[4][b:b + m, h], *wv, what + " dv")
        a, b = a + n, b + m
    # rows of no sequence
    assert not o[a:].any() and (lse is None or bool((lse[:, a:] == -math.inf).all()))
    if g is not None:
        assert not got[2][a:].any() and not got[3][b:].any() and not got[4][b:].any()


LENS = [(1,), (128,), (129, 1, 300), (0, 5, 0, 64, 200, 0), tuple(i % 7 + 1 for i in range(45)), (700, 33, 512), (256, 257, 255)]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt,Hq,Hkv", [("bf16", 4, 4), ("f16", 8, 2), ("bf16", 3, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_forward_and_gradients(lens, D, dt, Hq, Hkv, causal):
    from tinytorch_b200 import op
    T, dtype = sum(lens) + 3, DTYPES[dt]
    q, k, v, g = (make(T, h, D, dtype, 10 + i) for i, h in enumerate((Hq, Hkv, Hkv, Hq)))
    cu, status = offsets(lens), torch.zeros(1, dtype=torch.int32, device="cuda")
    o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, causal, status=status)
    grads = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, causal)
    check((o, lse, *grads), q, k, v, lens, causal, g=g)
    assert int(status) == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,Hq,Hkv", [((2000,), 4, 1), ((1500, 3, 700), 8, 1), ((5, 1100, 0, 900), 6, 2)])
def test_divided_walks(D, causal, lens, Hq, Hkv):
    """Few key tiles: their walks are divided among the CTAs; dK and dV are the same to the bit every time."""
    from tinytorch_b200 import op
    T = sum(lens) + 2
    q, k, v, g = (make(T, h, D, torch.bfloat16, 30 + i) for i, h in enumerate((Hq, Hkv, Hkv, Hq)))
    cu = offsets(lens)
    o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, causal)
    grads = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, causal)
    check((o, lse, *grads), q, k, v, lens, causal, g=g)
    again = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, causal)
    assert torch.equal(grads[1], again[1]) and torch.equal(grads[2], again[2])
    for i in (1, 2):
        one = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, causal, needs=tuple(j == i for j in range(3)))
        assert torch.equal(one[i], grads[i])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", ["bottom-right", True, False])
@pytest.mark.parametrize("lens,lens_k", [((5, 130, 1), (700, 130, 1)), ((200, 40, 7), (60, 0, 300)), ((0, 300, 1), (9, 299, 1500))])
def test_keys_with_lengths_of_their_own(D, causal, lens, lens_k):
    """Chunks at the end of longer keys; with more queries than keys some see none; keys without queries."""
    from tinytorch_b200 import op
    q, g = make(sum(lens), 6, D, torch.bfloat16, 1), make(sum(lens), 6, D, torch.bfloat16, 2)
    k, v = make(sum(lens_k) + 5, 2, D, torch.bfloat16, 3), make(sum(lens_k) + 5, 2, D, torch.bfloat16, 4)
    cu, cuk = offsets(lens), offsets(lens_k)
    o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, causal, cuSeqlensK=cuk, scale=0.2)
    grads = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, causal, 0.2, cuk)
    check((o, lse, *grads), q, k, v, lens, causal, lens_k, 0.2, g)


def test_a_sequence_alone_and_among_others_is_the_same():
    from tinytorch_b200 import op
    lens = (300, 128, 77, 1000)
    q, k, v = (make(sum(lens), h, 128, torch.bfloat16, h) for h in (8, 2, 2))
    o, lse = op.sdpAttentionPackedFwd(q, k, v, offsets(lens), True)
    at = 0
    for n in lens:
        rows = slice(at, at + n)
        one, one_lse = op.sdpAttentionPackedFwd(q[rows], k[rows], v[rows], offsets((n,)), True)
        assert torch.equal(one, o[rows]) and torch.equal(one_lse, lse[:, rows])
        at += n


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("poison", [math.inf, math.nan])
def test_neighbours_are_not_touched(D, poison):
    """Infinities in the sequences before and behind, and in rows of no sequence, stay there."""
    from tinytorch_b200 import op
    lens = (70, 200, 90)
    x = [make(sum(lens) + 40, h, D, torch.bfloat16, 20 + i) for i, h in enumerate((4, 2, 2, 4))]
    cu = offsets(lens)

    def run(q, k, v, g):
        o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, True)
        return (o, lse.t(), *op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, True))
    clean = run(*x)
    for t in x:
        t[:70] = poison
        t[270:] = poison
    dirty = run(*x)
    for name, a, b in zip(("o", "lse", "dq", "dk", "dv"), clean, dirty):
        if name == "dq":  # (its sums come in any order)
            assert torch.isfinite(b[70:270]).all() and (a - b)[70:270].abs().max() <= 2 ** -6 * a[70:270].abs().max()
        else:
            assert torch.equal(a[70:270], b[70:270]), name
    assert not dirty[0][360:].any() and not any(t[360:].any() for t in dirty[2:])


@pytest.mark.parametrize("D", [64, 128])
def test_strided_operands(D):
    """q, k and v as parts of one projection's output, offsets at other rows, a gradient of any strides."""
    from tinytorch_b200 import function
    lens = (100, 31, 257)
    T = sum(lens)
    qkv = make(T, 12, D, torch.float16, 7)
    q, k, v = (x.detach().requires_grad_() for x in (qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]))
    g = make(8, T, D, torch.float16, 8).transpose(0, 1)
    o = function.sdpAttentionPacked(q, k, v, offsets(lens), True)
    got = torch.autograd.grad(o, (q, k, v), g)
    check((o, None, *got), q.detach(), k.detach(), v.detach(), lens, True, g=g)
    o = function.sdpAttentionPacked(q, k, v, offsets(lens), True)
    got = torch.autograd.grad(o.sum(), (q, k, v))  # (a gradient of one value, expanded)
    check((o, None, *got), q.detach(), k.detach(), v.detach(), lens, True, g=torch.ones_like(g))
    odd = torch.zeros(T * 8 * D + 1, dtype=torch.float16, device="cuda")[1:].view(T, 8, D)  # not on 16 bytes
    odd.copy_(g)
    o = function.sdpAttentionPacked(q, k, v, offsets(lens), True)
    check((o, None, *torch.autograd.grad(o, (q, k, v), odd)), q.detach(), k.detach(), v.detach(), lens, True, g=g)


@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales(scale):
    from tinytorch_b200 import op
    lens = (200, 3)
    q, k, v, g = (make(203, h, 64, torch.bfloat16, h + i) for i, h in enumerate((4, 2, 2, 4)))
    o, lse = op.sdpAttentionPackedFwd(q, k, v, offsets(lens), False, scale=scale)
    check((o, lse, *op.sdpAttentionPackedBwd(g, q, k, v, o, lse, offsets(lens), False, scale)), q, k, v, lens, False, scale=scale, g=g)


@pytest.mark.parametrize("cu", [[0, 50, 40, 100], [0, 101], [-1, 50], [10, 5], [0, 2 ** 31 - 1, 100]])
def test_bad_offsets_are_reported_and_give_zeros(cu):
    from tinytorch_b200 import op
    q, k, v, g = (make(100, h, 64, torch.bfloat16, h) for h in (4, 2, 2, 4))
    cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, True, status=status)
    assert int(status) == 16 and not o.any() and bool((lse == -math.inf).all())
    assert not any(x.any() for x in op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, True))


def test_offsets_that_start_later():
    from tinytorch_b200 import op
    q, k, v, g = (make(100, h, 64, torch.bfloat16, h) for h in (4, 2, 2, 4))
    cu = torch.tensor([30, 60, 90], dtype=torch.int32, device="cuda")
    o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, True)
    grads = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, True)
    assert not o[:30].any() and bool((lse[:, :30] == -math.inf).all()) and not any(x[:30].any() for x in grads)
    check((o[30:], lse[:, 30:], *(x[30:] for x in grads)), q[30:], k[30:], v[30:], (30, 30), True, g=g[30:])


def test_no_rows():
    from tinytorch_b200 import function, op
    q, k, v = (make(0, h, 64, torch.bfloat16, h).requires_grad_() for h in (4, 2, 2))
    cu = offsets((0, 0))
    o = function.sdpAttentionPacked(q, k, v, cu, True)
    assert o.shape == q.shape and all(x.shape[0] == 0 for x in torch.autograd.grad(o, (q, k, v), o.detach()))
    q = make(7, 4, 64, torch.bfloat16, 1).requires_grad_()  # queries without any keys
    o = function.sdpAttentionPacked(q, k, v, offsets((3, 4)), cuSeqlensK=cu)
    assert not o.any() and not torch.autograd.grad(o, q, torch.ones_like(o))[0].any()
    assert bool((op.sdpAttentionPackedFwd(q.detach(), k.detach(), v.detach(), offsets((3, 4)), cuSeqlensK=cu)[1] == -math.inf).all())


def test_which_gradients():
    from tinytorch_b200 import op
    lens = (64, 200)
    q, k, v, g = (make(264, h, 128, torch.bfloat16, h + i) for i, h in enumerate((4, 2, 2, 4)))
    cu = offsets(lens)
    o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, True)
    every = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, True)
    for i in range(3):
        needs = tuple(j == i for j in range(3))
        some = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, True, needs=needs)
        assert [x is not None for x in some] == list(needs)
        if i > 0:
            assert torch.equal(some[i], every[i])


def test_gradients_against_differences():
    """The loss is linear in O with weights g; its difference along a direction, in 64 bits, against the gradients."""
    from tinytorch_b200 import function
    lens = (90, 40, 150)
    T = sum(lens)
    q, k, v, g = (make(T, h, 64, torch.float16, 40 + i, 0.7) for i, h in enumerate((4, 2, 2, 4)))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(function.sdpAttentionPacked(*leaves, offsets(lens), True), leaves, g)

    def loss(q, k, v):
        total, a = 0.0, 0
        for n in lens:
            for h in range(2):
                o, _, _ = ref.attention(q[a:a + n, 2 * h:2 * h + 2].transpose(0, 1), k[a:a + n, h], v[a:a + n, h], 0.125, ref.visible(n, n, True, q.device))
                total = total + (o * g[a:a + n, 2 * h:2 * h + 2].double().transpose(0, 1)).sum()
            a += n
        return total.item()
    x = [t.double() for t in (q, k, v)]
    gen = torch.Generator(device="cuda").manual_seed(5)
    for i in range(3):
        d = torch.randn(x[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        plus, minus = ([t + s * 1e-4 * d if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        want = (loss(*plus) - loss(*minus)) / 2e-4
        got = (grads[i].double() * d).sum().item()
        # independent errors of half a 16-bit step in P, dS and the result: their sum along a random direction is that of a random walk
        size = (grads[i].double() * d).square().sum().sqrt().item()
        assert abs(got - want) <= 0.02 * size + 1e-6 * abs(want), (i, got, want, size)


def test_streams_and_graphs():
    """Another stream than the default; a captured pass follows new lengths in the same tensor; two graphs do not share scratch."""
    from tinytorch_b200 import function
    q, k, v = (make(640, h, 128, torch.bfloat16, 60 + h).requires_grad_() for h in (8, 2, 2))
    g = make(640, 8, 128, torch.bfloat16, 70)
    cus = [offsets(lens) for lens in ((640,), (100, 40, 500), (1, 0, 600))]
    cus = [torch.cat([c, c[-1:].expand(4 - len(c))]).contiguous() for c in cus]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            cu = cus[0].clone()
            for _ in range(2):
                o = function.sdpAttentionPacked(q, k, v, cu, True)
                torch.autograd.grad(o, (q, k, v), g)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                o = function.sdpAttentionPacked(q, k, v, cu, True)
                grads = torch.autograd.grad(o, (q, k, v), g)
            graphs.append((graph, cu, o.detach(), grads))
            del o  # (torch captures no backward of leaves whose eager graph is still held)
    torch.cuda.synchronize()
    for a, b in ((0, 1), (2, 0), (1, 2)):
        graphs[0][1].copy_(cus[a]), graphs[1][1].copy_(cus[b])
        torch.cuda.synchronize()
        one, two = torch.cuda.Stream(), torch.cuda.Stream()
        for s, gr in ((one, graphs[0]), (two, graphs[1])):
            with torch.cuda.stream(s):
                for _ in range(3):
                    gr[0].replay()
        torch.cuda.synchronize()
        for which, gr in ((a, graphs[0]), (b, graphs[1])):
            o = function.sdpAttentionPacked(q, k, v, cus[which], True)
            want = torch.autograd.grad(o, (q, k, v), g)
            assert torch.equal(gr[2], o) and torch.equal(gr[3][1], want[1]) and torch.equal(gr[3][2], want[2])
            assert (gr[3][0] - want[0]).abs().max() <= 2 ** -6 * want[0].abs().max()


@pytest.mark.parametrize("D", [64, 128])
def test_plans_that_follow_one_another(D):
    """Calls right behind one another, whose plans lie in the same scratch memory and differ, each on operands of its own."""
    from tinytorch_b200 import op

    g = torch.Generator().manual_seed(D)
    base = [64, 1, 130, 300, 17, 128, 0, 40]
    cases = []
    for i in range(30):
        lens = [base[j] for j in torch.randperm(len(base), generator=g)]
        cases.append([make(sum(lens), h, D, torch.bfloat16, 10 * i + h) for h in (8, 2, 2)] + [offsets(lens)])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [op.sdpAttentionPackedFwd(*c, True) for c in cases]
        grads = [op.sdpAttentionPackedBwd(c[0], *c[:3], *f, c[3], True) for c, f in zip(cases, got)]
    side.synchronize()
    for c, f, b in zip(cases, got, grads):
        one = op.sdpAttentionPackedFwd(*c, True)
        torch.cuda.synchronize()
        assert torch.equal(f[0], one[0]) and torch.equal(f[1], one[1])
        back = op.sdpAttentionPackedBwd(c[0], *c[:3], *one, c[3], True)
        torch.cuda.synchronize()
        # (dq is summed in any order)
        assert torch.equal(b[1], back[1]) and torch.equal(b[2], back[2])
        assert (b[0].float() - back[0].float()).abs().max() <= 2 ** -7 * back[0].float().abs().max()


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 8, 1), (64, 3, 3)])
def test_operands_that_end_where_their_memory_does(D, Hq, Hkv):
    from tinytorch_b200 import op

    lens = (200, 1, 900, 40)
    q, k, v, g = (make(sum(lens), h, D, torch.bfloat16, h) for h in (Hq, Hkv, Hkv, Hq))
    want = op.sdpAttentionPackedFwd(q, k, v, offsets(lens), True)
    qe, ke, ve, ge = (ref.at_the_end(x) for x in (q, k, v, g))
    cu = ref.at_the_end(offsets(lens))
    got = op.sdpAttentionPackedFwd(qe, ke, ve, cu, True)
    oe, le = ref.at_the_end(got[0]), ref.at_the_end(got[1]).contiguous()
    grads = op.sdpAttentionPackedBwd(ge, qe, ke, ve, oe, le, cu, True)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    back = op.sdpAttentionPackedBwd(g, q, k, v, *want, offsets(lens), True)
    assert torch.equal(grads[1], back[1]) and torch.equal(grads[2], back[2])


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 2, 1), (128, 3, 3)])
def test_thousands_of_sequences(D, Hq, Hkv):
    """More than the plan keeps in shared memory: each of 0 to 3 rows, and a long one among them."""
    lens = [(7 * i) % 4 for i in range(2500)]
    lens[1700] = 400
    q, k, v, g = (make(sum(lens) + 5, h, D, torch.float16, 3 + h) for h in (Hq, Hkv, Hkv, Hq))
    from tinytorch_b200 import op
    o, lse = op.sdpAttentionPackedFwd(q, k, v, offsets(lens), True)
    grads = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, offsets(lens), True)
    # the first 40, those around the long one, the last 40, each part a call of its own
    at = [0] + list(offsets(lens).tolist())[1:]
    for a, b in ((0, 40), (1690, 1712), (2460, 2500)):
        rows = slice(at[a], at[b])
        part = [x[rows] for x in (q, k, v)]
        po, pl = op.sdpAttentionPackedFwd(*part, offsets(lens[a:b]), True)
        back = op.sdpAttentionPackedBwd(g[rows], *part, po, pl, offsets(lens[a:b]), True)
        check((po, pl, *back), *part, lens[a:b], True, g=g[rows])
        assert torch.equal(o[rows], po) and torch.equal(lse[:, rows], pl)
        for x, y in zip(grads, back):
            assert (x[rows].float() - y.float()).abs().max() <= 2 ** -9 * y.float().abs().max()
    assert not o[at[-1]:].any() and not any(x[at[-1]:].any() for x in grads)


def test_rows_far_away():
    """Elements of q, o and dq beyond 2^31, bytes of the sum for dq beyond 2^32."""
    from tinytorch_b200 import op

    total, Hq, Hkv, D, n = 540_000, 32, 1, 128, 300
    q = torch.zeros(total, Hq, D, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.zeros(total, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert q.numel() > 2 ** 31
    for i, x in enumerate((q, k, v)):
        x[-n:] = make(n, x.shape[1], D, torch.bfloat16, i)
    cu = torch.tensor([total - n, total - 100, total], dtype=torch.int32, device="cuda")
    o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, True)
    part = [x[-n:].clone() for x in (q, k, v)]
    po, pl = op.sdpAttentionPackedFwd(*part, cu - (total - n), True)
    assert torch.equal(o[-n:], po) and torch.equal(lse[:, -n:], pl) and not o[:-n].any()
    grads = op.sdpAttentionPackedBwd(q, q, k, v, o, lse, cu, True)
    back = op.sdpAttentionPackedBwd(part[0], *part, po, pl, cu - (total - n), True)
    for x, y in zip(grads, back):
        assert (x[-n:].float() - y.float()).abs().max() <= 2 ** -6 * y.float().abs().max() and not x[:-n].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("most", [32, 64])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (4, 2), (6, 2), (16, 2), (14, 2), (6, 1), (3, 3)])
def test_short_sequences(D, Hq, Hkv, most):
    """Sequences of up to 32 or 64 rows, whose heads share tiles where they share keys, a longer one among them; lengths of the keys of their own."""
    from tinytorch_b200 import op

    lens, lens_k = ((1, 32, 0, 17, 31, 2, 33, 5, 32, 8, 20, 1), (32, 1, 4, 17, 0, 32, 33, 40, 9, 8, 31, 1))
    if most == 64:
        lens, lens_k = (64, 33, 0, 50, 63, 2, 65, 40, 64, 40, 1, 40), (64, 1, 9, 64, 0, 2, 70, 33, 80, 200, 1, 63)
    for causal, keys in ((True, None), (False, None), ("bottom-right", lens_k), (True, lens_k)):
        m, tail = sum(keys or lens), 0 if keys else 3
        q, k, v = (make(n + tail, h, D, torch.bfloat16, 5 + h) for n, h in ((sum(lens), Hq), (m, Hkv), (m, Hkv)))
        cu_k = None if keys is None else offsets(keys)
        o, lse = op.sdpAttentionPackedFwd(q, k, v, offsets(lens), causal, cuSeqlensK=cu_k)
        g = make(sum(lens) + tail, Hq, D, torch.bfloat16, 9)
        grads = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, offsets(lens), causal, cuSeqlensK=cu_k)
        check((o, lse, *grads), q, k, v, lens, causal, lens_k=keys, g=g)


@pytest.mark.parametrize("poison", [math.inf, math.nan])
def test_short_sequences_keep_to_themselves(poison):
    """An infinite value of one sequence, or of one kv head, is in no other's results."""
    from tinytorch_b200 import op

    lens, Hq, Hkv, D = (20, 9, 32, 16), 8, 2, 64
    q, k, v = (make(sum(lens), h, D, torch.bfloat16, h) for h in (Hq, Hkv, Hkv))
    want = op.sdpAttentionPackedFwd(q, k, v, offsets(lens), True)
    v[22, 1], k[23, 1] = poison, poison
    got = op.sdpAttentionPackedFwd(q, k, v, offsets(lens), True)
    keep = torch.ones(sum(lens), Hq, dtype=torch.bool, device="cuda")
    keep[20:29, 4:] = False
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1].t()[keep], want[1].t()[keep])
    assert not got[0][22:29, 4:].isfinite().all()
    g = make(sum(lens), Hq, D, torch.bfloat16, 4)
    back = op.sdpAttentionPackedBwd(g, q, k, v, *got, offsets(lens), True)
    v[22, 1], k[23, 1] = 0, 0
    clean = op.sdpAttentionPackedFwd(q, k, v, offsets(lens), True)
    fine = op.sdpAttentionPackedBwd(g, q, k, v, *clean, offsets(lens), True)
    for i, (x, y) in enumerate(zip(back, fine)):
        keep = torch.ones(x.shape[:2], dtype=torch.bool, device="cuda")
        keep[20:29, 4 if i == 0 else 1:] = False
        assert torch.equal(x[keep], y[keep])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (6, 2), (14, 2), (3, 3)])
@pytest.mark.parametrize("causal", ["bottom-right", True, False])
def test_few_new_rows_behind_many(D, Hq, Hkv, causal):
    """Short queries over long keys: heads share tiles of queries that walk over many tiles of keys."""
    from tinytorch_b200 import op

    for lens, keys in (((20, 1, 32, 0, 9, 40, 3), (700, 129, 300, 50, 0, 500, 128)), ((60, 64, 1, 40, 33, 90, 5), (1000, 64, 257, 1, 384, 90, 70))):
        q = make(sum(lens), Hq, D, torch.float16, 1)
        k, v = (make(sum(keys), Hkv, D, torch.float16, i) for i in (2, 3))
        cu, cu_k = offsets(lens), offsets(keys)
        o, lse = op.sdpAttentionPackedFwd(q, k, v, cu, causal, cuSeqlensK=cu_k)
        g = make(sum(lens), Hq, D, torch.float16, 4)
        grads = op.sdpAttentionPackedBwd(g, q, k, v, o, lse, cu, causal, cuSeqlensK=cu_k)
        check((o, lse, *grads), q, k, v, lens, causal, lens_k=keys, g=g)


@pytest.mark.parametrize("D", [64, 128])
def test_short_sequences_of_other_layouts(D):
    """Parts of a projection's output, heads outside rows, gradients of any strides, no keys at all."""
    from tinytorch_b200 import op

    lens, Hq, Hkv = (20, 0, 31, 5, 32, 1), 8, 2
    n = sum(lens)
    qkv = make(n, Hq + 2 * Hkv, D, torch.bfloat16, 1)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    g = make(n, Hq, D, torch.bfloat16, 2)
    want = op.sdpAttentionPackedFwd(q.contiguous(), k.contiguous(), v.contiguous(), offsets(lens), True)
    back = op.sdpAttentionPackedBwd(g, q.contiguous(), k.contiguous(), v.contiguous(), *want, offsets(lens), True)
    swap = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, g)]
    for a, b, c, d in ((q, k, v, g), swap):
        o, lse = op.sdpAttentionPackedFwd(a, b, c, offsets(lens), True)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        got = op.sdpAttentionPackedBwd(d, a, b, c, o, lse, offsets(lens), True)
        assert torch.equal(got[1], back[1]) and torch.equal(got[2], back[2])
        assert (got[0].float() - back[0].float()).abs().max() <= 2 ** -7 * back[0].float().abs().max()
    none = torch.zeros(0, Hkv, D, dtype=torch.bfloat16, device="cuda")
    o, lse = op.sdpAttentionPackedFwd(q, none, none, offsets(lens), True, cuSeqlensK=torch.zeros(7, dtype=torch.int32, device="cuda"))
    assert not o.any() and bool((lse == -math.inf).all())


def test_offsets_changed_between_the_passes_are_an_error():
    from tinytorch_b200 import function
    q, k, v = (make(64, h, 64, torch.bfloat16, h).requires_grad_() for h in (4, 2, 2))
    cu = offsets((30, 34))
    o = function.sdpAttentionPacked(q, k, v, cu, True)
    cu[1] = 20
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_python_function_has_the_same_results():
    from tinytorch_b200 import function
    lens = (64, 100)
    q, k, v = (make(164, h, 64, torch.bfloat16, h).requires_grad_() for h in (4, 2, 2))
    g = make(164, 4, 64, torch.bfloat16, 9)
    a = function.sdpAttentionPacked(q, k, v, offsets(lens), True)
    b = function.FuncSDPAttentionPacked.apply(q, k, v, offsets(lens), None, True, 0.125)
    assert torch.equal(a, b)
    for x, y in zip(torch.autograd.grad(a, (q, k, v), g)[1:], torch.autograd.grad(b, (q, k, v), g)[1:]):
        assert torch.equal(x, y)
