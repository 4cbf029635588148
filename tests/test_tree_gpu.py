"""GPU: trees of drafted tokens over a cache, and what is accepted of them, against a 64-bit form."""
import math

import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def randn(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def tree(B, T, seed):
    """Ancestors of every draft and itself; parents are earlier drafts or the sequence's last token."""
    g = torch.Generator().manual_seed(seed)
    m = torch.eye(T, dtype=torch.bool).repeat(B, 1, 1)
    for b in range(B):
        for i in range(1, T):
            p = int(torch.randint(-1, i, (1,), generator=g))
            if p >= 0:
                m[b, i] |= m[b, p]
    return m.cuda()


def bound_f32(p, v, o, s_size):
    """fp32: a score, D products in chains of D / 4 sums of 4, is off by (D / 4 + 8) steps of 2^-24 of the sum of its products' sizes, which
    moves a probability by as much; the exponential by 2^-22, sums over keys (chains of one tile's 64, tiles, pieces) by 200 steps."""
    return ((s_size + 4 + 200) * 2.0 ** -24) * (p @ v.abs() + o.abs()) + 2.0 ** -126


def check(q, kd, vd, kc, vc, lens, mask, scale=None, **kw):
    from tinytorch_b200 import op
    B, Hq, T, D = q.shape
    Hkv, group = kc.shape[1], Hq // kc.shape[1]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o, lse = op.sdpAttentionTree(q, kd, vd, kc, vc, None if lens is None else ints(lens), mask, scale, needLse=True, status=status, **kw)
    scale = 1 / math.sqrt(D) if scale is None else scale
    assert int(status) == 0
    for b in range(B):
        n = kc.shape[2] if lens is None else max(0, min(lens[b], kc.shape[2]))
        m = torch.ones(T, T, dtype=torch.bool, device="cuda").tril() if mask is None else (mask[b if mask.shape[0] > 1 else 0] if mask.dim() == 3 else mask)
        sees = torch.cat((torch.ones(T, n, dtype=torch.bool, device="cuda"), m), 1)
        for h in range(Hkv):
            hs = slice(h * group, (h + 1) * group)
            k, v = (torch.cat((c[b, h, :n], d[b, h])).double() for c, d in ((kc, kd), (vc, vd)))
            qh = q[b, hs].double()
            wo, wl, p = ref.attention(qh, k, v, scale, sees)
            if q.dtype == torch.float32:
                size = ((qh.abs() @ k.abs().t()) * abs(scale)).amax().item() * (D / 4 + 8)
                bound = bound_f32(p, v, wo, size)
                lse_bound = (size + 204) * 2.0 ** -24 + wl.abs() * 2.0 ** -22
            else:
                # (halves and pieces of a walk round P against maxima of their own: still one rounding of every term)
                bound, lse_bound = ref.attention_bound(p, v, wo, q.dtype), torch.full_like(wl, ref.SLOP)
            ref.within(o[b, hs], wo, bound, "sequence %d head %d" % (b, h))
            assert torch.equal(lse[b, hs] == -math.inf, wl == -math.inf)
            some = wl > -math.inf
            assert bool(((lse[b, hs].double() - wl).abs() <= lse_bound)[some].all())
    return o, lse


def operands(B, Hq, Hkv, T, cap, D, dtype, seed=1):
    return [randn(s, dtype, seed + i) for i, s in enumerate(((B, Hq, T, D), (B, Hkv, T, D), (B, Hkv, T, D), (B, Hkv, cap, D), (B, Hkv, cap, D)))]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv,T,cap,lens", [
    (1, 1, 1, 1, (1,)),                                    # the smallest call
    (4, 4, 1, 300, (0, 1, 128, 300)),                      # one draft; an empty cache, a full one
    (8, 2, 5, 700, (129, 0, 64, 63, 700, 511)),            # either side of tiles
    (12, 4, 33, 260, (256, 3)),                            # groups that do not divide a block
    (5, 1, 64, 1000, (999,)),
    (32, 8, 32, 2100, (2048, 100)),                        # whole blocks of 128 rows
    (6, 2, 128, 400, (257, 400)),                          # the most drafts
    (2, 2, 127, 130, (0, 2)),
])
def test_trees(dt, D, Hq, Hkv, T, cap, lens):
    x = operands(len(lens), Hq, Hkv, T, cap, D, DTYPES[dt])
    check(*x, lens, tree(len(lens), T, 5))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_chains_and_shared_masks(dt, D):
    x = operands(3, 8, 2, 20, 200, D, DTYPES[dt])
    check(*x, (150, 0, 200), None)
    check(*x, None, None, 0.3)
    check(*x, (150, 0, 200), tree(1, 20, 6)[0], -0.2)
    check(*x, (150, 0, 200), tree(1, 20, 7), 0.0)
    wide = torch.zeros(3, 25, 41, dtype=torch.bool, device="cuda")  # rows at any offset and stride
    wide[:, 2:22, 7:27] = tree(3, 20, 8)
    check(*x, (150, 7, 200), wide[:, 2:22, 7:27])
    check(*x, (150, 7, 200), tree(3, 20, 9).transpose(1, 2))  # (what sees what is the caller's business)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_see_nothing(dt, D):
    from tinytorch_b200 import op
    x = operands(2, 4, 2, 40, 100, D, DTYPES[dt])
    m = tree(2, 40, 3)
    m[:, 5] = False
    m[1, 30:] = False
    o, lse = check(*x, (0, 0), m)
    assert not o[:, :, 5].any() and not o[1, :, 30:].any() and bool((lse[:, :, 5] == -math.inf).all())
    check(*x, (0, 100), torch.zeros_like(m))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_what_lies_behind_the_length(dt, poison):
    x = operands(2, 8, 2, 9, 400, 128, DTYPES[dt])
    x[3][0, :, 130:] = poison
    x[4][0, :, 130:] = poison
    x[3][1] = poison
    x[4][1] = poison
    check(*x, (130, 0), tree(2, 9, 4))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_long_caches_and_many_sequences(dt):
    """Walks that are broken into many pieces; more sequences than threads look at a time; lengths outside the cache."""
    x = operands(1, 8, 1, 16, 30000, 64, DTYPES[dt])
    check(*x, (29999,), tree(1, 16, 3))
    lens = [(i * 37) % 90 for i in range(600)]
    lens[3], lens[4] = -5, 1000
    check(*operands(600, 2, 1, 3, 80, 64, DTYPES[dt]), lens, tree(600, 3, 4))


def test_strides():
    """Token-major drafts, caches that are parts of larger tensors, one cache for all sequences."""
    B, Hq, Hkv, T, D = 2, 6, 2, 7, 64
    qkv = randn((B, T, Hq + 2 * Hkv, D), torch.bfloat16, 1)
    q, kd, vd = (x.transpose(1, 2) for x in qkv.split((Hq, Hkv, Hkv), 2))
    both = randn((2, B, 500, Hkv, D), torch.bfloat16, 2)
    kc, vc = (x[:, 100:400].transpose(1, 2) for x in both)
    check(q, kd, vd, kc, vc, (300, 177), tree(B, T, 3))
    one = [x[:1].contiguous().expand(B, -1, -1, -1) for x in (kc, vc)]
    check(q, kd, vd, *one, (300, 177), tree(B, T, 3))
    check(q[:, :, :1], kd[:, :, :1], vd[:, :, :1], kc, vc, (300, 177), None)


def test_scores_that_grow():
    """Later tiles with larger scores (the running maximum moves), and scores near the ends of the range."""
    x = operands(1, 4, 1, 6, 1500, 128, torch.bfloat16)
    x[3] *= torch.linspace(0.1, 6, 1500, device="cuda")[:, None].to(torch.bfloat16)
    check(*x, (1500,), tree(1, 6, 3), 0.3)


def test_workspaces_streams_and_graphs():
    from tinytorch_b200 import _capi, op
    B, Hq, Hkv, T, cap, D = 3, 8, 2, 12, 900, 128
    x, m = operands(B, Hq, Hkv, T, cap, D, torch.bfloat16), tree(B, T, 3)
    need = _capi.lib().tt_attn_tree_workspace_bytes(_capi.BF16, B, Hq, Hkv, T, cap, D)
    lens = [ints(l) for l in ((900, 3, 500), (0, 900, 1))]
    want = [op.sdpAttentionTree(*x, l, m)[0] for l in lens]
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert torch.equal(op.sdpAttentionTree(*x, lens[0], m, workspace=ws)[0], want[0])
    with pytest.raises(_capi.AttnError):
        op.sdpAttentionTree(*x, lens[0], m, workspace=ws[:need - 256])
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        held = lens[0].clone()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            op.sdpAttentionTree(*x, held, m)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                o = op.sdpAttentionTree(*x, held, m)[0]
        graphs.append((g, held, o))
    graphs[1][1].copy_(lens[1])
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (g, _, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][2], want[0]) and torch.equal(graphs[1][2], want[1])


# ---------------------------------------------------------------------------------------------------- accept --
def accepted(kd, vd, kc, vc, lens, path, counts):
    """What cacheAccept does, row by row -> (caches, new lengths, status)."""
    kc, vc, new, status = kc.clone(), vc.clone(), [], 0
    cap = kc.shape[2]
    for b, (n, c) in enumerate(zip(lens, counts)):
        n = max(0, min(n, cap))
        if not 0 <= c <= len(path[b]):
            status, c = status | 16, max(0, min(c, len(path[b])))
        done = 0
        for j in path[b][:c]:
            if not 0 <= j < kd.shape[2]:
                status |= 16
                break
            if n + done >= cap:
                status |= 4
                break
            kc[b, :, n + done], vc[b, :, n + done] = kd[b, :, j], vd[b, :, j]
            done += 1
        new.append(n + done)
    return kc, vc, new, status


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,path,counts", [
    ((0,), [[0]], (1,)),
    ((5, 90, 0), [[0, 2, 6], [1, 1, 1], [6, 0, 3]], (3, 2, 0)),      # the same draft twice, nothing accepted
    ((98, 100, 99), [[0, 1, 2], [0, 1, 2], [3, 4, 5]], (3, 1, 1)),   # full caches
    ((5, 6, 7), [[0, 7, 1], [-1, 0, 0], [0, 1, 2 ** 31 - 1]], (3, 3, 2)),  # drafts that do not exist, one of them not asked for
    ((-3, 200, 50), [[0, 1, 2]] * 3, (2, 2, 2)),
    ((5, 6, 7), [[0, 1, 2]] * 3, (-1, 4, 2 ** 31 - 1)),
    ((5, 6), [[]] * 2, (0, 0)),
])
def test_accept(dt, D, lens, path, counts):
    from tinytorch_b200 import op
    B, dtype = len(lens), DTYPES[dt]
    kd, vd = randn((B, 3, 7, D), dtype, 1), randn((B, 7, 3, D), dtype, 2).transpose(1, 2)
    kc, vc = randn((B, 3, 100, D), dtype, 3), randn((B, 100, 3, D), dtype, 4).transpose(1, 2)
    want = accepted(kd, vd, kc, vc, lens, path, counts)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    new = op.cacheAccept(kd, vd, kc, vc, ints(lens), ints(path).reshape(B, -1), ints(counts), status=status)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]) and new.tolist() == want[2] and int(status) == want[3]


def test_accept_long_paths():
    from tinytorch_b200 import op
    kd, vd = randn((2, 8, 128, 64), torch.float16, 1), randn((2, 8, 128, 64), torch.float16, 2)
    kc, vc = randn((2, 8, 400, 64), torch.float16, 3), randn((2, 8, 400, 64), torch.float16, 4)
    g = torch.Generator().manual_seed(1)
    path = torch.randint(0, 128, (2, 100), generator=g)
    path[1, 70] = 128
    want = accepted(kd, vd, kc, vc, (300, 17), path.tolist(), (100, 90))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    new = op.cacheAccept(kd, vd, kc, vc, ints((300, 17)), path.int().cuda(), ints((100, 90)), status=status)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]) and new.tolist() == [400, 87] and int(status) == 16


def test_a_cache_beyond_32_bits():
    """Rows whose offset in elements passes 2^32."""
    from tinytorch_b200 import op
    B, Hkv, cap, D, T = 1, 1, (1 << 25) + 700, 128, 3  # 8.6 GB a cache
    kc, vc = (torch.zeros(B, Hkv, cap, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, kd, vd = randn((B, 4, T, D), torch.bfloat16, 1), randn((B, Hkv, T, D), torch.bfloat16, 2), randn((B, Hkv, T, D), torch.bfloat16, 3)
    n = cap - 2
    new = op.cacheAccept(kd, vd, kc, vc, ints((n,)), ints([[2, 0]]), ints((2,)))
    assert int(new) == cap and torch.equal(kc[0, 0, n], kd[0, 0, 2]) and torch.equal(vc[0, 0, n + 1], vd[0, 0, 0])
    # all but the last two rows score 0 with values 0: the rest by hand
    o, lse = op.sdpAttentionTree(q, kd, vd, kc, vc, needLse=True)
    keys = torch.cat((kc[0, 0, n:], kd[0, 0])).double()
    values = torch.cat((vc[0, 0, n:], vd[0, 0])).double()
    x = q[0].double() @ keys.t() / math.sqrt(D)
    x[:, torch.ones(T, T, device="cuda").triu(1).bool().nonzero()[:, 0], 2 + torch.ones(T, T, device="cuda").triu(1).bool().nonzero()[:, 1]] = -math.inf
    total = x.exp().sum(-1) + n
    assert (lse[0].double() - total.log()).abs().max() <= ref.SLOP
    ref.within(o[0], (x.exp() @ values) / total[..., None], 2 ** -7 * (x.exp() @ values.abs()) / total[..., None], "o")


def test_a_layer_trains_and_serves():
    """The operators in a row as a program has them: a projection's q, k and v, normalised and rotated, through packed attention with
    gradients; then a step of the same weights with a tree of drafts over the prompts' cache, and what it accepts.  A path that is
    accepted gives the same outputs as the longer prompt."""
    from tinytorch_b200 import function, fused, op
    Hq, Hkv, D, hidden, dtype = 8, 2, 64, 256, torch.bfloat16
    prompts, T, path = (40, 129, 7), 6, [0, 2, 5]
    B = len(prompts)
    w = randn(((Hq + 2 * Hkv) * D, hidden), dtype, 1, 0.06).requires_grad_()
    nq, nk = ((1 + 0.1 * randn((D,), dtype, i)).requires_grad_() for i in (2, 3))
    cos, sin = op.ropeTables(400, D)

    def project(x, pos):
        q, k, v = fused.linear(x, w).view(-1, Hq + 2 * Hkv, D).split((Hq, Hkv, Hkv), 1)
        return (*fused.qkNormRope(q, k, nq, nk, cos, sin, pos), v)
    cu = ints([0] + list(prompts)).cumsum(0, dtype=torch.int32)
    x = randn((sum(prompts), hidden), dtype, 4).requires_grad_()
    pos = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in prompts])
    q, k, v = project(x, pos)
    o = function.sdpAttentionPacked(q, k, v, cu, isCausal=True)
    grads = torch.autograd.grad(o, (x, w, nq, nk), randn(o.shape, dtype, 5))
    assert all(torch.isfinite(g).all() and g.any() for g in grads)

    kc, vc = (torch.full((B, Hkv, 200, D), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    at = 0
    for b, n in enumerate(prompts):
        kc[b, :, :n], vc[b, :, :n] = k[at:at + n].detach().transpose(0, 1), v[at:at + n].detach().transpose(0, 1)
        at += n
    lens, mask = ints(prompts), torch.eye(T, dtype=torch.bool, device="cuda")
    mask[2, 0] = mask[5, 0] = mask[5, 2] = mask[1, 0] = mask[3, 1] = mask[3, 0] = True
    depth = mask.sum(1, dtype=torch.int32) - 1
    drafts = randn((B * T, hidden), dtype, 6)
    with torch.no_grad():
        q, kd, vd = (t.view(B, T, -1, D).transpose(1, 2) for t in project(drafts, (lens[:, None] + depth).flatten()))
    out, _ = op.sdpAttentionTree(q, kd, vd, kc, vc, lens, mask)
    new = op.cacheAccept(kd, vd, kc, vc, lens, ints([path] * B), ints([3] * B))
    assert new.tolist() == [n + 3 for n in prompts]
    with torch.no_grad():
        xs, ps = [], []
        for b, part in enumerate(x.split(prompts)):
            xs += [part, drafts.view(B, T, hidden)[b, path]]
            ps.append(torch.arange(prompts[b] + 3, device="cuda", dtype=torch.int32))
        q2, k2, v2 = project(torch.cat(xs), torch.cat(ps))
        longer = function.sdpAttentionPacked(q2, k2, v2, ints([0] + [n + 3 for n in prompts]).cumsum(0, dtype=torch.int32), isCausal=True)
    at = 0
    for b, n in enumerate(prompts):
        assert torch.equal(kc[b, :, n:n + 3], k2[at + n:at + n + 3].transpose(0, 1))
        # the same rows rounded against other maxima: two results within a rounding of P and of O each
        a, c = out[b, :, path].transpose(0, 1).double(), longer[at + n:at + n + 3].double()
        assert (a - c).abs().max() <= 4 * 2.0 ** -8 * v2[at:at + n + 3].abs().max().item()
        at += n + 3


@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_operands_that_end_where_their_memory_does(dt, D):
    from tinytorch_b200 import op

    g = torch.Generator(device="cuda").manual_seed(D)
    q, kd, vd, kc, vc = (torch.randn(2, h, n, D, generator=g, device="cuda").to(dt) for h, n in ((6, 5), (2, 5), (2, 5), (2, 301), (2, 301)))
    lens = torch.tensor([301, 77], dtype=torch.int32, device="cuda")
    mask = (torch.rand(2, 5, 5, generator=g, device="cuda") < 0.6) | torch.eye(5, dtype=torch.bool, device="cuda")
    path, counts = torch.tensor([[0, 2], [1, 4]], dtype=torch.int32, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    want = op.sdpAttentionTree(q, kd, vd, kc, vc, lens, mask, needLse=True)
    e = [ref.at_the_end(x) for x in (q, kd, vd, kc, vc, lens, mask, path, counts)]
    got = op.sdpAttentionTree(*e[:7], needLse=True)
    new = op.cacheAccept(*e[1:6], *e[7:])
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert new.tolist() == [301, 79] and torch.equal(e[3][1, :, 77:79], kd[1][:, [1, 4]])
