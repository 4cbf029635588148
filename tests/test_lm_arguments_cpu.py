"""CPU: arguments of the operators around attention that do not belong together are refused before anything is launched; their
64-bit forms' gradients against differences.

The tensors are fake CUDA tensors (no memory behind them), so a call that is let through fails on the missing driver, with
another error than the ValueError asked for here."""
import ctypes as C
import math
import os

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import lm_reference as ref
from conftest import ROOT
from tinytorch_b200 import _capi, function, fused, op


@pytest.fixture(autouse=True)
def built():
    if not os.path.exists(os.path.join(ROOT, "tinytorch_b200", "lib", "_native.so")):
        from tinytorch_b200.build import build, build_native
        build()
        build_native()


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield


def t(*shape, dtype=torch.bfloat16, device="cuda"):
    return torch.empty(shape, dtype=dtype, device=device)


def ints(*shape, device="cuda", dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device=device)


# ------------------------------------------------------------------------------------------ norm and rotation --
def rope_args(**kw):
    a = dict(q=t(9, 8, 64), k=t(9, 2, 64), qWeight=t(64), kWeight=t(64), cos=t(50, 32, dtype=torch.float32), sin=t(50, 32, dtype=torch.float32),
             positions=ints(9))
    a.update({n: f() if callable(f) else f for n, f in kw.items()})
    return a


@pytest.mark.parametrize("kw", [
    dict(q=lambda: t(9, 8, 64, device="cpu")), dict(q=lambda: t(9, 8, 64, dtype=torch.float64)), dict(q=lambda: t(8, 64)),
    dict(k=lambda: t(8, 2, 64)), dict(k=lambda: t(9, 2, 128)), dict(k=lambda: t(9, 2, 64, dtype=torch.float16)), dict(k=lambda: t(1, 2, 9, 64)),
    dict(q=lambda: t(9, 64, 8).transpose(1, 2)), dict(qWeight=lambda: t(32)), dict(kWeight=lambda: t(64, dtype=torch.float32)),
    dict(qWeight=lambda: t(128)[::2]), dict(kWeight=lambda: t(64, device="cpu")), dict(cos=None), dict(sin=None), dict(positions=None),
    dict(cos=None, sin=None), dict(cos=lambda: t(50, 64, dtype=torch.float32)), dict(sin=lambda: t(49, 32, dtype=torch.float32)),
    dict(cos=lambda: t(50, 32)), dict(positions=lambda: ints(8)), dict(positions=lambda: ints(9, dtype=torch.int64)),
    dict(positions=lambda: ints(1, 9)), dict(positions=lambda: ints(9, device="cpu")), dict(sections=(16, 16)),
    dict(positions=lambda: ints(2, 9), sections=(16, 17)), dict(positions=lambda: ints(2, 9), sections=(33, -1)),
    dict(positions=lambda: ints(3, 9), sections=(16, 16)), dict(positions=lambda: ints(5, 9), sections=(8, 8, 8, 4, 4)), dict(positions=lambda: ints(1, 9), sections=()),
    dict(status=lambda: ints(1, dtype=torch.int64)),
])
def test_norm_rope_refuses(fake, kw):
    with pytest.raises(ValueError):
        fused.qkNormRope(**rope_args(**kw))


def test_norm_rope_refuses_types(fake):
    with pytest.raises(TypeError):
        fused.qkNormRope(**rope_args(q=3))
    with pytest.raises(TypeError):
        fused.qkNormRope(**rope_args(positions=ints(2, 9), sections=5))


def test_norm_rope_batched_positions(fake):
    q, k = t(2, 8, 9, 64), t(2, 2, 9, 64)
    for bad in (ints(3, 9), ints(2, 8), ints(2, 2, 9)):
        with pytest.raises(ValueError):
            fused.qkNormRope(**rope_args(q=q, k=k, positions=bad))


def rope_params(**kw):
    p = _capi.QkNormRopeParams()
    p.struct_size = C.sizeof(p)
    p.dtype, p.B, p.Hq, p.Hkv, p.S, p.D = 2, 1, 8, 2, 9, 64
    p.q = p.k = p.q_out = p.k_out = p.q_weight = p.rope_cos = p.rope_sin = p.positions = 0x1000
    p.rope_positions, p.n_axes = 50, 1
    for n, v in kw.items():
        setattr(p, n, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), -8), (dict(dtype=3), -2), (dict(Hkv=0), -3), (dict(S=-1), -3), (dict(D=96), -4), (dict(q=None), -1), (dict(k_out=None), -1),
    (dict(q=0x1004), -5), (dict(q_weight=0x1002), -5), (dict(rope_cos=None), -1), (dict(rope_sin=0x1008), -5), (dict(rope_positions=0), -3),
    (dict(n_axes=0), -3), (dict(n_axes=5), -3), (dict(n_axes=2), -3), (dict(positions=None), -1), (dict(positions=0x1001), -5),
    (dict(position_axis_stride=-1), -3), (dict(q_strides=_capi.Strides(4096, 64, 60)), -5), (dict(S=2 ** 31 - 1, B=2), -10), (dict(Hq=70000), -10),
    (dict(S=0), 0),
])
def test_norm_rope_abi(kw, code):
    lib = _capi.lib()
    assert lib.tt_qk_norm_rope(C.byref(rope_params(**kw))) == code
    assert lib.tt_qk_norm_rope(None) == -1 and lib.tt_qk_norm_rope_bwd(None) == -1


def test_norm_rope_backward_abi():
    lib = _capi.lib()

    def params(fwd=(), **kw):
        p = _capi.QkNormRopeBwdParams()
        p.fwd, p.struct_size = rope_params(**dict(fwd)), C.sizeof(p)
        p.dq_out = p.dk_out = p.dq_weight = 0x1000
        for n, v in kw.items():
            setattr(p, n, v)
        return C.byref(p)
    assert lib.tt_qk_norm_rope_bwd(params(struct_size=8)) == -8
    assert lib.tt_qk_norm_rope_bwd(params(dict(D=32))) == -4
    assert lib.tt_qk_norm_rope_bwd(params(dq_out=None)) == -1
    assert lib.tt_qk_norm_rope_bwd(params(dk_weight=0x1000)) == -1  # (k has no norm)
    assert lib.tt_qk_norm_rope_bwd(params(dq_out=0x1008)) == -5
    assert lib.tt_qk_norm_rope_bwd(params(dq_weight=0x1001)) == -5
    assert lib.tt_qk_norm_rope_bwd(params(dict(q_out=None, k_out=None), dq_weight=None)) == 0  # (nothing is asked for)
    # shares of dw for every CTA, of which there are no more than 4 to an SM
    w = lib.tt_qk_norm_rope_workspace_bytes
    assert w(1, 32, 8, 100000, 128) == 4 * 148 * 128 * 4 and 0 < w(1, 1, 1, 1, 64) <= 1024 and w(1, 0, 1, 1, 64) == 0


# ---------------------------------------------------------------------------------------------------- packed --
PACKED = [
    dict(q=lambda: t(1, 40, 8, 64)), dict(q=lambda: t(40, 8, 64, device="cpu")), dict(k=lambda: t(40, 2, 128)), dict(v=lambda: t(40, 4, 64)),
    dict(v=lambda: t(39, 2, 64)), dict(k=lambda: t(41, 2, 64), v=lambda: t(41, 2, 64)), dict(k=lambda: t(40, 2, 64, dtype=torch.float16)),
    dict(cu=lambda: ints(1)), dict(cu=lambda: ints(2, 2)), dict(cu=lambda: ints(3, dtype=torch.int64)), dict(cu=lambda: ints(3, device="cpu")),
    dict(cu=lambda: ints(6)[::2]), dict(cuk=lambda: ints(4)), dict(cuk=lambda: ints(3, dtype=torch.int64)), dict(q=lambda: t(40, 64, 8).transpose(1, 2)),
]


@pytest.mark.parametrize("kw", PACKED)
def test_packed_refuses(fake, kw):
    a = dict(q=t(40, 8, 64), k=t(40, 2, 64), v=t(40, 2, 64), cu=ints(3), cuk=None)
    a.update({n: f() for n, f in kw.items()})
    args = a["q"], a["k"], a["v"], a["cu"]
    with pytest.raises(ValueError):
        function.sdpAttentionPacked(*args, cuSeqlensK=a["cuk"])
    with pytest.raises(ValueError):
        op.sdpAttentionPackedFwd(*args, cuSeqlensK=a["cuk"])
    with pytest.raises(ValueError):
        op.sdpAttentionPackedBwd(t(40, 8, 64), *args[:3], t(40, 8, 64), t(8, 40, dtype=torch.float32), args[3], cuSeqlensK=a["cuk"])


def test_packed_refuses_single_precision(fake):
    x = t(40, 8, 64, dtype=torch.float32)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        function.sdpAttentionPacked(x, x, x, ints(3))


@pytest.mark.parametrize("name,x", [("dO", lambda: t(39, 8, 64)), ("dO", lambda: t(40, 8, 64, dtype=torch.float16)), ("o", lambda: t(40, 7, 64)),
                                    ("lse", lambda: t(8, 39, dtype=torch.float32)), ("lse", lambda: t(8, 40))])
def test_packed_backward_operands(fake, name, x):
    a = dict(dO=t(40, 8, 64), q=t(40, 8, 64), k=t(40, 2, 64), v=t(40, 2, 64), o=t(40, 8, 64), lse=t(8, 40, dtype=torch.float32))
    a[name] = x()
    with pytest.raises(ValueError):
        op.sdpAttentionPackedBwd(*a.values(), ints(3))


def packed_params(cls, **kw):
    p = cls()
    p.struct_size = C.sizeof(p)
    p.dtype, p.n_seqs, p.Hq, p.Hkv, p.total_q, p.total_k, p.D = 2, 3, 8, 2, 100, 100, 64
    p.q = p.k = p.v = p.o = p.cu_q = 0x1000
    if cls is _capi.PackedBwdParams:
        p.d_o = p.lse = p.dq = p.dk = p.dv = 0x1000
    for n, v in kw.items():
        setattr(p, n, v)
    return C.byref(p)


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), -8), (dict(dtype=0), -2), (dict(n_seqs=0), -3), (dict(Hq=9), -3), (dict(total_q=-1), -3), (dict(D=96), -4), (dict(q=None), -1),
    (dict(cu_q=None), -1), (dict(total_k=99), -3), (dict(cu_k=0x1002), -5), (dict(is_causal=3), -3), (dict(k=0x1008), -5),
    (dict(q_strides=_capi.Strides(0, 64, 60)), -5), (dict(q_strides=_capi.Strides(0, 64, -512)), -5), (dict(Hq=131072), -10),
    (dict(n_seqs=2 ** 31 - 1), -10),
])
def test_packed_abi(kw, code):
    lib = _capi.lib()
    assert lib.tt_attn_packed_fwd(packed_params(_capi.PackedFwdParams, **kw)) == code
    assert lib.tt_attn_packed_bwd(packed_params(_capi.PackedBwdParams, **kw)) == code
    assert lib.tt_attn_packed_fwd(None) == -1 and lib.tt_attn_packed_bwd(None) == -1


def test_packed_abi_nothing_to_do():
    lib = _capi.lib()
    assert lib.tt_attn_packed_fwd(packed_params(_capi.PackedFwdParams, total_q=0, total_k=0)) == 0
    assert lib.tt_attn_packed_bwd(packed_params(_capi.PackedBwdParams, dq=None, dk=None, dv=None)) == 0


def test_packed_workspace():
    """Whatever the lengths are, the items fit: every sequence can have one tile more than its rows fill."""
    w = _capi.lib().tt_attn_packed_workspace_bytes
    for n, Hq, Hkv, T in ((1, 8, 2, 1), (7, 8, 8, 1000), (100, 32, 8, 3000)):
        group = Hq // Hkv
        items = (n - 1 + max(1, math.ceil((T - (n - 1)) / 128))) * group
        assert w(_capi.KIND_FWD, n, Hq, Hkv, T, T, 128) >= items * 32 + n * 4 * 128 + 8
        assert w(_capi.KIND_BWD, n, Hq, Hkv, T, T, 128) >= items // group * 32 + n * 7 * 128 + Hq * T * (1 + 128) * 4 + 8
    assert w(2, 1, 8, 2, 1, 1, 128) == 0 and w(0, 0, 8, 2, 1, 1, 128) == 0


# ------------------------------------------------------------------------------------------------ the forms --
def test_the_forms_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    q, k, v, do = r(3, 7, 8), r(5, 8), r(5, 8), r(3, 7, 8)
    sees = torch.rand(7, 5, generator=g) < 0.6
    sees[2] = False
    o, _, p = ref.attention(q, k, v, 0.3, sees)
    got = ref.attention_grads(q, k, v, o, do, p, 0.3, torch.bfloat16)
    for i, x in enumerate((q, k, v)):
        d = r(*x.shape)
        f = lambda s: (ref.attention(*(y + s * d if j == i else y for j, y in enumerate((q, k, v))), 0.3, sees)[0] * do).sum()
        assert abs((f(1e-6) - f(-1e-6)) / 2e-6 - (got[i][0] * d).sum()) <= 1e-7
    for interleaved in (False, True):
        x, w, go = r(6, 2, 8), r(8), r(6, 2, 8)
        a = r(6, 1, 4)
        cs = a.cos(), a.sin()
        u = ref.turn(go, cs[0], -cs[1], interleaved)
        rr = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-3)
        n = x * rr
        dx = rr * (u * w - n * (u * w * n).mean(-1, keepdim=True))
        dw = (u * n).sum((0, 1))
        for i, (y, want) in enumerate(((x, dx), (w, dw))):
            d = r(*y.shape)
            f = lambda s: (ref.norm_rope(x + s * d if i == 0 else x, w + s * d if i == 1 else w, cs, 1e-3, interleaved) * go).sum()
            assert abs((f(1e-6) - f(-1e-6)) / 2e-6 - (want * d).sum()) <= 1e-7


# ---------------------------------------------------------------------------------------------- tree and accept --
def tree_args(**kw):
    a = dict(q=t(3, 8, 5, 64), kDraft=t(3, 2, 5, 64), vDraft=t(3, 2, 5, 64), kCache=t(3, 2, 90, 64), vCache=t(3, 2, 90, 64), kvLens=ints(3),
             treeMask=t(3, 5, 5, dtype=torch.bool))
    a.update({n: f() if callable(f) else f for n, f in kw.items()})
    return a


@pytest.mark.parametrize("kw", [
    dict(q=lambda: t(3, 8, 5, 64, device="cpu")), dict(q=lambda: t(3, 8, 64)), dict(kDraft=lambda: t(3, 2, 4, 64)), dict(vDraft=lambda: t(3, 2, 6, 64)),
    dict(kDraft=lambda: t(3, 4, 5, 64)), dict(kDraft=lambda: t(2, 2, 5, 64)), dict(vDraft=lambda: t(3, 2, 5, 64, dtype=torch.float16)),
    dict(kCache=lambda: t(2, 2, 90, 64)), dict(vCache=lambda: t(3, 2, 89, 64)), dict(kCache=lambda: t(3, 2, 90, 128)), dict(kCache=lambda: t(3, 2, 64, 90).transpose(2, 3)),
    dict(kvLens=lambda: ints(2)), dict(kvLens=lambda: ints(3, dtype=torch.int64)), dict(treeMask=lambda: t(3, 5, 5)), dict(treeMask=lambda: t(3, 4, 5, dtype=torch.bool)),
    dict(treeMask=lambda: t(2, 5, 5, dtype=torch.bool)), dict(treeMask=lambda: t(3, 1, 5, 5, dtype=torch.bool)), dict(treeMask=lambda: t(5, 5, dtype=torch.bool, device="cpu")),
    dict(workspace=lambda: t(99, device="cpu")), dict(status=lambda: ints(0)),
])
def test_tree_refuses(fake, kw):
    with pytest.raises(ValueError):
        op.sdpAttentionTree(**tree_args(**kw))


def accept_args(**kw):
    a = dict(kDraft=t(3, 2, 5, 64), vDraft=t(3, 2, 5, 64), kCache=t(3, 2, 90, 64), vCache=t(3, 2, 90, 64), kvLens=ints(3), path=ints(3, 4), counts=ints(3))
    a.update({n: f() if callable(f) else f for n, f in kw.items()})
    return a


@pytest.mark.parametrize("kw", [
    dict(kDraft=lambda: t(3, 4, 5, 64)), dict(vDraft=lambda: t(3, 2, 4, 64)), dict(kCache=lambda: t(2, 2, 90, 64)), dict(vCache=lambda: t(3, 2, 91, 64)),
    dict(kvLens=lambda: ints(2)), dict(kvLens=lambda: ints(3, device="cpu")), dict(counts=lambda: ints(4)), dict(counts=lambda: ints(3, dtype=torch.int64)),
    dict(path=lambda: ints(2, 4)), dict(path=lambda: ints(3)), dict(path=lambda: ints(3, 8)[:, ::2]), dict(path=lambda: ints(3, 4, device="cpu")),
    dict(kCache=lambda: t(1, 2, 90, 64).expand(3, -1, -1, -1)), dict(vCache=lambda: t(3, 1, 90, 64).expand(-1, 2, -1, -1)),
])
def test_accept_refuses(fake, kw):
    with pytest.raises(ValueError):
        op.cacheAccept(**accept_args(**kw))


def test_accept_refuses_drafts_that_lie_in_the_cache(fake):
    c = t(3, 2, 90, 64)
    with pytest.raises(ValueError, match="memory"):
        op.cacheAccept(**accept_args(kCache=c, kDraft=c[:, :, 80:85]))


def tree_params(cls, **kw):
    p = cls()
    p.struct_size = C.sizeof(p)
    p.dtype, p.B, p.Hkv, p.T, p.capacity, p.D = 2, 3, 2, 5, 90, 64
    p.k_draft = p.v_draft = p.k = p.v = 0x1000
    if cls is _capi.TreeParams:
        p.Hq, p.q, p.o = 8, 0x1000, 0x1000
    else:
        p.N, p.kv_lens, p.path, p.counts, p.new_lens = 4, 0x1000, 0x1000, 0x1000, 0x2000
    for n, v in kw.items():
        setattr(p, n, v)
    return C.byref(p)


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), -8), (dict(dtype=3), -2), (dict(B=0), -3), (dict(T=0), -3), (dict(capacity=0), -3), (dict(D=96), -4), (dict(k_draft=None), -1),
    (dict(v=0x1008), -5), (dict(k_strides=_capi.Strides(0, 64, 60)), -5), (dict(B=70000), -10),
])
def test_tree_and_accept_abi(kw, code):
    lib = _capi.lib()
    assert lib.tt_attn_tree(tree_params(_capi.TreeParams, **kw)) == code
    assert lib.tt_attn_cache_accept(tree_params(_capi.CacheAcceptParams, **kw)) == code
    assert lib.tt_attn_tree(None) == -1 and lib.tt_attn_cache_accept(None) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(T=129), -10), (dict(Hq=258), -10), (dict(dtype=0, Hq=66), -10), (dict(Hq=9), -3), (dict(q=None), -1), (dict(o=0x1004), -5),
    (dict(mask=0x1000, mask_strides=(C.c_int64 * 2)(-1, 5)), -3), (dict(B=60000, capacity=2 ** 31 - 200), -10),
])
def test_tree_abi(kw, code):
    assert _capi.lib().tt_attn_tree(tree_params(_capi.TreeParams, **kw)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(N=-1), -3), (dict(path=None), -1), (dict(counts=None), -1), (dict(new_lens=0x1000), -3), (dict(N=2 ** 30), -10),
    (dict(k_strides=_capi.Strides(0, 128, 64)), -3), (dict(v_strides=_capi.Strides(11520, 0, 64)), -3),
])
def test_accept_abi(kw, code):
    assert _capi.lib().tt_attn_cache_accept(tree_params(_capi.CacheAcceptParams, **kw)) == code


def test_tree_workspace():
    """Two partial results of 128 rows for each of up to 148 CTAs, and a line for each."""
    w = _capi.lib().tt_attn_tree_workspace_bytes
    assert w(2, 32, 32, 8, 32, 8192, 128) == 148 * 2 * 128 * 130 * 4 + 2560
    assert 0 < w(2, 1, 1, 1, 1, 1, 64) <= 256 + 8 * 2 * 128 * 66 * 4  # (a piece for every two tiles, or what counts as tiles)
    assert w(2, 1, 1, 1, 129, 1, 64) == 0 and w(0, 1, 64, 1, 1, 1, 64) == 0 and w(2, 0, 1, 1, 1, 1, 64) == 0
