"""CPU: operands whose rows share memory (a tensor expanded over its rows) are refused, not read as dense ones: three strides of zero
mean a dense tensor to the C ABI, and the kernels would read as much memory as one has.

Fake CUDA tensors, as in test_lm_arguments_cpu.py: a call that is let through fails on the missing driver, with another error."""
import os

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from conftest import ROOT
from tinytorch_b200 import function, op


@pytest.fixture(autouse=True)
def fake():
    if not os.path.exists(os.path.join(ROOT, "tinytorch_b200", "lib", "_native.so")):
        from tinytorch_b200.build import build, build_native
        build()
        build_native()
    with FakeTensorMode():
        yield


def t(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def ints(*shape):
    return t(*shape, dtype=torch.int32)


def all_rows(x, rows):
    """One row for all of a tensor, and one for the rows of each of its other dimensions."""
    one = x[(0,) * (x.dim() - 1)].view([1] * (x.dim() - 1) + [-1]).expand(x.shape)
    part = x.narrow(rows, 0, 1).expand(x.shape)
    assert not any(one.stride()[:-1]) and part.stride(rows) == 0 and any(part.stride()[:-1])
    return one, part


def refused(call, args, names, rows):
    for name in names:
        for x in all_rows(args[name], rows):
            with pytest.raises(ValueError, match="own memory"):
                call(**dict(args, **{name: x}))


DENSE = dict(query=(2, 8, 40, 64), key=(2, 4, 50, 64), value=(2, 4, 50, 64))


def test_attention():
    a = {n: t(*s) for n, s in DENSE.items()}
    refused(function.sdpAttention, a, a, 2)
    refused(op.sdpAttentionFwd, dict(zip("qkv", a.values())), "qkv", 2)
    b = dict(dO=t(2, 8, 40, 64), q=a["query"], k=a["key"], v=a["value"], o=t(2, 8, 40, 64), lse=t(2, 8, 40, dtype=torch.float32))
    refused(op.sdpAttentionBwd, b, ("dO", "q", "k", "v", "o"), 2)


def test_caches():
    a = dict(q=t(2, 8, 1, 64), kCache=t(2, 4, 50, 64), vCache=t(2, 4, 50, 64))
    refused(op.sdpAttentionDecode, a, ("kCache", "vCache"), 2)
    a.update(kNew=t(2, 4, 1, 64), vNew=t(2, 4, 1, 64), kvLens=ints(2))
    refused(op.sdpAttentionDecodeAppend, a, ("kCache", "vCache"), 2)


@pytest.mark.parametrize("separate", [False, True])
def test_packed(separate):
    a = dict(query=t(40, 8, 64), key=t(40, 4, 64), value=t(40, 4, 64), cuSeqlens=ints(3))
    if separate:
        a.update(key=t(90, 4, 64), value=t(90, 4, 64), cuSeqlensK=ints(3))
    refused(function.sdpAttentionPacked, a, ("query", "key", "value"), 0)
    b = dict(q=a["query"], k=a["key"], v=a["value"], cuSeqlens=ints(3), cuSeqlensK=a.get("cuSeqlensK"))
    refused(op.sdpAttentionPackedFwd, b, "qkv", 0)
    b.update(dO=t(40, 8, 64), o=t(40, 8, 64), lse=t(8, 40, dtype=torch.float32))
    refused(op.sdpAttentionPackedBwd, b, ("q", "k", "v", "o"), 0)


def test_trees_and_what_is_accepted():
    drafts, caches = (2, 4, 5, 64), (2, 4, 90, 64)
    a = dict(q=t(2, 8, 5, 64), kDraft=t(*drafts), vDraft=t(*drafts), kCache=t(*caches), vCache=t(*caches))
    refused(op.sdpAttentionTree, a, a, 2)
    del a["q"]
    a.update(kvLens=ints(2), path=ints(2, 3), counts=ints(2))
    refused(op.cacheAccept, a, ("kDraft", "vDraft", "kCache", "vCache"), 2)
