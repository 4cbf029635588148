"""What attention gives for operands that are not finite, in 64 bits, and how a kernel's result is compared with it (test infrastructure).

A row whose softmax is over a NaN, or over +inf (inf - inf), is NaN in all of O and in LSE; a score of -inf is a probability of 0."""
import math

import torch

import lm_reference as ref

POISON = [(math.nan, "one"), (math.nan, "all"), (math.inf, "one"), (-math.inf, "one")]


def poison(x, at, value, where):
    """A copy of x with `value` in the row `at`, in one of its channels (the one that the largest of a few random rows has) or all of them."""
    x = x.clone()
    x[at][..., 5 if where == "one" else slice(None)] = value
    return x


def attention(q, k, v, scale, sees, added=None):
    """64 bits, [.., L, D], [.., S, D] and sees [.., L, S] -> O, LSE, P; rows that see nothing: 0, -inf, 0."""
    x = (q @ k.transpose(-1, -2)) * scale
    if added is not None:
        x = x + added
    x = x.masked_fill(~sees, -math.inf)
    m = x.amax(-1, keepdim=True)  # (NaN where there is one)
    empty = ~sees.any(-1, keepdim=True)
    e = torch.exp(x - m.masked_fill(empty, 0.0)).masked_fill(~sees, 0.0)
    l = e.sum(-1, keepdim=True)
    p = e / l.masked_fill(empty, 1.0)
    return p @ v, (m + torch.log(l))[..., 0].masked_fill(empty[..., 0], -math.inf), p


def agree(o, lse, want, want_lse, p, v, dtype):
    """NaN where the 64-bit form is NaN and nowhere else, infinities likewise; the finite elements within the roundings of P and of the result (32 bits: 2^-12
    of the sizes, far from any error of a key that is lost)."""
    o, want = o.double(), want.to(o.device)
    for name, a, b in (("O", o, want), ("LSE", lse.double(), want_lse)):
        assert torch.equal(a.isnan(), b.isnan()), "%s is NaN in %d elements, not %d" % (name, a.isnan().sum(), b.isnan().sum())
        assert torch.equal(a.isinf(), b.isinf()) and torch.equal(a[a.isinf()], b[b.isinf()]), name
    fine = want.isfinite()
    size = torch.nan_to_num(p, 0.0) @ v.nan_to_num(0.0, 0.0, 0.0).abs()
    h = ref.HALF[dtype] + ref.SLOP if dtype != torch.float32 else 2.0 ** -12
    bound = h * (1 + 2.0 ** -6) * (size + torch.nan_to_num(want, 0.0, 0.0, 0.0).abs()) + 4 * ref.TINY[dtype] * (1 + v.nan_to_num(0.0, 0.0, 0.0).abs().sum(-2, keepdim=True))
    assert bool(((o - want).abs() <= bound)[fine].all()), "finite rows"
    some = want_lse.isfinite()
    assert bool(((lse.double() - want_lse).abs() <= ref.SLOP + 2.0 ** -20 * want_lse.abs())[some].all()), "LSE"
