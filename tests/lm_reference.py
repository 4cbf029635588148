"""Plain 64-bit forms of the operators around attention, with bounds on how far a 16- or 32-bit kernel may be off (test
infrastructure; runs on any device)."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}  # half of the smallest step


def within(got, want, bound, what=""):
    """|got - want| <= bound element by element; prints the largest share of the bound."""
    got, want, bound = got.detach().double(), want.double().to(got.device), bound.double().to(got.device)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    assert bool(torch.isfinite(got).all()), what + ": not finite"
    share = ((got - want).abs() / bound.clamp(min=1e-300)).max().item()
    print("%s: %.3f of the bound, largest error %.2e" % (what, share, (got - want).abs().max().item()))
    assert share <= 1.0, "%s: %.3f times the bound" % (what, share)


# ------------------------------------------------------------------------------------------ norm and rotation --
def turn(x, cos, sin, interleaved):
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    c, d = a * cos - b * sin, b * cos + a * sin
    return torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)


def angles(cos, sin, positions, sections, dims):
    """cos, sin of every row and pair, beside x [B, H, S, D] (dims 4) or [T, H, D] (dims 3); rows outside the tables: 1, 0."""
    half = cos.shape[1]
    pos = positions.long() if sections is not None else positions.long()[None]
    axis = torch.cat([torch.full((n,), a) for a, n in enumerate(sections or [half])]).to(pos.device)
    at = pos.movedim(0, -1)[..., axis]  # [.., S, half]
    inside = (at >= 0) & (at < cos.shape[0])
    at = at.clamp(0, cos.shape[0] - 1)
    pair = torch.arange(half, device=pos.device)
    c = torch.where(inside, cos.double()[at, pair], 1.0)
    s = torch.where(inside, sin.double()[at, pair], 0.0)
    if dims == 4:
        c, s = (x if x.dim() == 3 else x[None] for x in (c, s))
        return c[:, None], s[:, None]
    return c[:, None], s[:, None]


def norm_rope(x, w, cs, eps, interleaved):
    """One operand, 64 bits, differentiable: x [.., D], w [D] or None, cs = (cos, sin) beside x, or None."""
    y = x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    return y if cs is None else turn(y, cs[0], cs[1], interleaved)


def pair_size(x, interleaved):
    """|a| + |b| of the pair that a channel belongs to."""
    x, half = x.abs(), x.shape[-1] // 2
    s = x[..., 0::2] + x[..., 1::2] if interleaved else x[..., :half] + x[..., half:]
    return torch.stack((s, s), -1).flatten(-2) if interleaved else torch.cat((s, s), -1)


def norm_rope_check(got, x, w, cs, eps, interleaved, dtype, what):
    """fp32 arithmetic: the mean of squares, a sum of D terms in chains of 16 and a tree, is off by less than 24 steps of 2^-24, half of
    it reaches y; with the root's, the products' and the rotation's own roundings less than 32 steps of |a| + |b| of a pair.  Then one rounding."""
    want = norm_rope(x, w, cs, eps, interleaved)
    size = pair_size(norm_rope(x, w, None, eps, interleaved), interleaved)
    within(got, want, HALF[dtype] * want.abs() * (1 + 2 ** -7) + 32 * 2.0 ** -24 * size + TINY[dtype], what)


def norm_rope_grads_check(dx, dw, g, x, w, cs, eps, interleaved, dtype, what):
    """dx = r (u w - n mean(u w n)): less than 64 steps of 2^-24 of r (|u w| + |n| mean |u w n|), u being off by three steps of its pair's size.
    dw: a sum over rows, in chains no longer than the rows of one warp's lanes (here: all rows / 8) and a tree of less than 32, and
    a row's n is off by 16 steps."""
    D = x.shape[-1]
    u = g if cs is None else turn(g, cs[0], -cs[1], interleaved)
    size = u.abs() if cs is None else pair_size(g, interleaved)
    if w is None:
        if dx is not None:
            within(dx, u, HALF[dtype] * u.abs() * (1 + 2 ** -7) + 4 * 2.0 ** -24 * size + TINY[dtype], what + " dx")
        return
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r
    if dx is not None:
        t = u * w
        want = r * (t - n * (t * n).mean(-1, keepdim=True))
        s = size * w.abs()
        amp = r * (s + n.abs() * (s * n.abs()).mean(-1, keepdim=True))
        within(dx, want, HALF[dtype] * want.abs() * (1 + 2 ** -7) + 64 * 2.0 ** -24 * amp + TINY[dtype], what + " dx")
    if dw is not None:
        want = (u * n).reshape(-1, D).sum(0)
        amp = (size * n.abs()).reshape(-1, D).sum(0)
        within(dw, want, HALF[dtype] * want.abs() * (1 + 2 ** -7) + (48 + x.numel() // D / 8) * 2.0 ** -24 * amp + TINY[dtype], what + " dw")


# ------------------------------------------------------------------------------------------------- attention --
# What a 16-bit kernel may add besides roundings: exponentials (ex2: 2^-22; a cubic on the FMA pipe: 7.5e-5), scores summed in fp32 (D = 128
# products of size 3: 1e-4 in the exponent), for a probability and for the sum it is divided by.
SLOP = 5e-4


def visible(lq, lk, causal, device):
    i, j = torch.arange(lq, device=device)[:, None], torch.arange(lk, device=device)
    if causal == "bottom-right":
        return j <= i + (lk - lq)
    return j <= i if causal else torch.ones(lq, lk, dtype=torch.bool, device=device)


def attention(q, k, v, scale, sees):
    """64 bits, one kv head: q [G, L, D], k, v [S, D], sees [L, S] -> (O, LSE, P); rows that see nothing: 0, -inf, 0."""
    x = (q @ k.t()) * scale
    x = x.masked_fill(~sees, -math.inf)
    m = x.amax(-1, keepdim=True) if k.shape[0] else torch.full((*q.shape[:2], 1), -math.inf, dtype=q.dtype, device=q.device)
    e = torch.exp(x - m.masked_fill(m == -math.inf, 0.0)).masked_fill(~sees, 0.0)
    l = e.sum(-1, keepdim=True)
    p = e / l.masked_fill(l == 0, 1.0)
    return p @ v, (m + torch.log(l))[..., 0], p


def attention_bound(p, v, o, dtype):
    """P is rounded to the tensor type before the product, the result once more."""
    h = HALF[dtype]
    return (h + SLOP) * (p @ v.abs()) * (1 + 2 ** -6) + (h + SLOP) * o.abs() + TINY[dtype] * (2 + 2 * v.abs().sum(0))


def attention_grads(q, k, v, o, do, p, scale, dtype):
    """((dQ, bound), (dK, bound), (dV, bound)) of one kv head; the bounds count the roundings of P and dS to the tensor type, of O in
    delta, and of the results."""
    h = HALF[dtype]
    dp = do @ v.t()
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
    bo = attention_bound(p, v, o, dtype)
    e_ds = p * abs(scale) * ((do.abs() * bo).sum(-1, keepdim=True) + (do.abs() @ v.abs().t()) * SLOP) + (h + SLOP) * ds.abs() + TINY[dtype]
    dq, dk, dv = ds @ k, (ds.transpose(1, 2) @ q).sum(0), (p.transpose(1, 2) @ do).sum(0)
    bq = e_ds @ k.abs() + 2 * h * dq.abs() + 2 * TINY[dtype]
    bk = (e_ds.transpose(1, 2) @ q.abs()).sum(0) + 2 * h * dk.abs() + 2 * TINY[dtype]
    bv = (((h + SLOP) * p + TINY[dtype]).transpose(1, 2) @ do.abs()).sum(0) * (1 + 2 ** -6) + 2 * h * dv.abs() + 2 * TINY[dtype]
    return (dq, bq), (dk, bk), (dv, bv)


def at_the_end(x, size=32 << 20):
    """A copy of x that ends where its memory does: what is read behind it is not mapped, as a rule."""
    block = torch.empty(size, dtype=torch.uint8, device=x.device)
    y = block[size - x.numel() * x.element_size():].view(x.dtype).view(x.shape)
    return y.copy_(x)
