"""Performance cases of the operators around attention in a language model's layer: what a model does to its queries and
keys before attention, attention over prompts of different lengths packed behind one another, and a serving step that
verifies drafted tokens.

Four operators ("op" of a case):
  norm_rope  fused.qkNormRope: the RMS norm of every head of q and k and the rotation to their positions, in one pass;
             alone (serving) or with its gradients (training)
  packed     function.sdpAttentionPacked: attention over packed sequences; alone (a batch of prompts) or with gradients
  tree       op.sdpAttentionTree: a tree of drafted tokens of each sequence against its cache and its own ancestors
  accept     op.cacheAccept: the accepted drafts' keys and values go behind the cache's rows
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # one decoding step of 16 sequences of a grouped-query model: what a launch costs
        dict(name="norm_rope_step", op="norm_rope", dtype="bfloat16", layout="packed", batch=1, tokens=16, Hq=32, Hkv=8, D=128,
             axes=1, interleaved=False, grad=False),
        # prompts of 8200 tokens in all, packed, from the projection's output
        dict(name="norm_rope_prompt", op="norm_rope", dtype="bfloat16", layout="packed", batch=1, tokens=8200, Hq=32, Hkv=8,
             D=128, axes=1, interleaved=False, grad=False),
        # a training step over images and text: positions of three axes (time, height, width), forward and gradients
        dict(name="norm_rope_axes_train", op="norm_rope", dtype="float16", layout="batched", batch=4, tokens=2048, Hq=16, Hkv=16,
             D=64, axes=3, interleaved=False, grad=True),
        # a few short prompts that arrived together: how soon their first tokens come
        dict(name="packed_short", op="packed", dtype="bfloat16", lengths="37,128,1,300,211", tail=0, Hq=32, Hkv=8, D=128,
             causal=True, grad=False),
        # a prefill batch of a grouped-query model, requests of very different lengths, with room behind the last
        dict(name="packed_prompts", op="packed", dtype="bfloat16",
             lengths="4096,1500,777,3333,2048,64,513,900,1,1200,129,1823", tail=100, Hq=32, Hkv=8, D=128, causal=True, grad=False),
        # a training step on packed documents, grouped heads
        dict(name="packed_train", op="packed", dtype="bfloat16", lengths="3000,1024,700,2048,255,1165", tail=0, Hq=32, Hkv=8,
             D=128, causal=True, grad=True),
        # a training step on packed documents of a model without grouped heads, head dimension 64
        dict(name="packed_train_d64", op="packed", dtype="float16", lengths="2048,2048,1000,3096,517,1531,640,1360", tail=48,
             Hq=16, Hkv=16, D=64, causal=True, grad=True),
        # one user's sequence and a small tree of drafts: a step's latency
        dict(name="tree_single", op="tree", dtype="bfloat16", B=1, drafts=8, shortest=2000, longest=2000, capacity=4096, Hq=32,
             Hkv=8, D=128, mask=True),
        # 32 sequences of a server with trees of 32 drafts over caches of different lengths
        dict(name="tree_batch", op="tree", dtype="bfloat16", B=32, drafts=32, shortest=1000, longest=8160, capacity=8192, Hq=32,
             Hkv=8, D=128, mask=True),
        # a single-precision model without grouped heads, a chain of drafts
        dict(name="tree_f32", op="tree", dtype="float32", B=4, drafts=5, shortest=500, longest=1003, capacity=1024, Hq=16,
             Hkv=16, D=64, mask=False),
        # one sequence accepts a path of its tree
        dict(name="accept_single", op="accept", dtype="bfloat16", B=1, drafts=8, path=5, capacity=4096, Hkv=8, D=128),
        # 64 sequences accept paths of different lengths
        dict(name="accept_batch", op="accept", dtype="bfloat16", B=64, drafts=64, path=12, capacity=1000, Hkv=8, D=128),
    ]


# ------------------------------------------------------------------------------------------------ drawn cases --
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    """Query and key heads."""
    return rng.choice([(32, 8), (16, 16), (8, 1), (12, 4), (28, 4), (8, 8), (6, 2), (40, 8), (24, 8), (5, 5)])


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / (1.4e15 if case["dtype"] != "float32" else 5e13)


def _draw(rng):
    op = rng.choice(["norm_rope", "packed", "packed", "tree", "tree", "accept"])
    half = rng.choice(["float16", "bfloat16"])
    Hq, Hkv = _heads(rng)
    D = rng.choice([64, 128])
    if op == "norm_rope":
        tokens = _log(rng, 1, 20000)
        batch = rng.choice([b for b in (1, 2, 3, 4, 7) if b <= tokens])
        return dict(op=op, dtype=rng.choice(["float32", half, half]), layout=rng.choice(["packed", "batched"]), batch=batch,
                    tokens=tokens // batch, Hq=Hq, Hkv=Hkv, D=D, axes=rng.choice([1, 1, 2, 3]),
                    interleaved=rng.random() < 0.3, grad=rng.random() < 0.5)
    if op == "packed":
        n = _log(rng, 1, 40)
        longest = _log(rng, 1, 4096)
        lengths = [_log(rng, 1, longest) for _ in range(n)]
        return dict(op=op, dtype=half, lengths=",".join(map(str, lengths)), tail=rng.choice([0, 0, 1, 77]), Hq=Hq, Hkv=Hkv, D=D,
                    causal=rng.random() < 0.8, grad=rng.random() < 0.5)
    drafts = _log(rng, 1, 128 if op == "accept" else 100)
    if op == "tree":
        longest = _log(rng, 1, 20000)
        return dict(op=op, dtype=rng.choice(["float32", half, half, half]), B=_log(rng, 1, 48), drafts=drafts,
                    shortest=rng.randint(0, longest), longest=longest, capacity=longest + rng.choice([0, 1, 100]), Hq=Hq, Hkv=Hkv,
                    D=D, mask=rng.random() < 0.8)
    return dict(op=op, dtype=rng.choice(["float32", half, half]), B=_log(rng, 1, 100), drafts=drafts, path=rng.randint(1, min(drafts, 20)),
                capacity=_log(rng, 200, 2000), Hkv=Hkv, D=D)


def draw(rng):
    """One more case of the ranges above, no dearer than the dearest listed one of its operator."""
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _cost(c))
    while True:
        case = _draw(rng)
        # (an accept's caches are an output, and are compared whole)
        if _cost(case) <= most[case["op"]] and (case["op"] != "accept" or case["B"] * case["capacity"] * case["Hkv"] <= 1 << 19):
            return case


# ------------------------------------------------------------------------------------------------------ inputs --
def _lengths(case):
    return [int(x) for x in case["lengths"].split(",")]


def _cache_lens(case):
    B = case["B"]
    lo, hi = case["shortest"], case["longest"]
    return [hi - (hi - lo) * b // max(1, B - 1) for b in range(B)]


def _sections(case):
    """Pairs of channels of each axis: the first axis has what the others leave."""
    half, axes = case["D"] // 2, case["axes"]
    rest = [half * 3 // 8] * (axes - 1)
    return [half - sum(rest)] + rest


def _tables(positions, D, dev):
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
    ang = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * inv
    return ang.cos().float().contiguous(), ang.sin().float().contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(dt)

    s = dict(case=case)
    if case["op"] == "norm_rope":
        B, S, Hq, Hkv, D = case["batch"], case["tokens"], case["Hq"], case["Hkv"], case["D"]
        # q and k are parts of the projection's output, token by token
        qkv = randn(B, S, Hq + 2 * Hkv, D)
        q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
        base = torch.randint(0, 3000, (B, 1), generator=g, device=dev, dtype=torch.int32)
        step = torch.arange(S, device=dev, dtype=torch.int32)
        # text moves all axes alike; of an image, the second and third go over its rows and columns
        pos = torch.stack([base + step // (1, 1, 32)[a] % (1 << 30, 64, 64)[a] for a in range(case["axes"])])
        gq, gk = randn(B, S, Hq, D), randn(B, S, Hkv, D)
        if case["layout"] == "packed":
            q, k, gq, gk = (x.flatten(0, 1) for x in (q, k, gq, gk))
            pos = pos.reshape(case["axes"], -1)
        else:
            q, k, gq, gk = (x.transpose(1, 2) for x in (q, k, gq, gk))
        s.update(q=q, k=k, wq=1 + 0.2 * randn(D), wk=1 + 0.2 * randn(D), gq=gq, gk=gk,
                 pos=pos.contiguous() if case["axes"] > 1 else pos[0].contiguous(), sections=_sections(case) if case["axes"] > 1 else None)
        s["cos"], s["sin"] = _tables(3000 + S, D, dev)
        if case["grad"]:
            for n in ("q", "k", "wq", "wk"):
                s[n] = s[n].detach().requires_grad_()
    elif case["op"] == "packed":
        lens = _lengths(case)
        T, Hq, Hkv, D = sum(lens) + case["tail"], case["Hq"], case["Hkv"], case["D"]
        s.update(q=randn(T, Hq, D), k=randn(T, Hkv, D), v=randn(T, Hkv, D), g=randn(T, Hq, D))
        s["cu"] = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)
        if case["grad"]:
            for n in "qkv":
                s[n].requires_grad_()
    elif case["op"] == "tree":
        B, T, Hq, Hkv, D, cap = case["B"], case["drafts"], case["Hq"], case["Hkv"], case["D"], case["capacity"]
        s.update(q=randn(B, Hq, T, D), kd=randn(B, Hkv, T, D), vd=randn(B, Hkv, T, D), kc=randn(B, Hkv, cap, D), vc=randn(B, Hkv, cap, D))
        s["lens"] = torch.tensor(_cache_lens(case), dtype=torch.int32, device=dev)
        s["mask"] = None
        if case["mask"]:
            # every draft's parent is an earlier one, or the sequence's last token
            parent = (torch.rand(B, T, generator=g, device=dev) * (torch.arange(T, device=dev) + 1)).long() - 1
            m = torch.eye(T, dtype=torch.bool, device=dev).repeat(B, 1, 1)
            every = torch.arange(B, device=dev)
            for i in range(1, T):
                m[:, i] |= m[every, parent[:, i].clamp(min=0)] & (parent[:, i] >= 0)[:, None]
            s["mask"] = m
    else:
        B, T, Hkv, D, cap, n = case["B"], case["drafts"], case["Hkv"], case["D"], case["capacity"], case["path"]
        s.update(kd=randn(B, Hkv, T, D), vd=randn(B, Hkv, T, D), kc=randn(B, Hkv, cap, D), vc=randn(B, Hkv, cap, D))
        # paths go from ancestors to descendants
        s["path"] = torch.rand(B, T, generator=g, device=dev).argsort(1)[:, :n].sort(1)[0].to(torch.int32).contiguous()
        s["counts"] = torch.randint(0, n + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        s["lens"] = torch.randint(0, cap - n + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    return s


# ------------------------------------------------------------------------------------------------- plain forms --
def _by_token(x):
    """[B, H, S, D] as [B, S, H, D]; packed rows [T, H, D] as they are."""
    return x.transpose(1, 2) if x.dim() == 4 else x


def _norm_rope_plain(s):
    case = s["case"]
    D, half = case["D"], case["D"] // 2
    pos, axes = s["pos"].long(), case["axes"]
    if axes == 1:
        cos, sin = s["cos"][pos], s["sin"][pos]
    else:
        axis = torch.repeat_interleave(torch.arange(axes, device=pos.device), torch.tensor(s["sections"], device=pos.device))
        at = pos.movedim(0, -1)[..., axis]  # [.., half]: the position of every pair
        pair = torch.arange(half, device=pos.device)
        cos, sin = s["cos"][at, pair], s["sin"][at, pair]
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)  # beside [.., heads, half]
    out, grads = [], []
    for x, w, g in ((s["q"], s["wq"], s["gq"]), (s["k"], s["wk"], s["gk"])):
        x, wf = _by_token(x.detach()).float(), w.detach().float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        n = x * r
        y = n * wf
        lo, hi = (y[..., 0::2], y[..., 1::2]) if case["interleaved"] else (y[..., :half], y[..., half:])
        a, b = lo * cos - hi * sin, hi * cos + lo * sin
        z = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
        out.append(_by_token(z.to(w.dtype)))
        if case["grad"]:
            g = _by_token(g).float()
            lo, hi = (g[..., 0::2], g[..., 1::2]) if case["interleaved"] else (g[..., :half], g[..., half:])
            a, b = lo * cos + hi * sin, hi * cos - lo * sin
            u = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
            dw = (u * n).flatten(0, -2).sum(0, dtype=torch.float64)
            u = u * wf
            dx = r * (u - n * (u * n).mean(-1, keepdim=True))
            grads += [_by_token(dx.to(w.dtype)), dw.to(w.dtype)]
    return out + grads


def _packed_plain(s):
    case = s["case"]
    q, k, v = s["q"].detach(), s["k"].detach(), s["v"].detach()
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    group, scale = Hq // Hkv, 1.0 / math.sqrt(D)
    o = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if case["grad"] else []
    at = 0
    for n in _lengths(case):
        rows = slice(at, at + n)
        at += n
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1) if case["causal"] else None
        for h in range(Hkv):  # (a head's group at a time: the scores of all heads of a long sequence would be large)
            heads = slice(h * group, (h + 1) * group)
            qf = q[rows, heads].float().transpose(0, 1)
            kf, vf = k[rows, h].float(), v[rows, h].float()
            x = (qf @ kf.t()) * scale
            if hidden is not None:
                x = x.masked_fill(hidden, -math.inf)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            of = p @ vf
            o[rows, heads] = of.transpose(0, 1).to(o.dtype)
            if grads:
                gf = s["g"][rows, heads].float().transpose(0, 1)
                dp = gf @ vf.t()
                ds = p * (dp - (gf * of).sum(-1, keepdim=True)) * scale
                grads[0][rows, heads] = (ds @ kf).transpose(0, 1).to(o.dtype)
                grads[1][rows, h] = (ds.transpose(1, 2) @ qf).sum(0).to(o.dtype)
                grads[2][rows, h] = (p.transpose(1, 2) @ gf).sum(0).to(o.dtype)
    return [o] + grads


def _tree_plain(s):
    case = s["case"]
    q = s["q"]
    B, Hq, T, D = q.shape
    Hkv = case["Hkv"]
    o, lse = torch.empty_like(q), torch.empty(B, Hq, T, device=q.device)
    chain = torch.ones(T, T, dtype=torch.bool, device=q.device).tril()
    for b, n in enumerate(_cache_lens(case)):
        kf = torch.cat((s["kc"][b, :, :n], s["kd"][b]), 1).float()
        vf = torch.cat((s["vc"][b, :, :n], s["vd"][b]), 1).float()
        x = (q[b].float().reshape(Hkv, -1, D) @ kf.transpose(1, 2)).reshape(Hq, T, -1) / math.sqrt(D)
        sees = chain if s["mask"] is None else s["mask"][b]
        x[:, :, n:] = x[:, :, n:].masked_fill(~sees, -math.inf)
        m = x.amax(-1, keepdim=True)
        p = torch.exp(x - m)
        l = p.sum(-1, keepdim=True)
        o[b] = ((p / l).reshape(Hkv, -1, n + T) @ vf).reshape(Hq, T, D).to(o.dtype)
        lse[b] = (m + torch.log(l))[..., 0]
    return [o, lse]


def _accept_plain(s):
    rank = torch.arange(s["path"].shape[1], device=s["path"].device)
    b, i = (rank < s["counts"][:, None]).nonzero(as_tuple=True)
    row, src = s["lens"].long()[b] + i, s["path"].long()[b, i]
    s["kc"][b, :, row] = s["kd"][b, :, src]
    s["vc"][b, :, row] = s["vd"][b, :, src]
    return [s["kc"], s["vc"], s["lens"] + s["counts"]]


# ---------------------------------------------------------------------------------------------------- one pass --
def _run_own(s):
    from tinytorch_b200 import function, fused, op as ops
    case = s["case"]
    if case["op"] == "norm_rope":
        out = fused.qkNormRope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["pos"], eps=1e-6,
                               interleaved=case["interleaved"], sections=s["sections"])
        if not case["grad"]:
            return list(out)
        dq, dk, dwq, dwk = torch.autograd.grad(out, (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
        return [out[0].detach(), out[1].detach(), dq, dwq, dk, dwk]
    if case["op"] == "packed":
        o = function.sdpAttentionPacked(s["q"], s["k"], s["v"], s["cu"], isCausal=case["causal"])
        return [o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["g"])] if case["grad"] else [o]
    if case["op"] == "tree":
        return list(ops.sdpAttentionTree(s["q"], s["kd"], s["vd"], s["kc"], s["vc"], s["lens"], s["mask"], needLse=True))
    return [s["kc"], s["vc"], ops.cacheAccept(s["kd"], s["vd"], s["kc"], s["vc"], s["lens"], s["path"], s["counts"])]


def run(state):
    if own:
        return _run_own(state)
    return {"norm_rope": _norm_rope_plain, "packed": _packed_plain, "tree": _tree_plain, "accept": _accept_plain}[state["case"]["op"]](state)


# -------------------------------------------------------------------------------------------------------- work --
def work(case):
    es = SIZE[case["dtype"]]
    if case["op"] == "norm_rope":
        rows = case["batch"] * case["tokens"]
        x = rows * (case["Hq"] + case["Hkv"]) * case["D"]
        # x in, y out (and for the gradients x and dy in, dx out); the angles of every token once
        return dict(bytes=x * es * (5 if case["grad"] else 2) + rows * case["D"] * 4, flops=x * (30 if case["grad"] else 10))
    if case["op"] == "packed":
        lens, Hq, Hkv, D = _lengths(case), case["Hq"], case["Hkv"], case["D"]
        T = sum(lens) + case["tail"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        # q, k, v in and o out; for the gradients q, k, v, o and dO in, dq, dk, dv out
        nbytes = T * (2 * Hq + 2 * Hkv) * D * es + (T * (4 * Hq + 4 * Hkv) * D * es if case["grad"] else 0)
        return dict(bytes=nbytes, flops=pairs * Hq * D * (14 if case["grad"] else 4))
    if case["op"] == "tree":
        B, T, Hq, Hkv, D = case["B"], case["drafts"], case["Hq"], case["Hkv"], case["D"]
        rows = sum(_cache_lens(case)) + B * T
        return dict(bytes=(rows * 2 * Hkv + 2 * B * T * Hq) * D * es + B * T * (T + 4 * Hq), flops=4 * D * Hq * T * rows)
    moved = case["B"] * case["path"] / 2 * case["Hkv"] * case["D"] * 2  # half of the longest path, as a rule
    return dict(bytes=int(2 * moved * es) + case["B"] * (4 * case["path"] + 12), flops=0)


# -------------------------------------------------------------------------------------- by definition, 64 bits --
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _norm_rope_exact, "packed": _packed_exact, "tree": _tree_exact, "accept": _accept_exact}[case["op"]](case, s)


def _norm_rope_exact(case, s):
    """The rotation as a product with cos + i sin, gradients by the chain rule over the whole tensor."""
    D = case["D"]
    pos = s["pos"].long() if case["axes"] > 1 else s["pos"].long()[None]
    at = torch.cat([pos[a][..., None].expand(*pos.shape[1:], n) for a, n in enumerate(s["sections"] or [D // 2])], -1)
    pair = torch.arange(D // 2, device=at.device).expand_as(at)
    turn = torch.complex(s["cos"].double()[at, pair], s["sin"].double()[at, pair])
    turn = turn[:, None]  # [T, 1, D / 2], or [B, 1, S, D / 2]: beside the heads

    def pairs(x):
        return torch.complex(x[..., 0::2], x[..., 1::2]) if case["interleaved"] else torch.complex(x[..., :D // 2], x[..., D // 2:])

    def flat(z):
        return torch.view_as_real(z.contiguous()).flatten(-2) if case["interleaved"] else torch.cat((z.real, z.imag), -1)

    outs, grads = [], []
    for x, w, g in ((s["q"], s["wq"], s["gq"]), (s["k"], s["wk"], s["gk"])):
        x, w = x.detach().double(), w.detach().double()
        size = (x.square().sum(-1, keepdim=True) / D + 1e-6).sqrt()
        outs.append(flat(pairs(x / size * w) * turn))
        if case["grad"]:
            u = flat(pairs(g.double()) * turn.conj())
            dw = (u * x / size).reshape(-1, D).sum(0) if x.dim() == 3 else (u * x / size).sum((0, 1, 2))
            t = u * w
            grads += [t / size - x * (t * x).sum(-1, keepdim=True) / (D * size ** 3), dw]
    return outs + grads


def _packed_exact(case, s):
    D = case["D"]
    q, k, v, g = (s[n].detach() for n in "qkvg")
    group = case["Hq"] // case["Hkv"]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device=q.device) for x in (q, k, v))
    ends = s["cu"].tolist()
    for a, e in zip(ends, ends[1:]):
        for h in range(case["Hq"]):
            qh, kh, vh, gh = q[a:e, h].double(), k[a:e, h // group].double(), v[a:e, h // group].double(), g[a:e, h].double()
            x = torch.mm(qh, kh.t()) / math.sqrt(D)
            if case["causal"]:
                i = torch.arange(e - a, device=x.device)
                x[i[:, None] < i] = -math.inf
            p = torch.softmax(x, -1)
            o[a:e, h] = torch.mm(p, vh)
            if case["grad"]:
                dv[a:e, h // group] += torch.mm(p.t(), gh)
                dp = torch.mm(gh, vh.t())
                ds = (p * dp - p * (p * dp).sum(1, keepdim=True)) / math.sqrt(D)
                dq[a:e, h] = torch.mm(ds, kh)
                dk[a:e, h // group] += torch.mm(ds.t(), qh)
    return [o, dq, dk, dv] if case["grad"] else [o]


def _tree_exact(case, s):
    q = s["q"]
    B, Hq, T, D = q.shape
    group = Hq // case["Hkv"]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(B, Hq, T, dtype=torch.float64, device=q.device)
    for b, n in enumerate(s["lens"].tolist()):
        see = torch.ones(T, n + T, dtype=torch.bool, device=q.device)
        see[:, n:] = torch.ones_like(see[:, n:]).tril() if s["mask"] is None else s["mask"][b]
        for h in range(case["Hkv"]):
            keys = torch.cat((s["kc"][b, h, :n], s["kd"][b, h])).double()
            values = torch.cat((s["vc"][b, h, :n], s["vd"][b, h])).double()
            x = torch.einsum("gtd,sd->gts", q[b, h * group:(h + 1) * group].double(), keys) / D ** 0.5
            x = torch.where(see, x, -math.inf)
            lse[b, h * group:(h + 1) * group] = torch.logsumexp(x, -1)
            o[b, h * group:(h + 1) * group] = torch.einsum("gts,sd->gtd", torch.softmax(x, -1), values)
    return [o, lse]


def _accept_exact(case, s):
    kc, vc = s["kc"].double(), s["vc"].double()
    new = []
    for b, (n, c) in enumerate(zip(s["lens"].tolist(), s["counts"].tolist())):
        for i, j in enumerate(s["path"][b, :c].tolist()):
            kc[b, :, n + i], vc[b, :, n + i] = s["kd"][b, :, j].double(), s["vd"][b, :, j].double()
        new.append(n + c)
    return [kc, vc, torch.tensor(new, device=kc.device)]
