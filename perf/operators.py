"""Measured cases of the block's attention stretch: the q/k norm with rotary
positions, attention, and both with their gradients.

``run`` computes the operators in plain fp32 torch operations, or, where
``own`` is true, through this package's entry points.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # q of the 1.3B video block at 480p, 81 frames: 21 x 30 x 52 latent tokens, 12 heads of 128 (inference)
        dict(name="norm_rope_32760x1536", op="rope", train=False, batch=1, tokens=32760, t=21, h=30, w=52, heads=12,
             dim=128, rope=True, half=False, dtype="bf16"),
        # q of the 14B block in training, a quarter of the tokens: forward and gradient
        dict(name="norm_rope_train_8190x5120", op="rope", train=True, batch=1, tokens=8190, t=21, h=15, w=26, heads=40,
             dim=128, rope=True, half=False, dtype="bf16"),
        # two samples of the 4096-wide video model in fp16, pairs split over the halves of a head
        dict(name="norm_rope_train_2x6144x4096", op="rope", train=True, batch=2, tokens=6144, t=16, h=16, w=24,
             heads=32, dim=128, rope=True, half=True, dtype="f16"),
        # the text keys of the cross-attention: norm alone, a call whose latency counts
        dict(name="norm_512x1536", op="rope", train=False, batch=1, tokens=512, t=1, h=1, w=512, heads=12, dim=128,
             rope=False, half=False, dtype="bf16"),
        # a padded batch of small clips in fp32: 3 x 7 x 9 tokens and 11 of padding, odd head count
        dict(name="norm_rope_train_2x200x320_f32", op="rope", train=True, batch=2, tokens=200, t=3, h=7, w=9, heads=5,
             dim=64, rope=True, half=False, dtype="f32"),
        # self-attention of the 1.3B block over all tokens of the clip (inference): the largest call
        dict(name="self_32760_h12", op="attn", train=False, batch=1, q=32760, k=32760, heads=12, kv_heads=12, dim=128,
             lengths=False, packed=False, dtype="bf16"),
        # its cross-attention: all tokens over 512 text tokens, of which a prompt fills a part
        dict(name="cross_32760x512_h12", op="attn", train=False, batch=1, q=32760, k=512, heads=12, kv_heads=12,
             dim=128, lengths=True, packed=False, dtype="bf16"),
        # one new row over a long context: few rows, many keys
        dict(name="one_row_32760_h12", op="attn", train=False, batch=1, q=1, k=32760, heads=12, kv_heads=12, dim=128,
             lengths=False, packed=False, dtype="bf16"),
        # training: self-attention of the 4096-wide model, two samples of 6144 tokens, q, k, v in one buffer
        dict(name="train_2x6144_h32", op="attn", train=True, batch=2, q=6144, k=6144, heads=32, kv_heads=32, dim=128,
             lengths=False, packed=True, dtype="bf16"),
        # training: cross-attention of the 14B block in fp16 with a prompt's length
        dict(name="train_cross_8190x512_h40_f16", op="attn", train=True, batch=1, q=8190, k=512, heads=40, kv_heads=40,
             dim=128, lengths=True, packed=False, dtype="f16"),
        # training: a ragged batch with shared key heads, one sample of it without any key
        dict(name="train_3x1285_h10_kv2_d64", op="attn", train=True, batch=3, q=1285, k=1285, heads=10, kv_heads=2,
             dim=64, lengths=True, packed=False, dtype="bf16"),
        # training in fp32: a small clip
        dict(name="train_189_h5_d64_f32", op="attn", train=True, batch=1, q=189, k=189, heads=5, kv_heads=5, dim=64,
             lengths=False, packed=False, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        t, h, w = _log(rng, 1, 24), _log(rng, 1, 40), _log(rng, 1, 60)
        batch, dim, heads = rng.choice([1, 1, 2, 3]), rng.choice([64, 128]), rng.randint(1, 40)
        tokens = t * h * w + rng.choice([0, 0, rng.randint(1, 40)])
        while batch * tokens * heads * dim > 32760 * 1536:
            heads, batch = max(1, heads // 2), 1
        return dict(op="rope", train=rng.random() < 0.5, batch=batch, tokens=tokens, t=t, h=h, w=w, heads=heads,
                    dim=dim, rope=rng.random() < 0.8, half=rng.random() < 0.4,
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
    train = rng.random() < 0.5
    top = 600 if dtype == "f32" else 9000
    q = _log(rng, 1 if not train else 16, top)
    k = rng.choice([q, q, _log(rng, 1, top), 512])
    kv_heads = rng.randint(1, 12)
    heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
    batch, dim = rng.choice([1, 1, 2, 3]), rng.choice([64, 128, 128])
    while batch * heads * q * k > (2 if train else 4) * 32 * 6144 ** 2 // 2:
        heads, kv_heads, batch = max(1, kv_heads // 2), max(1, kv_heads // 2), 1
    return dict(op="attn", train=train, batch=batch, q=q, k=k, heads=heads, kv_heads=kv_heads, dim=dim,
                lengths=rng.random() < 0.4, packed=q == k and heads == kv_heads and rng.random() < 0.5, dtype=dtype)


def _axes(dim):
    """Rotated features of a head on the time, height and width axes."""
    side = 2 * (dim // 6)
    return dim - 2 * side, side, side


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def randn(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(dt)

    if case["op"] == "rope":
        c = case["heads"] * case["dim"]
        state = dict(case=case, x=randn(case["batch"], case["tokens"], c, scale=1.7),
                     weight=(1.0 + 0.2 * torch.randn(c, generator=gen, device="cuda")).to(dt), table=None,
                     dout=randn(case["batch"], case["tokens"], c) if case["train"] else None)
        if case["rope"]:
            # (cos, sin) of every position of every axis, computed in 64 bits: kept by a program between its steps
            rows = []
            for size, feat in zip((case["t"], case["h"], case["w"]), _axes(case["dim"])):
                freq = 10000.0 ** (-torch.arange(0, feat, 2, dtype=torch.float64, device="cuda") / feat)
                ang = torch.arange(size, dtype=torch.float64, device="cuda")[:, None] * freq
                rows.append(torch.stack((ang.cos(), ang.sin()), -1).reshape(-1, 2))
            state["table"] = torch.cat(rows).float()
        return state
    b, q, k, h, hk, d = (case[n] for n in ("batch", "q", "k", "heads", "kv_heads", "dim"))
    state = dict(case=case, lengths=None)
    if case["packed"]:
        qkv = randn(b, q, 3, h, d, scale=1.3)
        state["q"], state["k"], state["v"] = qkv.unbind(2)
    else:
        state["q"], state["k"], state["v"] = randn(b, q, h, d, scale=1.3), randn(b, k, hk, d, scale=1.3), randn(b, k, hk, d)
    if case["lengths"]:
        n = torch.randint((k + 1) // 2, k + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        if b > 2:
            n[1] = 0
        state["lengths"] = n
    state["dout"] = randn(b, q, h, d) if case["train"] else None
    return state


# ------------------------------------------------------------- plain forms
def _pair_tables(state):
    """cos and sin, (tokens, dim / 2), of a sample's tokens in raster order; padding is not rotated."""
    case, table = state["case"], state["table"]
    sizes, feats = (case["t"], case["h"], case["w"]), _axes(case["dim"])
    i = torch.arange(case["t"] * case["h"] * case["w"], device="cuda")
    coords = (i // (case["h"] * case["w"]), i // case["w"] % case["h"], i % case["w"])
    parts, at = [], 0
    for pos, size, feat in zip(coords, sizes, feats):
        parts.append(table[at:at + size * feat // 2].view(size, feat // 2, 2)[pos])
        at += size * feat // 2
    cs = torch.cat(parts, 1)
    full = torch.zeros((case["tokens"], case["dim"] // 2, 2), device="cuda")
    full[..., 0] = 1.0
    full[:cs.shape[0]] = cs
    return full[..., 0], full[..., 1]


def _rotate(n, cos, sin, half):
    """n (batch, tokens, heads, dim) turned by the angles of its tokens."""
    cos, sin = cos[:, None, :], sin[:, None, :]
    if half:
        a, b = n.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    a, b = n[..., 0::2], n[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _plain_rope(state):
    case, dt = state["case"], state["x"].dtype
    x, w = state["x"].float(), state["weight"].float()
    r = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    u = x * r
    y = u * w
    heads = (*x.shape[:2], case["heads"], case["dim"])
    if case["rope"]:
        cos, sin = _pair_tables(state)
        y = _rotate(y.view(heads), cos, sin, case["half"]).view(x.shape)
    if not case["train"]:
        return y.to(dt)
    g = state["dout"].float()
    if case["rope"]:
        g = _rotate(g.view(heads), cos, -sin, case["half"]).view(x.shape)
    g = g * w
    dx = r * (g - u * (g * u).mean(-1, keepdim=True))
    return y.to(dt), dx.to(dt)


def _plain_attention(state):
    case, dt = state["case"], state["q"].dtype
    scale, group = case["dim"] ** -0.5, case["heads"] // case["kv_heads"]
    q = state["q"].float().transpose(1, 2)
    k = state["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    v = state["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    if case["lengths"]:
        gone = torch.arange(case["k"], device="cuda") >= state["lengths"][:, None]
        p.masked_fill_(gone[:, None, None, :], -math.inf)
    m = p.amax(-1, keepdim=True)
    p.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).squeeze(-1)
    p.div_(total.masked_fill(total == 0.0, 1.0))
    o = torch.matmul(p, v)
    out = o.transpose(1, 2).to(dt).contiguous()
    if not case["train"]:
        return out, lse

    def back(g, shared):
        """(batch, heads, tokens, dim) to the input's layout, summed over the heads that share it."""
        if shared:
            g = g.unflatten(1, (case["kv_heads"], group)).sum(2)
        return g.transpose(1, 2).to(dt).contiguous()

    do = state["dout"].float().transpose(1, 2)
    dv = back(torch.matmul(p.transpose(-1, -2), do), True)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = back(torch.matmul(ds, k), False)
    dk = back(torch.matmul(ds.transpose(-1, -2), q), True)
    return out, lse, dq, dk, dv


def run(state):
    case = state["case"]
    if not own:
        return _plain_rope(state) if case["op"] == "rope" else _plain_attention(state)
    import reels_b200 as reels
    if case["op"] == "rope":
        rope = None
        if case["rope"]:
            rope = reels.RopeTable(state["table"], (case["t"], case["h"], case["w"]), _axes(case["dim"]),
                                   interleaved=not case["half"])
        y = reels.rms_norm_rope(state["x"], case["heads"], state["weight"], rope)
        if not case["train"]:
            return y
        return y, reels.rms_norm_rope_backward(state["x"], state["dout"], case["heads"], state["weight"], rope)
    q, k, v, lengths = state["q"], state["k"], state["v"], state["lengths"]
    out, lse = reels.attention(q, k, v, kv_lengths=lengths, return_lse=True)
    if not case["train"]:
        return out, lse
    return (out, lse, *reels.attention_backward(state["dout"], q, k, v, out, lse, kv_lengths=lengths))


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        n = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": (4 if case["train"] else 2) * n * e, "flops": (22 if case["train"] else 8) * n}
    rows, keys = case["batch"] * case["q"] * case["heads"], case["batch"] * case["k"] * case["kv_heads"]
    flops = (14 if case["train"] else 4) * rows * case["k"] * case["dim"]
    if case["lengths"]:  # drawn between a half and all of the keys, none for the second of three samples
        flops = flops * 3 // 4 * (case["batch"] - (case["batch"] > 2)) // case["batch"]
    bytes_ = (2 * rows + 2 * keys) * case["dim"] * e + 4 * rows
    if case["train"]:  # the output's gradient, and the gradients of q, k and v
        bytes_ += (2 * rows + 2 * keys) * case["dim"] * e
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------ 64-bit values
def _exact_rope(state):
    case = state["case"]
    x, w = state["x"].double(), state["weight"].double()
    b, n, c = x.shape
    d, half = case["dim"], case["dim"] // 2
    rms = torch.sqrt((x * x).sum(-1, keepdim=True) / c + 1e-6)
    turn = torch.ones((n, half), dtype=torch.complex128, device="cuda")
    if case["rope"]:
        grid = turn[:case["t"] * case["h"] * case["w"]].view(case["t"], case["h"], case["w"], half)
        table = torch.view_as_complex(state["table"].double())
        at = col = 0
        for axis, feat in enumerate(_axes(d)):
            size, f = grid.shape[axis], feat // 2
            shape = [1, 1, 1, f]
            shape[axis] = size
            grid[..., col:col + f] = table[at:at + size * f].view(shape)
            at, col = at + size * f, col + f

    def spin(z, angle):
        if case["half"]:
            z = z.view(b, n, case["heads"], 2, half).transpose(-1, -2)
        else:
            z = z.view(b, n, case["heads"], half, 2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * angle[:, None, :])
        return (z.transpose(-1, -2) if case["half"] else z).reshape(b, n, c)

    y = spin(x / rms * w, turn)
    if not case["train"]:
        return y
    g = spin(state["dout"].double(), turn.conj()) * w
    return y, g / rms - x * (g * x).sum(-1, keepdim=True) / (c * rms ** 3)


def _exact_attention(state):
    case = state["case"]
    b, nq, nk, h, hk, d = (case[n] for n in ("batch", "q", "k", "heads", "kv_heads", "dim"))
    q, k, v = (state[n].double() for n in ("q", "k", "v"))
    out = torch.zeros((b, nq, h, d), dtype=torch.float64, device="cuda")
    lse = torch.full((b, h, nq), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    lengths = state["lengths"].tolist() if case["lengths"] else [nk] * b
    for i in range(b):
        n = lengths[i]
        for j in range(h if n else 0):
            kj, vj = k[i, :n, j * hk // h], v[i, :n, j * hk // h]
            s = q[i, :, j] @ kj.T / math.sqrt(d)
            lse[i, j] = torch.logsumexp(s, -1)
            p = s.sub_(lse[i, j][:, None]).exp_()
            out[i, :, j] = p @ vj
            if case["train"]:
                do = state["dout"][i, :, j].double()
                dv[i, :n, j * hk // h] += p.T @ do
                dp = do @ vj.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[i, :, j] = ds @ kj
                dk[i, :n, j * hk // h] += ds.T @ q[i, :, j]
    return (out, lse, dq, dk, dv) if case["train"] else (out, lse)


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_rope(state) if case["op"] == "rope" else _exact_attention(state)
