"""Plain 64-bit attention and its gradient for the parity tests, with an
elementwise bound on what a correct kernel may be off.

The bounds count roundings: u is half a step of the element type.  Scores are
fp32 sums of exact products, so a score is off by at most gd times the sum of
its products' magnitudes (gd = (D + 8) steps of fp32), and a probability by a
relative ep made of its score's, its row's and the exponential's errors.  A
probability or dS that feeds a tensor-core product is rounded once more (u of
the type; fp32 runs unrounded), and the product's fp32 sum over n terms is
off by at most gn = (n + 16) fp32 steps of its terms' magnitudes.  delta is
formed from the rounded output: off by u sum |dO| |o|."""
import math

import torch

STEP = 2.0 ** -23


class Case:
    def __init__(self, B, Sq, Sk, H, HK, D, dtype, lengths=None, packed=False, scale=None, seed=0, spread=1.3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype, self.scale = dtype, D ** -0.5 if scale is None else scale

        def randn(*shape):
            return (spread * torch.randn(shape, generator=gen, device="cuda")).to(dtype)

        if packed:
            self.q, self.k, self.v = randn(B, Sq, 3, H, D).unbind(2)
        else:
            self.q, self.k, self.v = randn(B, Sq, H, D), randn(B, Sk, HK, D), randn(B, Sk, HK, D)
        self.dout = randn(B, Sq, H, D)
        self.lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")


def reference(c, backward=True):
    """{name: (value, bound)} in fp64, laid out as the kernels' outputs."""
    B, Sq, H, D = c.q.shape
    Sk, HK = c.k.shape[1:3]
    group, f64 = H // HK, torch.float64
    u = torch.finfo(c.dtype).eps / 2
    up = u if c.dtype != torch.float32 else 0.0
    tiny = torch.finfo(c.dtype).smallest_normal * torch.finfo(c.dtype).eps  # a subnormal step
    gone = torch.zeros((B, 1, 1, Sk), dtype=torch.bool, device="cuda")
    if c.lengths is not None:
        gone = (torch.arange(Sk, device="cuda") >= c.lengths[:, None])[:, None, None, :]
    dead = gone.transpose(-1, -2)
    q = c.q.to(f64).transpose(1, 2)
    # what lies behind a sample's length takes no part, whatever it holds
    k = c.k.to(f64).transpose(1, 2).repeat_interleave(group, 1).masked_fill(dead, 0.0)
    v = c.v.to(f64).transpose(1, 2).repeat_interleave(group, 1).masked_fill(dead, 0.0)
    s = c.scale * (q @ k.transpose(-1, -2))
    es = c.scale * (q.abs() @ k.abs().transpose(-1, -2)) * (D + 8) * STEP + 4 * STEP * s.abs()
    s = s.masked_fill(gone, -math.inf)
    lse = torch.logsumexp(s, -1) if Sk else torch.full((B, H, Sq), -math.inf, dtype=f64, device="cuda")
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
    es = es.masked_fill(gone, 0.0)
    top = es.amax(-1, keepdim=True) if Sk else torch.zeros((B, H, Sq, 1), dtype=f64, device="cuda")
    ep = es + top + 8 * STEP * (1 + lse.abs().masked_fill(lse == -math.inf, 0.0)[..., None]) + (Sk + 16) * STEP
    gk, gq, gd = (Sk + 16) * STEP, (group * Sq + 16) * STEP, (D + 16) * STEP
    o = p @ v
    # fp16 probabilities below 2^-31 of the row's largest are lost: Sk of them weigh Sk 2^-31
    lost = Sk * 2.0 ** -31 * v.abs().amax() if Sk else 0.0
    eo = u * o.abs() + (p * (up + ep + gk)) @ v.abs() + tiny + lost

    def out_layout(x):
        return x.transpose(1, 2)

    def shared(x):
        return x.unflatten(1, (HK, group)).sum(2).transpose(1, 2)

    res = {"out": (out_layout(o), out_layout(eo)),
           "lse": (lse, top.squeeze(-1) + 8 * STEP * (1 + lse.abs().masked_fill(lse == -math.inf, 0.0)) + gk)}
    if not backward:
        return res
    do = c.dout.to(f64).transpose(1, 2)
    dp = do @ v.transpose(-1, -2)
    adp = do.abs() @ v.abs().transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    edelta = (do.abs() * (eo + gd * o.abs())).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # fp16: dS is scaled by a power of two into its range; what is below 2^-24 of 2^14 / (|dO| |v|) is lost
    floor = 2.0 ** -36 * do.norm(dim=-1).amax() * v.norm(dim=-1).amax() if Sk and Sq else 0.0
    eds = up * ds.abs() + ep * ds.abs() + p * (gd * adp + edelta + 2 * STEP * (dp.abs() + delta.abs()))
    if c.dtype == torch.float16:
        eds = eds + floor
    eds = eds.masked_fill(gone, 0.0)
    dv, edv = p.transpose(-1, -2) @ do, (p * (up + ep + gq) + lost).masked_fill(gone, 0.0).transpose(-1, -2) @ do.abs()
    dk = c.scale * (ds.transpose(-1, -2) @ q)
    edk = c.scale * ((eds + gq * ds.abs()).transpose(-1, -2) @ q.abs())
    dq = c.scale * (ds @ k)
    edq = c.scale * ((eds + gk * ds.abs()) @ k.abs())
    res["dq"] = out_layout(dq), out_layout(edq + (u + STEP) * dq.abs() + tiny)
    for name, x, e in (("dk", dk, edk), ("dv", dv, edv)):
        x = shared(x)
        res[name] = x, shared(e) + (u + STEP) * x.abs() + tiny
    return res


def check(name, got, want):
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), name
    got = got.double()
    fin = torch.isfinite(value)
    assert torch.equal(got[~fin], value[~fin]), f"{name}: infinities differ"
    off = (got - value).abs()[fin]
    over = off / bound[fin].clamp_min(1e-300)
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound (largest error {float(off.max()):.3g})"
