"""GPU parity of the q/k norm with rotary positions and of its pullback where
a block of the vector form works through many rows, for rows of very small
values and for weights of another type than the rows, against plain 64-bit
arithmetic.

Bound per element: u |y| for the output's rounding (u half a step of the
type) and g = (C + 32) fp32 steps of the magnitudes that enter it: |n| of both
features of the pair forward, r (|h| of the pair + |x| r^2 mean |h x|) backward."""
import pytest

pytestmark = pytest.mark.gpu

BF, HF, FL = "bfloat16", "float16", "float32"


@pytest.fixture(scope="module")
def torch():
    import torch as _t
    from reels_b200 import build
    build.build()
    return _t


def _check(torch, x, dout, w, y, dx, eps, cs, heads, half):
    """y and dx (M, C) against the definition; cs (M, D/2, 2) 64-bit (cos, sin), or None."""
    M, C = x.shape
    u, g = torch.finfo(x.dtype).eps / 2, (C + 32) * 2.0 ** -23
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps

    def spin(t, back=False, magnitude=False):
        if cs is None:
            return t.abs() if magnitude else t
        t = t.view(M, heads, C // heads)
        a, b = t.chunk(2, -1) if half else (t[..., 0::2], t[..., 1::2])
        if magnitude:
            p = q = a.abs() + b.abs()
        else:
            c, s = cs[:, None, :, 0], cs[:, None, :, 1] * (-1 if back else 1)
            p, q = a * c - b * s, a * s + b * c
        return (torch.cat((p, q), -1) if half else torch.stack((p, q), -1).flatten(-2)).reshape(M, C)

    xd, gd, wd = x.double(), dout.double(), 1.0 if w is None else w.double()
    r = 1 / (xd.square().mean(-1, keepdim=True) + eps).sqrt()
    n = xd * r * wd
    want = spin(n)
    bound = u * want.abs() + g * spin(n, magnitude=True) + tiny
    assert float(((y.double() - want).abs() / bound).max()) <= 1.0
    h, hm = spin(gd, back=True) * wd, spin(gd, magnitude=True) * (1.0 if w is None else wd.abs())
    want = r * (h - xd * r * r * (h * xd).mean(-1, keepdim=True))
    bound = u * want.abs() + g * r * (hm + xd.abs() * r * r * (hm * xd.abs()).mean(-1, keepdim=True)) + tiny
    fits = want.abs() < torch.finfo(x.dtype).max
    assert float(((dx.double() - want).abs() / bound)[fits].max()) <= 1.0


def _angles(torch, rope, coords, on):
    """(cos, sin) of the table at a token's coordinates, in 64 bits; tokens that are not `on` are not turned."""
    parts, at = [], 0
    for size, dim, pos in zip(rope.sizes, rope.dims, coords):
        t = rope.table[at:at + size * dim // 2].view(size, dim // 2, 2).double()
        parts.append(t[pos.clamp(0, size - 1)])
        at += size * dim // 2
    still = torch.tensor([1.0, 0.0], dtype=torch.float64, device="cuda")
    return torch.where(on[:, None, None], torch.cat(parts, 1), still)


@pytest.mark.parametrize("B,T,heads,D,sizes,half,dtype,given", [
    (1, 7001, 12, 128, (7, 20, 50), False, BF, False),   # one token of padding
    (3, 4003, 8, 64, (10, 20, 20), True, HF, False),     # samples begin inside a block's walk
    (7, 1003, 5, 64, (4, 10, 25), False, FL, False),     # padding in every sample
    (2, 2500, 3, 16, (25, 10, 10), True, FL, True),      # narrow rows, given positions
    (1, 3001, 128, 128, (3, 20, 50), True, BF, False),   # the widest rows
    (1, 2203, 72, 128, (2, 20, 50), False, FL, True),    # wide, fp32 (the pullback's scalar form)
    (11, 509, 40, 128, (5, 10, 10), False, HF, True),
    (1, 6007, 24, 64, None, False, BF, False),           # the norm alone
    (2, 3001, 100, 128, None, False, HF, False),
])
def test_many_rows_a_block(torch, B, T, heads, D, sizes, half, dtype, given):
    from reels_b200 import check_device_status, rms_norm_rope, rms_norm_rope_backward, rope_table
    gen = torch.Generator(device="cuda").manual_seed(T)
    dt, C, eps = getattr(torch, dtype), heads * D, 1e-6
    x = (1.7 * torch.randn((B, T, C), generator=gen, device="cuda")).to(dt)
    dout = torch.randn((B, T, C), generator=gen, device="cuda").to(dt)
    w = (1 + 0.2 * torch.randn(C, generator=gen, device="cuda")).to(dt)
    rope = pos = cs = None
    if sizes is not None:
        rope = rope_table(D, sizes, interleaved=not half)
        i = torch.arange(T, device="cuda").repeat(B)
        if given:
            pos = torch.stack([torch.randint(-1 if n == 0 else 0, s, (B, T), generator=gen, device="cuda")
                               for n, s in enumerate(sizes)], -1)
            coords = pos.view(-1, 3).unbind(1)
            on = coords[0] >= 0
        else:
            coords = (i // (sizes[1] * sizes[2]), i // sizes[2] % sizes[1], i % sizes[2])
            on = coords[0] < sizes[0]
        cs = _angles(torch, rope, coords, on)
    y = rms_norm_rope(x, heads, w, rope, eps, positions=pos)
    dx = rms_norm_rope_backward(x, dout, heads, w, rope, eps, positions=pos)
    check_device_status()
    flat = lambda t: t.view(-1, C)
    for part in torch.arange(B * T, device="cuda").split(4096):  # the 64-bit values of all rows would take many GB
        _check(torch, flat(x)[part], flat(dout)[part], w, flat(y)[part], flat(dx)[part], eps,
               None if cs is None else cs[part], heads, half)


@pytest.mark.parametrize("dtype", [BF, FL])
@pytest.mark.parametrize("C,heads", [(256, 2), (100, 5)])  # the vector and the scalar form
@pytest.mark.parametrize("rotated", [False, True])
def test_rows_of_very_small_values(torch, dtype, C, heads, rotated):
    """r = 1e13 and more without epsilon: r^3 is beyond fp32, dx = r (h - x r^2 mean(h x)) is not."""
    from reels_b200 import rms_norm_rope, rms_norm_rope_backward, rope_table
    gen = torch.Generator(device="cuda").manual_seed(2)
    dt = getattr(torch, dtype)
    sizes = torch.tensor([1e-13, 1e-14, 3e-16, 1e-17], device="cuda")[:, None]
    x = (sizes * torch.randn((4, C), generator=gen, device="cuda")).to(dt)
    dout = torch.randn((4, C), generator=gen, device="cuda").to(dt)
    w = (1 + 0.2 * torch.randn(C, generator=gen, device="cuda")).to(dt)
    rope = rope_table(C // heads, (4,), (C // heads,)) if rotated else None
    cs = _angles(torch, rope, (torch.arange(4, device="cuda"),), torch.ones(4, dtype=torch.bool, device="cuda")) if rotated else None
    y = rms_norm_rope(x, heads, w, rope, 0.0)
    dx = rms_norm_rope_backward(x, dout, heads, w, rope, 0.0)
    assert bool(torch.isfinite(dx.float()).all())
    _check(torch, x, dout, w, y, dx, 0.0, cs, heads, False)


@pytest.mark.parametrize("x_type,w_type", [(BF, FL), (HF, FL), (BF, HF), (FL, BF), (HF, "float64")])
@pytest.mark.parametrize("C,heads,T", [(512, 4, 700), (10240, 80, 300), (100, 5, 9)])
@pytest.mark.parametrize("rotated", [0, 1, 2])
def test_a_weight_of_another_type_keeps_its_bits(torch, x_type, w_type, C, heads, T, rotated):
    """The weight enters in fp32, whatever x is: nothing of it is rounded to x's type."""
    from reels_b200 import RMSNormRopeFunction, check_device_status, rms_norm_rope, rope_table
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((T, C), generator=gen, device="cuda").to(getattr(torch, x_type)).requires_grad_(True)
    dout = torch.randn((T, C), generator=gen, device="cuda").to(x.dtype)
    # quarters of x's step next to 1, where w's type holds them: rounding would lose them
    step = torch.finfo(x.dtype).eps / 4
    w = (1 + step * (1 + torch.randint(0, 3, (C,), generator=gen, device="cuda"))).to(getattr(torch, w_type))
    rope = rope_table(C // heads, (T,), (C // heads,), interleaved=rotated == 1) if rotated else None
    at = torch.arange(T, device="cuda")
    cs = _angles(torch, rope, (at,), at >= 0) if rotated else None
    y = RMSNormRopeFunction.apply(x, heads, w, rope)
    y.backward(dout)
    check_device_status()
    x, dx = x.detach(), x.grad
    assert torch.equal(y.detach(), rms_norm_rope(x, heads, w, rope))
    assert y.dtype == x.dtype and dx.dtype == x.dtype
    # against the same weight in 64 bits: rounded to x's type it would be off by up to half a step,
    # which the bound allows for the output's rounding alone
    _check(torch, x, dout, w, y.detach(), dx, 1e-6, cs, heads, rotated == 2)


def test_a_view_by_head_is_not_normed_per_head(torch):
    """The norm spans all heads: a view by head, which shows only one head as
    its last dimension, is refused where nothing else tells it from tokens."""
    from reels_b200 import rms_norm_rope, rms_norm_rope_backward
    x = torch.randn((2, 6, 8, 64), device="cuda").bfloat16()
    for call in (lambda: rms_norm_rope(x, 8), lambda: rms_norm_rope_backward(x, x, 8)):
        with pytest.raises(ValueError, match="view by head"):
            call()
    want = rms_norm_rope(x.flatten(-2), 8)
    assert want.shape == (2, 6, 512)
    # 8 tokens of 64 features in 8 heads, said so
    assert torch.equal(rms_norm_rope(x, 8, tokens_per_sample=8), rms_norm_rope(x.view(12, 8, 64), 8).view(x.shape))
