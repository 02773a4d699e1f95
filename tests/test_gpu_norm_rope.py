"""GPU parity of the q/k norm with rotary positions and of its pullback
against plain 64-bit arithmetic.

Bound per element: u |y| for the output's rounding (u half a step of the
type) and g = (C + 32) fp32 steps of the magnitudes that enter it for the
fp32 sums and products: |n| of both features of the pair forward,
r (|h| of the pair + |x| r^2 mean |h x|) backward."""
import pytest

pytestmark = pytest.mark.gpu

BF, HF, FL = "bfloat16", "float16", "float32"


@pytest.fixture(scope="module")
def torch():
    import torch as _t
    from reels_b200 import build
    build.build()
    return _t


def _angles(torch, rope, sizes, dims, coords):
    """Angles (tokens, D/2) from the table itself, in 64 bits; nan coordinates are not turned."""
    cs, at = [], 0
    for size, dim, pos in zip(sizes, dims, coords):
        t = rope.table[at:at + size * dim // 2].view(size, dim // 2, 2).double()
        cs.append(t[pos.clamp(0, size - 1)])
        at += size * dim // 2
    cs = torch.cat(cs, 1)
    ok = torch.stack([(pos >= 0) & (pos < size) for pos, size in zip(coords, sizes)]).all(0)
    one = torch.tensor([1.0, 0.0], dtype=torch.float64, device="cuda")
    return torch.where(ok[:, None, None], cs, one)


def _spin(torch, x, cs, half, back=False, magnitude=False):
    c, s = cs[..., 0][:, None], cs[..., 1][:, None]
    if back:
        s = -s
    D = x.shape[-1]
    a, b = (x[..., :D // 2], x[..., D // 2:]) if half else (x[..., 0::2], x[..., 1::2])
    if magnitude:
        u = v = a.abs() + b.abs()
    else:
        u, v = a * c - b * s, a * s + b * c
    return torch.cat((u, v), -1) if half else torch.stack((u, v), -1).flatten(-2)


CASES = [
    # samples, tokens, heads, D, sizes, dims, half, dtype, weight
    (1, 60, 12, 128, (3, 4, 5), None, False, BF, True),
    (2, 65, 5, 64, (3, 4, 5), None, False, FL, True),        # padding tokens, restart per sample
    (2, 24, 32, 128, (2, 3, 4), None, True, HF, True),
    (1, 30, 40, 128, (2, 3, 5), None, True, BF, False),
    (1, 7, 128, 128, (1, 1, 7), None, False, BF, True),      # the widest row
    (3, 5, 1, 64, (1, 1, 5), None, False, HF, True),
    (1, 12, 3, 48, (3, 2, 2), None, False, BF, True),        # head size outside the vector form
    (1, 12, 3, 22, (3, 2, 2), (10, 6, 6), True, FL, True),
    (1, 9, 7, 32, (9,), (32,), False, BF, True),             # one axis
    (2, 12, 4, 64, (3, 4), (24, 40), True, BF, True),        # two axes
    (1, 3, 2, 16, (1, 1, 3), (0, 0, 16), False, HF, False),
    (1, 17, 12, 128, None, None, False, BF, True),           # the norm alone
    (1, 17, 3, 7, None, None, False, HF, True),              # odd features
    (1, 1, 5, 100, None, None, False, FL, False),
]


@pytest.mark.parametrize("B,T,H,D,sizes,dims,half,dtype,weighted", CASES)
@pytest.mark.parametrize("given", [False, True])
def test_parity(torch, B, T, H, D, sizes, dims, half, dtype, weighted, given):
    from reels_b200 import check_device_status, rms_norm_rope, rms_norm_rope_backward, rope_table
    if given and sizes is None:
        pytest.skip("positions need a table")
    gen = torch.Generator(device="cuda").manual_seed(B * T + H)
    dt, C, eps = getattr(torch, dtype), H * D, 1e-6
    x = (1.7 * torch.randn((B, T, C), generator=gen, device="cuda")).to(dt)
    x[0, 0] = 0  # a row without length: r = 1 / sqrt(epsilon)
    dout = torch.randn((B, T, C), generator=gen, device="cuda").to(dt)
    w = (1 + 0.2 * torch.randn(C, generator=gen, device="cuda")).to(dt) if weighted else None
    rope = pos = None
    cs = torch.zeros((B * T, D // 2, 2), dtype=torch.float64, device="cuda")
    cs[..., 0] = 1
    if sizes is not None:
        rope = rope_table(D, sizes, dims, interleaved=not half)
        if given:
            coords = [torch.randint(-1 if i == 0 else 0, s, (B * T,), generator=gen, device="cuda")
                      for i, s in enumerate(sizes)]
            pos = torch.stack(coords, -1).view(B, T, len(sizes))
        else:
            i = torch.arange(T, device="cuda").repeat(B)
            coords = []
            for a in range(len(sizes)):
                inner = 1
                for s in sizes[a + 1:]:
                    inner *= s
                coords.append(i // inner if a == 0 else i // inner % sizes[a])
        cs = _angles(torch, rope, sizes, rope.dims, coords)
    y = rms_norm_rope(x, H, w, rope, eps, positions=pos)
    dx = rms_norm_rope_backward(x, dout, H, w, rope, eps, positions=pos)
    check_device_status()
    u, g = torch.finfo(dt).eps / 2, (C + 32) * 2.0 ** -23
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    xd, wd = x.double().view(-1, C), w.double() if weighted else 1.0
    rope_on = sizes is not None
    r = 1 / (xd.square().mean(-1, keepdim=True) + eps).sqrt()
    heads = lambda t: t.view(-1, H, D)
    spin = lambda t, **k: (_spin(torch, heads(t), cs, half, **k) if rope_on else heads(t).abs() if k.get("magnitude")
                           else heads(t)).reshape(-1, C)
    n = xd * r * wd
    want = spin(n)
    bound = u * want.abs() + g * spin(n, magnitude=True) + tiny
    assert float(((y.double().view(-1, C) - want).abs() / bound).max()) <= 1.0
    gd = dout.double().view(-1, C)
    h = spin(gd, back=True) * wd
    hm = spin(gd, magnitude=True) * (wd.abs() if weighted else 1.0)
    want = r * (h - xd * r * r * (h * xd).mean(-1, keepdim=True))
    bound = u * want.abs() + g * r * (hm + xd.abs() * r * r * (hm * xd.abs()).mean(-1, keepdim=True)) + tiny
    finite = want.abs() < torch.finfo(dt).max  # the zero row's gradient is 1000 times dout
    assert float(((dx.double().view(-1, C) - want).abs() / bound)[finite].max()) <= 1.0


def test_gradient_against_differences(torch):
    from reels_b200 import RMSNormRopeFunction, rms_norm_rope, rope_table
    gen = torch.Generator(device="cuda").manual_seed(1)
    rope = rope_table(16, (2, 2, 2), (8, 4, 4))
    x = torch.randn((1, 8, 48), generator=gen, device="cuda", requires_grad=True)
    w = 1 + 0.2 * torch.randn(48, generator=gen, device="cuda")
    dout = torch.randn((1, 8, 48), generator=gen, device="cuda")
    RMSNormRopeFunction.apply(x, 3, w, rope).backward(dout)
    f = lambda t: float((rms_norm_rope(t, 3, w, rope).double() * dout.double()).sum())
    # step 2^-8: truncation h^2 / 6 f''' ~ 1e-5, rounding sqrt(384) 2^-24 / h ~ 3e-4
    h = 2.0 ** -8
    for i in ((0, 0, 0), (0, 3, 17), (0, 7, 47)):
        e = torch.zeros_like(x)
        e[i] = h
        diff = (f((x + e).detach()) - f((x - e).detach())) / (2 * h)
        assert float(x.grad[i]) == pytest.approx(diff, rel=2e-3, abs=2e-3)


def test_position_behind_the_table_is_reported(torch):
    from reels_b200 import check_device_status, rms_norm_rope, rope_table
    from reels_b200._native import NativeError
    rope = rope_table(64, (2, 2, 2))
    x = torch.randn((1, 3, 128), device="cuda").bfloat16()
    pos = torch.tensor([[[0, 1, 1], [2, 0, 0], [-1, 5, 5]]], device="cuda")
    y = rms_norm_rope(x, 2, None, rope, positions=pos)
    with pytest.raises(NativeError, match="position"):
        check_device_status()
    plain = rms_norm_rope(x, 2)
    assert torch.equal(y[0, 1:], plain[0, 1:]) and not torch.equal(y[0, 0], plain[0, 0])
    check_device_status()


def test_in_place_and_unaligned(torch):
    """The C entry point writes over its input, and takes pointers that are not 16-byte aligned."""
    import ctypes
    from reels_b200 import _native as nat
    from reels_b200 import rms_norm_rope, rope_table
    rope = rope_table(64, (1, 2, 3))
    store = torch.randn(6 * 128 + 1, device="cuda").bfloat16()
    x = store[1:].view(6, 128)  # 2 bytes off
    want = rms_norm_rope(x.clone(), 2, None, rope)
    sizes, dims, pairing = rope._args
    r = ctypes.byref(nat.Rope(rope.table.data_ptr(), None, sizes, dims, pairing))
    nat.check("norm", nat.lib().reels_rms_norm_rope(x.data_ptr(), 6, 2, 64, None, r, 6, 1e-6, nat.BF16, x.data_ptr(),
                                                    torch.cuda.current_stream().cuda_stream))
    # the two forms sum a row in different orders: one rounding apart at most
    assert float((x.float() - want.float()).abs().max()) <= 2.0 ** -8 * float(want.float().abs().max())


def test_a_weight_that_asks_for_a_gradient_is_refused(torch):
    from reels_b200 import RMSNormRopeFunction
    x = torch.randn((4, 128), device="cuda", requires_grad=True)
    w = torch.ones(128, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="frozen"):
        RMSNormRopeFunction.apply(x, 2, w).sum().backward()
    with torch.no_grad():
        RMSNormRopeFunction.apply(x, 2, w)
    RMSNormRopeFunction.apply(x, 2, w.detach()).sum().backward()


def test_positions_past_32_bits_do_not_wrap(torch):
    from reels_b200 import check_device_status, rms_norm_rope, rope_table
    from reels_b200._native import NativeError
    rope = rope_table(64, (2, 2, 2))
    x = torch.randn((1, 2, 128), device="cuda").bfloat16()
    plain = rms_norm_rope(x, 2)
    pos = torch.tensor([[[1, 1, -2 ** 32 + 1], [-2 ** 40, 0, 0]]], device="cuda")
    assert torch.equal(rms_norm_rope(x, 2, None, rope, positions=pos), plain)
    check_device_status()
    pos = torch.tensor([[[1, 1, 2 ** 32 + 1], [2 ** 32, 1, 1]]], device="cuda")
    assert torch.equal(rms_norm_rope(x, 2, None, rope, positions=pos), plain)
    with pytest.raises(NativeError, match="position"):
        check_device_status()


def test_offsets_past_32_bits(torch):
    """1.4 million rows of 1536 features: the last lie 2.15e9 elements in."""
    from reels_b200 import rms_norm_rope, rms_norm_rope_backward, rope_table
    rope = rope_table(128, (10, 10, 10))
    part = torch.randn((1, 1000, 1536), device="cuda").bfloat16()
    x = part.expand(1400, -1, -1).contiguous()
    want = rms_norm_rope(part, 12, None, rope)
    y = rms_norm_rope(x, 12, None, rope)
    assert torch.equal(y[-1:], want) and torch.equal(y[:1], want)
    want = rms_norm_rope_backward(part, part.flip(1), 12, None, rope)
    y.copy_(part.flip(1).expand(1400, -1, -1))
    dx = rms_norm_rope_backward(x, y, 12, None, rope)
    assert torch.equal(dx[-1:], want) and torch.equal(dx[:1], want)
