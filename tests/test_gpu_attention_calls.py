"""GPU parity of the attention stretch in the forms a caller may give it: the
narrowest and odd head sizes, scales, orders of the dimensions, pointers that
are not aligned, and the norm written over what it reads."""
import ctypes

import pytest

import attention_case as ac

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as _t
    from reels_b200 import build
    build.build()
    return _t


@pytest.fixture(scope="module")
def reels(torch):
    import reels_b200
    return reels_b200


def _all(reels, c, dout=None, out=None):
    """Checks every output against 64 bits; returns them."""
    o, lse = reels.attention(c.q, c.k, c.v, c.scale, c.lengths, return_lse=True)
    grads = reels.attention_backward(c.dout if dout is None else dout, c.q, c.k, c.v, o if out is None else out(o), lse,
                                     c.scale, c.lengths)
    reels.check_device_status()
    want = ac.reference(c)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (o, lse, *grads)):
        ac.check(name, got, want[name])
    return o, lse, *grads


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("D", [8, 16, 24, 56, 72, 88, 120])
@pytest.mark.parametrize("Sq", [3, 150])
def test_head_sizes_in_multiples_of_8(torch, reels, D, dtype, Sq):
    _all(reels, ac.Case(2, Sq, 290, 4, 2, D, getattr(torch, dtype), [290, 131], seed=D))


@pytest.mark.parametrize("D", [1, 3, 65, 130, 255, 256])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_head_sizes_on_the_cuda_cores(torch, reels, D, dtype):
    _all(reels, ac.Case(1, 70, 90, 2, 1, D, getattr(torch, dtype), [77], seed=D))


@pytest.mark.parametrize("dtype,Sq", [("bfloat16", 200), ("float16", 200), ("bfloat16", 2), ("float32", 60)])
@pytest.mark.parametrize("scale", [2.0 ** -9, 0.37])
def test_scales(torch, reels, dtype, Sq, scale):
    _all(reels, ac.Case(1, Sq, 330, 2, 2, 64, getattr(torch, dtype), scale=scale, seed=31))


@pytest.mark.parametrize("dtype,Sq", [("bfloat16", 200), ("float16", 200), ("bfloat16", 2), ("float32", 60)])
@pytest.mark.parametrize("order", [(1, 0, 2, 3), (0, 2, 1, 3), (2, 1, 0, 3)])
def test_orders_of_the_dimensions(torch, reels, dtype, Sq, order):
    """(tokens, batch, heads, D), (batch, heads, tokens, D) and (heads, tokens, batch, D) in memory."""
    c = ac.Case(3, Sq, 260, 4, 2, 64, getattr(torch, dtype), [260, 7, 129], seed=32)
    want = _all(reels, c)
    back = [order.index(i) for i in range(4)]
    c.q, c.k, c.v = (t.permute(order).contiguous().permute(back) for t in (c.q, c.k, c.v))
    assert not c.q.is_contiguous()
    got = reels.attention(c.q, c.k, c.v, c.scale, c.lengths, return_lse=True)
    grads = reels.attention_backward(c.dout, c.q, c.k, c.v, *got, c.scale, c.lengths)
    assert all(torch.equal(a, b) for a, b in zip(want, (*got, *grads)))


@pytest.mark.parametrize("dtype,Sq,Sk", [("bfloat16", 200, 300), ("float16", 200, 300), ("float16", 2, 3000),
                                         ("float32", 60, 70)])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout", "out"])
def test_pointers_that_are_not_aligned(torch, reels, dtype, Sq, Sk, which):
    c = ac.Case(2, Sq, Sk, 2, 2, 64, getattr(torch, dtype), [Sk, 65], seed=33)

    def shift(t):
        store = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        got = store[1:].view(t.shape)
        got.copy_(t)
        return got

    if which in "qkv":
        setattr(c, which, shift(getattr(c, which)))
    _all(reels, c, dout=shift(c.dout) if which == "dout" else None, out=shift if which == "out" else None)


@pytest.mark.parametrize("C,heads", [(1536, 12), (16384, 32), (512, 1), (2560, 10), (96, 3)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_the_norm_in_place(torch, reels, C, heads, dtype):
    """out = x forward, dx = x and dx = dout backward, at several rows a block
    (16384 features: heads of 512, the widest the vector form takes)."""
    from reels_b200 import _native as nat
    dt, M = getattr(torch, dtype), 4000
    D, code = C // heads, {"bfloat16": nat.BF16, "float32": nat.F32}[dtype]
    rope = reels.rope_table(D, (10, 20, 20))
    x, dout = (torch.randn((M, C), device="cuda").to(dt) for _ in range(2))
    y, dx = reels.rms_norm_rope(x, heads, None, rope), reels.rms_norm_rope_backward(x, dout, heads, None, rope)
    sizes, dims, pairing = rope._args
    r = nat.Rope(rope.table.data_ptr(), None, sizes, dims, pairing)
    st = torch.cuda.current_stream().cuda_stream
    a = x.clone()
    nat.check("forward", nat.lib().reels_rms_norm_rope(a.data_ptr(), M, heads, D, None, ctypes.byref(r), M, 1e-6, code,
                                                       a.data_ptr(), st))
    assert torch.equal(a, y)
    for over in (0, 1):
        pair = [x.clone(), dout.clone()]
        nat.check("backward", nat.lib().reels_rms_norm_rope_backward(
            pair[0].data_ptr(), pair[1].data_ptr(), M, heads, D, None, ctypes.byref(r), M, 1e-6, code,
            pair[over].data_ptr(), st))
        assert torch.equal(pair[over], dx)
    reels.check_device_status()


@pytest.mark.parametrize("D", [256, 512])
@pytest.mark.parametrize("half", [False, True])
def test_wide_heads_of_the_norm(torch, reels, D, half):
    """One head and several, against the norm and the rotation in 64 bits."""
    for heads in (1, 5):
        T, C = 500, heads * D
        rope = reels.rope_table(D, (T,), (D,), interleaved=not half)
        x, dout = (torch.randn((T, C), device="cuda").bfloat16() for _ in range(2))
        cs = rope.table.view(T, 1, D // 2, 2).double()

        def spin(t, sign):
            t = t.view(T, heads, D)
            a, b = t.chunk(2, -1) if half else (t[..., 0::2], t[..., 1::2])
            p, q = a * cs[..., 0] - sign * b * cs[..., 1], sign * a * cs[..., 1] + b * cs[..., 0]
            return (torch.cat((p, q), -1) if half else torch.stack((p, q), -1).flatten(-2)).reshape(T, C)

        xd = x.double()
        r = (xd.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        h = spin(dout.double(), -1)
        want = r * (h - xd * r * r * (h * xd).mean(-1, keepdim=True))
        # half a bf16 step of the value, and (C + 32) fp32 steps of values up to a few units
        for got, ref in ((reels.rms_norm_rope(x, heads, None, rope), spin(xd * r, 1)),
                         (reels.rms_norm_rope_backward(x, dout, heads, None, rope), want)):
            assert float(((got.double() - ref).abs() - 2.0 ** -8 * ref.abs()).max()) <= (C + 32) * 2.0 ** -23 * 8
