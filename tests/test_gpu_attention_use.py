"""GPU tests of the attention stretch as a program uses it: the operators in
a run with the block's projections, captured graphs, other streams, padding
that holds anything, far offsets, falling and rising scores, small gradients."""
import math

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


def _plain_stretch(torch, q, k, v, wq, wk, cs, heads, eps=1e-6):
    """norm, rotation (interleaved) and attention in the tensors' own type, differentiable."""
    B, T, C = q.shape
    D = C // heads

    def norm_rope(x, w):
        n = (x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w).view(B, T, heads, D)
        a, b = n[..., 0::2], n[..., 1::2]
        c, s = cs[:, None, :, 0], cs[:, None, :, 1]
        return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2).transpose(1, 2)

    p = torch.softmax(norm_rope(q, wq) @ norm_rope(k, wk).transpose(-1, -2) * D ** -0.5, -1)
    return (p @ v.view(B, T, heads, D).transpose(1, 2)).transpose(1, 2).reshape(B, T, C)


def _raster(torch, rope):
    parts, at = [], 0
    t, h, w = rope.sizes
    i = torch.arange(t * h * w, device="cuda")
    for pos, size, dim in zip((i // (h * w), i // w % h, i % w), rope.sizes, rope.dims):
        parts.append(rope.table[at:at + size * dim // 2].view(size, dim // 2, 2).double()[pos])
        at += size * dim // 2
    return torch.cat(parts, 1)


def _stretch(reels, q, k, v, wq, wk, rope, heads):
    B, T, C = q.shape
    split = lambda t: t.view(B, T, heads, C // heads)
    q = reels.RMSNormRopeFunction.apply(q, heads, wq, rope)
    k = reels.RMSNormRopeFunction.apply(k, heads, wk, rope)
    return reels.AttentionFunction.apply(split(q), split(k), split(v)).reshape(B, T, C)


def test_the_stretch_and_its_gradient_fp32(torch, reels):
    """Both operators together through autograd against plain 64-bit autograd.
    Sums of up to 320 fp32 terms in four stages: 4 * 320 * 2^-24 = 8e-5 of the
    largest magnitude bounds what rounding can do to a value or gradient."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    heads, D, rope = 5, 64, reels.rope_table(64, (2, 5, 7))
    B, T, C = 2, 70, heads * D
    x = [torch.randn((B, T, C), generator=gen, device="cuda") for _ in range(4)]
    w = [1 + 0.2 * torch.randn(C, generator=gen, device="cuda") for _ in range(2)]
    ins = [t.clone().requires_grad_(True) for t in x[:3]]
    out = _stretch(reels, *ins, *w, rope, heads)
    out.backward(x[3])
    ref = [t.double().requires_grad_(True) for t in x[:3]]
    want = _plain_stretch(torch, *ref, *(t.double() for t in w), _raster(torch, rope), heads)
    want.backward(x[3].double())
    for name, a, b in [("out", out.detach(), want.detach())] + [("d" + n, i.grad, r.grad) for n, i, r in zip("qkv", ins, ref)]:
        assert float((a.double() - b).abs().max()) <= 8e-5 * float(b.abs().max()), name


def test_a_block_with_its_projections(torch, reels):
    """Quantised LoRA projections, norm and rotation, attention, output
    projection: the adapters of all four receive gradients, the same bits on
    every run."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    heads, D, rope = 4, 128, reels.rope_table(128, (3, 4, 8))
    C, T, r = heads * D, 96, 8
    layers = []
    for _ in range(4):
        W = 0.04 * torch.randn((C, C), generator=gen, device="cuda")
        A = (torch.randn((r, C), generator=gen, device="cuda") / C ** 0.5).bfloat16()
        Bm = (0.01 * torch.randn((C, r), generator=gen, device="cuda")).bfloat16()
        layers.append(reels.LoRALinear(reels.quantize_frozen_matrix(W, torch.bfloat16), None, A.t().contiguous().t(),
                                       Bm.t().contiguous().t(), float(r)))
    w = [(1 + 0.2 * torch.randn(C, generator=gen, device="cuda")).bfloat16() for _ in range(2)]
    x = torch.randn((1, T, C), generator=gen, device="cuda").bfloat16()
    dy = torch.randn((1, T, C), generator=gen, device="cuda").bfloat16()

    def step():
        leaves = [(l.A.detach().requires_grad_(True), l.B.detach().requires_grad_(True)) for l in layers]
        xin = x.clone().requires_grad_(True)
        q, k, v = (reels.LoRALinearFunction.apply(xin, *leaves[i], layers[i]) for i in range(3))
        o = _stretch(reels, q, k, v, *w, rope, heads)
        y = reels.LoRALinearFunction.apply(o, *leaves[3], layers[3])
        y.backward(dy)
        return [y.detach(), xin.grad] + [g.grad for pair in leaves for g in pair]

    first, second = step(), step()
    reels.check_device_status()
    for a, b in zip(first, second):
        assert a is not None and bool(torch.isfinite(a.float()).all()) and torch.equal(a, b)
        assert float(a.float().abs().max()) > 0


def test_gradient_against_differences(torch, reels):
    c = ac.Case(1, 40, 33, 4, 2, 64, torch.float32, [30], seed=3)
    out, lse = reels.attention(c.q, c.k, c.v, kv_lengths=c.lengths, return_lse=True)
    grads = reels.attention_backward(c.dout, c.q, c.k, c.v, out, lse, kv_lengths=c.lengths)
    f = lambda q, k, v: float((reels.attention(q, k, v, kv_lengths=c.lengths).double() * c.dout.double()).sum())
    h = 2.0 ** -7  # truncation h^2 ~ 6e-5, rounding sqrt(10240) 2^-24 * 2 / h ~ 2e-3
    for i, at in ((0, (0, 3, 1, 5)), (0, (0, 39, 3, 63)), (1, (0, 2, 0, 7)), (1, (0, 29, 1, 0)), (2, (0, 5, 1, 9)),
                  (1, (0, 31, 0, 4)), (2, (0, 30, 1, 1))):
        e = torch.zeros_like((c.q, c.k, c.v)[i])
        e[at] = h
        up, down = [c.q, c.k, c.v], [c.q, c.k, c.v]
        up[i], down[i] = up[i] + e, down[i] - e
        assert float(grads[i][at]) == pytest.approx((f(*up) - f(*down)) / (2 * h), rel=5e-3, abs=5e-3)


@pytest.mark.parametrize("Sq,Sk,D,dtype", [(300, 400, 128, "bfloat16"), (300, 400, 64, "float16"), (2, 400, 128, "bfloat16"),
                                           (90, 100, 64, "float32")])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf")])
def test_what_lies_behind_a_length_has_no_part(torch, reels, Sq, Sk, D, dtype, junk):
    lengths = [Sk // 2 + 3, 1, 0]
    c = ac.Case(3, Sq, Sk, 2, 2, D, getattr(torch, dtype), lengths, seed=4)
    dead = torch.arange(Sk, device="cuda")[None, :] >= c.lengths[:, None]
    runs = []
    for fill in (0.0, junk):
        k, v = c.k.clone(), c.v.clone()
        k[dead], v[dead] = fill, fill
        out, lse = reels.attention(c.q, k, v, kv_lengths=c.lengths, return_lse=True)
        runs.append((out, lse, *reels.attention_backward(c.dout, c.q, k, v, out, lse, kv_lengths=c.lengths)))
    reels.check_device_status()
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    out, lse, dq, dk, dv = runs[1]
    assert bool((dk[dead] == 0).all()) and bool((dv[dead] == 0).all())
    assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all()) and bool((dq[2] == 0).all())
    assert all(bool(torch.isfinite(t.float()).all()) for t in (out, dq, dk, dv))


def test_nan_reaches_what_it_should(torch, reels):
    c = ac.Case(1, 200, 300, 2, 2, 128, torch.bfloat16, seed=5)
    c.q[0, 7, 0] = float("nan")
    out = reels.attention(c.q, c.k, c.v)
    bad = torch.isnan(out.float()).any(-1)
    assert bool(bad[0, 7, 0]) and int(bad.sum()) == 1
    c.k[0, 250, 1, 3] = float("nan")  # a key of the other head: all its rows
    bad = torch.isnan(reels.attention(c.q, c.k, c.v).float()).any(-1)
    assert bool(bad[0, :, 1].all()) and int(bad[0, :, 0].sum()) == 1


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_keep_rising(torch, reels, dtype, rising):
    """The running maximum grows by more than its lag in every tile: O is rescaled throughout."""
    c = ac.Case(1, 260, 700, 2, 2, 128, getattr(torch, dtype), seed=6, spread=1.0)
    ramp = torch.linspace(0.0, 14.0, 700, device="cuda")
    c.k[..., 0] = (ramp if rising else ramp.flip(0)).to(c.k.dtype)[None, :, None]
    c.q[..., 0] = 14.0
    out, lse = reels.attention(c.q, c.k, c.v, return_lse=True)
    want = ac.reference(c)
    ac.check("out", out, want["out"])
    ac.check("lse", lse, want["lse"])
    for name, got in zip(("dq", "dk", "dv"), reels.attention_backward(c.dout, c.q, c.k, c.v, out, lse)):
        ac.check(name, got, want[name])


@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** 10])
def test_fp16_gradients_keep_their_range(torch, reels, size):
    """Probabilities of 1 / 3000 times small gradients would vanish in fp16,
    large ones overflow: dS is held by a power of two in between."""
    c = ac.Case(1, 256, 3000, 1, 1, 64, torch.float16, seed=7, spread=0.5)
    c.dout = (c.dout.float() * size).half()
    out, lse = reels.attention(c.q, c.k, c.v, return_lse=True)
    want = ac.reference(c)
    for name, got in zip(("dq", "dk", "dv"), reels.attention_backward(c.dout, c.q, c.k, c.v, out, lse)):
        ac.check(name, got, want[name])


@pytest.mark.parametrize("dtype,Sq", [("bfloat16", 150), ("bfloat16", 1), ("float32", 20)])
def test_offsets_past_32_bits(torch, reels, dtype, Sq):
    """Keys 2^20 elements apart: the last lie more than 2^31 elements in."""
    dt = getattr(torch, dtype)
    Sk, D, pitch = 2200, 64, 1 << 20
    store = torch.empty(Sk * pitch, dtype=dt, device="cuda")
    far = store.as_strided((1, Sk, 2, 2, D), (Sk * pitch, pitch, 2 * D, D, 1))
    c = ac.Case(1, Sq, Sk, 2, 2, D, dt, seed=8)
    far[:, :, 0], far[:, :, 1] = c.k, c.v
    k, v = far[:, :, 0], far[:, :, 1]
    near = reels.attention(c.q, c.k, c.v, return_lse=True)
    got = reels.attention(c.q, k, v, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(near, got))
    a = reels.attention_backward(c.dout, c.q, c.k, c.v, *near)
    b = reels.attention_backward(c.dout, c.q, k, v, *got)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_strides_the_kernels_cannot_follow_are_copied(torch, reels):
    c = ac.Case(2, 140, 150, 2, 2, 128, torch.bfloat16, seed=9)
    want = reels.attention(c.q, c.k, c.v)
    odd = torch.empty((2, 150, 2, 131), dtype=torch.bfloat16, device="cuda")[..., 1:129]
    odd.copy_(c.k)
    assert torch.equal(reels.attention(c.q, odd, c.v), want)
    swapped = c.v.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(reels.attention(c.q, c.k, swapped), want)
    one = c.k[:1].expand(2, -1, -1, -1)  # a broadcast sample
    assert torch.equal(reels.attention(c.q, one, c.v), reels.attention(c.q, one.contiguous(), c.v))


def test_empty_and_out_of_range_lengths(torch, reels):
    c = ac.Case(2, 30, 40, 2, 2, 64, torch.bfloat16, seed=10)
    none = c.k[:, :0]
    out, lse = reels.attention(c.q, none, none, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    dq, dk, dv = reels.attention_backward(c.dout, c.q, none, none, out, lse)
    assert bool((dq == 0).all()) and dk.shape == none.shape
    assert reels.attention(c.q[:, :0], c.k, c.v).shape == (2, 0, 2, 64)
    lengths = torch.tensor([2 ** 40, -5], device="cuda")
    got = reels.attention(c.q, c.k, c.v, kv_lengths=lengths)
    want = reels.attention(c.q, c.k, c.v, kv_lengths=torch.tensor([40, 0], device="cuda", dtype=torch.int32))
    assert torch.equal(got, want)
    wild = torch.tensor([2 ** 30, -7], device="cuda", dtype=torch.int32)
    assert torch.equal(reels.attention(c.q, c.k, c.v, kv_lengths=wild), want)


def test_refusals_of_the_python_layer(torch, reels):
    t = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device="cuda")
    q, k = t(2, 4, 4, 64), t(2, 5, 2, 64)
    for bad, word in (((q[0], k, k), "batch, tokens"), ((q, k, k[:, :4]), "same shape"), ((q, k[:1], k[:1]), "batch"),
                      ((q, t(2, 5, 3, 64), t(2, 5, 3, 64)), "multiple"), ((q, k.half(), k.half()), "dtype"),
                      ((q.double(), k.double(), k.double()), "precision")):
        with pytest.raises(ValueError, match=word):
            reels.attention(*bad)
    with pytest.raises(ValueError, match="scale"):
        reels.attention(q, k, k, scale=-1.0)
    with pytest.raises(ValueError, match="head_dim"):
        reels.attention(t(1, 4, 1, 264), t(1, 4, 1, 264), t(1, 4, 1, 264))
    with pytest.raises(ValueError, match="one integer"):
        reels.attention(q, k, k, kv_lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="lengths|CUDA"):
        reels.attention(q, k, k, kv_lengths=torch.zeros(2, dtype=torch.int32))
    out, lse = reels.attention(q, k, k, return_lse=True)
    with pytest.raises(ValueError, match="lse"):
        reels.attention_backward(q, q, k, k, out, lse.bfloat16())
    with pytest.raises(ValueError, match="shape of q"):
        reels.attention_backward(q[:, :3], q, k, k, out, lse)
    x = t(2, 4, 256)
    rope = reels.rope_table(64, (1, 2, 2))
    for kw, word in ((dict(heads=3), "heads"), (dict(heads=2, rope=rope), "sum"),
                     (dict(heads=4, weight=t(255)), "entries"), (dict(heads=4, positions=t(2, 4, 3).int()), "table"),
                     (dict(heads=4, rope=rope, positions=t(2, 3, 3).int()), "row"),
                     (dict(heads=4, tokens_per_sample=0), "positive"), (dict(heads=4, epsilon=float("nan")), "epsilon")):
        with pytest.raises(ValueError, match=word):
            reels.rms_norm_rope(x, **kw)
    with pytest.raises(ValueError, match="shape, dtype"):
        reels.rms_norm_rope_backward(x, x.half(), 4)


def test_captured_graphs_and_other_streams(torch, reels):
    """Forward and backward captured twice (a graph each, on one stream),
    replayed side by side on two streams on new data, against eager calls."""
    shapes = [(1, 300, 500, 4, 2, 128, torch.bfloat16), (2, 1, 700, 2, 2, 64, torch.float16)]
    cases = [ac.Case(*s, seed=11 + i) for i, s in enumerate(shapes)]
    x = torch.randn((1, 300, 512), device="cuda").bfloat16()
    rope = reels.rope_table(128, (3, 10, 10))

    def run(c):
        out, lse = reels.attention(c.q, c.k, c.v, return_lse=True)
        return (out, lse, *reels.attention_backward(c.dout, c.q, c.k, c.v, out, lse),
                reels.rms_norm_rope_backward(x, reels.rms_norm_rope(x, 4, None, rope), 4, None, rope))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for c in cases:
            run(c)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                kept = run(c)
            graphs.append((g, kept))
    torch.cuda.synchronize()
    for c in cases:
        for t in (c.q, c.k, c.v, c.dout):
            t.copy_(torch.randn_like(t, dtype=torch.float32).to(t.dtype))
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    reels.check_device_status()
    for (_, kept), ref in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(kept, ref))


def test_current_device_is_kept_and_the_c_calls_take_any_stream(torch, reels):
    import ctypes
    from reels_b200 import _native as nat
    c = ac.Case(1, 64, 64, 2, 2, 64, torch.float16, seed=13)
    want, lse = reels.attention(c.q, c.k, c.v, return_lse=True)
    s = torch.cuda.Stream()
    out, l2 = torch.empty_like(want), torch.empty_like(lse)
    i3 = ctypes.c_int64 * 3
    st = i3(*c.q.stride()[:3])
    shape = nat.AttnShape(1, 2, 2, 64, 64, 64, st, st, st)
    torch.cuda.synchronize()
    nat.check("forward", nat.lib().reels_attention_forward(
        ctypes.byref(shape), c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), None, 64 ** -0.5, nat.F16,
        out.data_ptr(), l2.data_ptr(), None, 0, s.cuda_stream))
    s.synchronize()
    assert torch.cuda.current_device() == 0 and torch.equal(out, want) and torch.equal(l2, lse)


def test_a_second_derivative_is_refused(torch, reels):
    """The gradients carry no graph of their own: differentiating them raises."""
    q, k, v = (torch.randn((1, 8, 2, 64), device="cuda", requires_grad=True) for _ in range(3))
    dq, = torch.autograd.grad(reels.AttentionFunction.apply(q, k, v).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dq.sum().backward()
    x = torch.randn((4, 128), device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(reels.RMSNormRopeFunction.apply(x, 2).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_calls_of_several_threads(torch, reels):
    """Two widths of one kernel's form, whose launches need different amounts
    of shared memory, from two threads at once: the results of the calls made alone."""
    import threading
    xs = [torch.randn((64, c), device="cuda").bfloat16() for c in (1536, 5120)]
    douts = [torch.randn_like(x) for x in xs]
    run = lambda i: (reels.rms_norm_rope(xs[i], 12 if i == 0 else 40),
                     reels.rms_norm_rope_backward(xs[i], douts[i], 12 if i == 0 else 40))
    want, bad = [run(0), run(1)], []
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(300):
                    got = run(i)
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                bad.append((i, "differs"))
        except Exception as e:  # reported below, by the test's own thread
            bad.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("Sq,H,D,dtype,length", [(1, 1, 128, "bfloat16", None), (1, 1, 64, "float16", 9001),
                                                 (2, 1, 128, "bfloat16", 70), (20, 1, 64, "float32", 12000)])
def test_many_key_splits(torch, reels, Sq, H, D, dtype, length):
    """More splits than a warp has lanes, some of them behind the sample's length."""
    import ctypes
    from reels_b200 import _native as nat
    Sk = 20011
    c = ac.Case(1, Sq, Sk, H, H, D, getattr(torch, dtype), None if length is None else [length], seed=17)
    i3 = ctypes.c_int64 * 3
    shape = nat.AttnShape(1, H, H, Sq, Sk, D, i3(*c.q.stride()[:3]), i3(*c.k.stride()[:3]), i3(*c.v.stride()[:3]))
    info, types = (ctypes.c_int64 * 4)(), {"bfloat16": nat.BF16, "float16": nat.F16, "float32": nat.F32}
    nat.check("plan", nat.lib().reels_attention_plan(ctypes.byref(shape), types[dtype], info))
    assert info[1] > 32
    out, lse = reels.attention(c.q, c.k, c.v, kv_lengths=c.lengths, return_lse=True)
    want = ac.reference(c, backward=False)
    ac.check("out", out, want["out"])
    ac.check("lse", lse, want["lse"])
