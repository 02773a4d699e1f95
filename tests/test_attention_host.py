"""CPU checks of the attention stretch's C ABI and Python layer: refusals
before anything is launched, empty inputs, plans and workspace sizes."""
import ctypes

import pytest

from reels_b200 import _native as nat
from reels_b200 import build as native_build

P = ctypes.c_void_p(0x1000)  # never dereferenced: checks run first


@pytest.fixture(scope="module")
def lib():
    native_build.build()
    return nat.lib()


def _shape(B=1, H=2, HK=2, Sq=256, Sk=256, D=128, **strides):
    i3 = ctypes.c_int64 * 3
    s = dict(q=(Sq * H * D, H * D, D), k=(Sk * HK * D, HK * D, D), v=(Sk * HK * D, HK * D, D))
    s.update(strides)
    return nat.AttnShape(B, H, HK, Sq, Sk, D, i3(*s["q"]), i3(*s["k"]), i3(*s["v"]))


def _rope(size=(2, 3, 4), dim=(44, 42, 42), table=0x1000, pairing=0):
    i3 = ctypes.c_int32 * 3
    return nat.Rope(table, None, i3(*size), i3(*dim), pairing)


def _err(lib):
    return lib.reels_lowvram_last_error().decode()


def test_norm_rope_rejects_bad_arguments(lib):
    def fwd(x=P, M=4, H=2, D=128, w=None, rope=None, tps=4, eps=1e-6, dt=nat.BF16, out=P):
        return lib.reels_rms_norm_rope(x, M, H, D, w, None if rope is None else ctypes.byref(rope), tps, eps, dt, out,
                                       None)

    bad = [dict(x=None), dict(M=-1), dict(H=0), dict(D=0), dict(H=129), dict(H=1 << 40, D=1 << 40), dict(tps=0),
           dict(eps=float("nan")), dict(eps=-1.0), dict(dt=9), dict(out=None)]
    for b in bad:
        assert fwd(**b) == nat.EINVAL and _err(lib), b
    for r, word in ((_rope(table=0), "table"), (_rope(table=0x1004), "aligned"), (_rope(dim=(44, 42, 40)), "sum"),
                    (_rope(dim=(43, 43, 42)), "even"), (_rope(size=(0, 3, 4)), "size"), (_rope(pairing=2), "pairing"),
                    (_rope(size=(1 << 30, 1 << 30, 4)), "large")):
        assert fwd(rope=r) == nat.EINVAL and word in _err(lib), word
    assert fwd(D=7, rope=_rope(dim=(3, 2, 2))) == nat.EINVAL
    bwd = lambda x, dout, dx: lib.reels_rms_norm_rope_backward(x, dout, 4, 2, 128, None, None, 4, 1e-6, nat.BF16, dx,
                                                               None)
    assert bwd(P, None, P) == nat.EINVAL and "dout" in _err(lib)
    assert bwd(P, P, None) == nat.EINVAL and "dx" in _err(lib)
    # no tokens: nothing is read
    assert fwd(x=None, M=0, out=None) == nat.OK


def _forward(lib, s, q=P, k=P, v=P, scale=0.1, dt=nat.BF16, out=P, lse=P, ws=None, wsn=0):
    return lib.reels_attention_forward(None if s is None else ctypes.byref(s), q, k, v, None, scale, dt, out, lse, ws,
                                       wsn, None)


def _backward(lib, s, q=P, k=P, v=P, out=P, lse=P, dout=P, scale=0.1, dt=nat.BF16, dq=P, dk=P, dv=P, ws=None, wsn=0):
    return lib.reels_attention_backward(ctypes.byref(s), q, k, v, out, lse, dout, None, scale, dt, dq, dk, dv, ws, wsn,
                                        None)


def test_attention_rejects_bad_arguments(lib):
    assert _forward(lib, None) == nat.EINVAL
    for b in (dict(H=3, HK=2), dict(H=0), dict(HK=0), dict(D=0), dict(D=257), dict(B=-1), dict(Sq=-1), dict(Sk=-1),
              dict(B=1 << 20, H=1 << 20, HK=1 << 20), dict(Sq=1 << 40), dict(q=(-1, 256, 128))):
        s = _shape(**b)
        assert _forward(lib, s) == nat.EINVAL and _err(lib), b
        assert _backward(lib, s) == nat.EINVAL, b
        assert lib.reels_attention_workspace_bytes(ctypes.byref(s), nat.BF16, nat.PASS_BACKWARD) == 0, b
    s = _shape()
    for b in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(lse=None), dict(scale=0.0),
              dict(scale=-1.0), dict(scale=float("inf")), dict(dt=7)):
        assert _forward(lib, s, **b) == nat.EINVAL and _err(lib), b
    for b in (dict(q=None), dict(k=None), dict(out=None), dict(lse=None), dict(dout=None), dict(dq=None),
              dict(dk=None), dict(dv=None), dict(scale=float("nan"))):
        assert _backward(lib, s, **b) == nat.EINVAL and _err(lib), b
    # the backward always needs scratch; it has to be large enough and aligned
    need = lib.reels_attention_workspace_bytes(ctypes.byref(s), nat.BF16, nat.PASS_BACKWARD)
    assert need > 0
    assert _backward(lib, s) == nat.EINVAL and "workspace" in _err(lib)
    assert _backward(lib, s, ws=P, wsn=need - 1) == nat.EINVAL and "small" in _err(lib)
    assert _backward(lib, s, ws=ctypes.c_void_p(0x1010), wsn=need) == nat.EINVAL and "aligned" in _err(lib)


def test_empty_attention_needs_no_gpu(lib):
    assert _forward(lib, _shape(B=0), q=None, k=None, v=None, out=None, lse=None) == nat.OK
    assert _forward(lib, _shape(Sq=0), q=None, out=None, lse=None) == nat.OK
    assert _backward(lib, _shape(B=0), q=None, k=None, v=None, out=None, lse=None, dout=None, dq=None, dk=None,
                     dv=None) == nat.OK


def _plan(lib, s, dt=nat.BF16):
    info = (ctypes.c_int64 * 4)()
    assert lib.reels_attention_plan(ctypes.byref(s), dt, info) == nat.OK
    return list(info)


def test_attention_plans(lib):
    # which kernels run: type, head size, strides
    assert _plan(lib, _shape())[0] == nat.PATH_TENSORCORE
    assert _plan(lib, _shape(), nat.F32)[0] == nat.PATH_CUDACORE
    assert _plan(lib, _shape(D=36))[0] == nat.PATH_CUDACORE
    assert _plan(lib, _shape(D=136))[0] == nat.PATH_CUDACORE
    assert _plan(lib, _shape(q=(256 * 256, 258, 128)))[0] == nat.PATH_CUDACORE
    assert _plan(lib, _shape(k=(256 * 256, 0, 128)))[0] == nat.PATH_CUDACORE
    # the strides of dimensions of one entry do not count
    assert _plan(lib, _shape(q=(3, 256, 128)))[0] == nat.PATH_TENSORCORE
    # key splits cover the keys, none is empty, and only few rows are split
    for Sq, Sk, H in ((1, 32760, 12), (130, 2051, 2), (1, 100, 1), (300, 5000, 1), (32760, 32760, 12), (1, 1, 1)):
        for dt in (nat.BF16, nat.F32):
            path, splits, keys, _ = _plan(lib, _shape(Sq=Sq, Sk=Sk, H=H, HK=H), dt)
            assert splits >= 1 and splits * keys >= Sk and (splits - 1) * keys < Sk
            rows = -(-Sq // (256 if path == nat.PATH_TENSORCORE else 32)) * H
            assert splits == 1 or splits * rows <= (148 if path == nat.PATH_TENSORCORE else 592)
    # the walk for dk and dv: never more ranges than steps
    for Sq, Sk, H, HK in ((8190, 512, 40, 40), (1285, 1285, 10, 2), (100, 5000, 4, 4), (6144, 6144, 32, 32)):
        n = _plan(lib, _shape(Sq=Sq, Sk=Sk, H=H, HK=HK))[3]
        steps = H // HK * -(-Sq // 128)
        per = -(-steps // n)
        assert 1 <= n <= steps and (n - 1) * per < steps <= n * per


def test_python_layer_refusals():
    import torch
    import reels_b200 as reels
    t = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt)
    with pytest.raises(ValueError, match="CUDA"):
        reels.attention(t(1, 4, 2, 8), t(1, 4, 2, 8), t(1, 4, 2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        reels.rms_norm_rope(t(4, 16), 2)
    with pytest.raises(ValueError, match="shape"):
        reels.RopeTable(t(10, 2, dt=torch.float32), (2, 2, 2), (4, 4, 4))
    with pytest.raises(ValueError, match="even"):
        reels.RopeTable(t(10, 2, dt=torch.float32), (2, 2, 2), (4, 3, 5))
    with pytest.raises(ValueError, match="axes"):
        reels.RopeTable(t(10, 2, dt=torch.float32), (2,) * 4, (4,) * 4)
    with pytest.raises(ValueError, match="sum"):
        reels.rope_table(64, (2, 2, 2), (20, 20, 20), device="cpu")
    table = reels.rope_table(128, (3, 4, 5), device="cpu")
    assert table.dims == (44, 42, 42) and table.head_dim == 128
    assert tuple(table.table.shape) == (3 * 22 + 4 * 21 + 5 * 21, 2)
    # position 2 of the time axis, its second pair: angle 2 * 10000 ** (-2 / 44)
    angle = 2 * 10000.0 ** (-2 / 44)
    got = table.table[2 * 22 + 1].double()
    want = torch.tensor([angle], dtype=torch.float64)
    assert abs(float(got[0] - want.cos())) < 2 ** -24 and abs(float(got[1] - want.sin())) < 2 ** -24


def test_every_programmatic_kernel_waits_first():
    """The rule of test_pdl_order.py for the kernels of attention.cu: each
    waits for the kernel ahead of it before any return."""
    import os
    import re
    import test_pdl_order as rule
    srcs = rule._sources()
    names = set(re.findall(r"host_launch_pdl\(\s*([A-Za-z_]\w*)", srcs["attention.cu"]))
    if "kern" in names:  # a variable: the kernels it is set to
        names = names - {"kern"} | set(re.findall(r"\bkern = (\w+)<", srcs["attention.cu"]))
    assert len(names) >= 9
    for name in sorted(names):
        body = next(b for b in (rule._kernel_body(s, name) for s in srcs.values()) if b)
        w = body.find("griddep_wait()")
        assert w >= 0 and "return" not in body[:w], name
