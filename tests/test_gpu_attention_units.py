"""GPU parity of attention and its gradient where a block of the tensor-core
kernels works through several units: odd tiles and samples without keys among
them, and calls that launch the two walks of the gradient apart."""
import types

import pytest

import attention_case as ac

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as _t
    from reels_b200 import build
    build.build()
    return _t


BF, HF = "bfloat16", "float16"
CASES = [
    # B, Sq, Sk, H, HK, D, dtype, lengths, packed
    (3, 385, 260, 40, 20, 64, BF, [260, 0, 131], False),   # 2 units a sample and head, the last of one tile
    (3, 385, 260, 40, 20, 128, BF, [260, 0, 131], False),
    (3, 385, 260, 40, 20, 64, HF, [260, 0, 131], False),
    (3, 385, 260, 40, 20, 128, HF, [260, 0, 131], False),
    (4, 130, 520, 48, 48, 128, HF, [0, 520, 1, 384], False),  # one short tile a unit's second half
    (5, 100, 300, 37, 37, 128, BF, [300, 129, 0, 128, 1], False),  # units of one tile
    (2, 700, 513, 33, 11, 64, BF, None, False),
    (2, 1300, 1300, 64, 64, 64, BF, None, True),            # 1408 units of each walk: launched apart
    (2, 1290, 1270, 64, 64, 128, HF, [1270, 900], False),
    (9, 1024, 257, 50, 50, 64, HF, [257, 256, 255, 129, 128, 127, 1, 0, 257], False),
]


@pytest.mark.parametrize("B,Sq,Sk,H,HK,D,dtype,lengths,packed", CASES)
def test_parity(torch, B, Sq, Sk, H, HK, D, dtype, lengths, packed):
    from reels_b200 import _native as nat
    from reels_b200 import attention, attention_backward, check_device_status
    c = ac.Case(B, Sq, Sk, H, HK, D, getattr(torch, dtype), lengths, packed, seed=Sq + Sk + D)
    tiles = lambda n: -(-n // 128)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert -(-Sq // 256) * B * H > sms or tiles(Sq) * B * H > sms  # what the case is for
    out, lse = attention(c.q, c.k, c.v, kv_lengths=c.lengths, return_lse=True)
    assert nat.last_path() == nat.PATH_TENSORCORE
    dq, dk, dv = attention_backward(c.dout, c.q, c.k, c.v, out, lse, kv_lengths=c.lengths)
    check_device_status()
    again = attention_backward(c.dout, c.q, c.k, c.v, out, lse, kv_lengths=c.lengths)
    assert all(torch.equal(x, y) for x, y in zip((dq, dk, dv), again))
    group = H // HK
    per = max(1, 16 // group)  # key heads at a time: the 64-bit scores of all would take many GB
    for g in range(0, HK, per):
        hk, h = slice(g, g + per), slice(g * group, (g + per) * group)
        part = types.SimpleNamespace(q=c.q[:, :, h], k=c.k[:, :, hk], v=c.v[:, :, hk], dout=c.dout[:, :, h],
                                     dtype=c.dtype, scale=c.scale, lengths=c.lengths)
        want = ac.reference(part)
        for name, got in (("out", out[:, :, h]), ("lse", lse[:, h]), ("dv", dv[:, :, hk]), ("dk", dk[:, :, hk]),
                          ("dq", dq[:, :, h])):
            ac.check(name, got, want[name])
