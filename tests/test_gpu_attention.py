"""GPU parity of attention and its gradient against plain 64-bit attention
(attention_case.py derives the elementwise bounds), at the sizes, layouts and
masks where the kernels can go wrong."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as _t
    from reels_b200 import build
    build.build()
    return _t


BF, HF, FL = "bfloat16", "float16", "float32"
CASES = [
    # B, Sq, Sk, H, HK, D, dtype, lengths, packed
    (1, 128, 128, 1, 1, 128, BF, None, False),    # one tile
    (1, 256, 128, 1, 1, 128, BF, None, False),    # both query tiles of a unit
    (1, 256, 384, 2, 2, 128, BF, None, False),    # several key tiles
    (1, 256, 384, 2, 2, 64, HF, None, False),
    (1, 1, 1, 1, 1, 128, BF, None, False),
    (2, 1, 4097, 3, 3, 128, BF, None, False),     # one row, key splits
    (3, 2, 300, 2, 2, 64, HF, [300, 0, 65], False),  # few rows: 2, 3, 4, 5, 8 a key head
    (1, 1, 129, 6, 2, 128, HF, None, False),
    (2, 2, 5000, 4, 2, 40, BF, [5000, 77], False),
    (1, 5, 63, 1, 1, 96, BF, None, False),
    (1, 4, 1000, 2, 1, 128, BF, [999], False),
    (1, 3, 3, 2, 2, 64, BF, None, True),
    (1, 130, 2051, 2, 1, 64, HF, None, False),    # few rows, key splits, shared heads
    (2, 129, 131, 3, 3, 128, HF, [131, 3], False),   # one past a tile; a short sample
    (3, 200, 300, 4, 2, 128, BF, [0, 300, 128], False),  # no keys; a whole tile exactly
    (2, 257, 257, 6, 6, 128, BF, None, True),     # parts of a fused projection
    (1, 300, 77, 8, 2, 64, BF, [50], False),
    (1, 100, 90, 3, 1, 80, BF, None, False),      # heads padded to 128
    (1, 100, 90, 2, 2, 40, HF, [89], False),      # heads padded to 64
    (1, 640, 200, 4, 4, 128, HF, None, False),    # dk, dv walk split
    (1, 70, 65, 2, 2, 36, BF, None, False),       # head size no multiple of 8
    (1, 45, 70, 2, 2, 192, BF, [33], False),      # large heads
    (2, 63, 65, 4, 2, 64, FL, [65, 0], False),
    (1, 33, 31, 2, 2, 128, FL, None, False),
    (1, 40, 50, 1, 1, 256, FL, None, False),
    (1, 5, 3000, 1, 1, 64, FL, None, False),      # key splits on the CUDA cores
    (1, 50, 50, 3, 3, 64, FL, None, True),
    (2, 130, 200, 60, 30, 64, FL, [200, 7], False),  # the larger tile on the CUDA cores
    (1, 70, 65, 200, 200, 100, FL, None, False),
    (1, 190, 90, 100, 100, 36, HF, None, False),
]


@pytest.mark.parametrize("B,Sq,Sk,H,HK,D,dtype,lengths,packed", CASES)
def test_parity(torch, B, Sq, Sk, H, HK, D, dtype, lengths, packed):
    import attention_case as ac
    from reels_b200 import _native as nat
    from reels_b200 import attention, attention_backward, check_device_status
    c = ac.Case(B, Sq, Sk, H, HK, D, getattr(torch, dtype), lengths, packed, seed=Sq + Sk)
    out, lse = attention(c.q, c.k, c.v, kv_lengths=c.lengths, return_lse=True)
    check_device_status()
    tc = dtype != FL and D % 8 == 0 and D <= 128 and Sq * H // HK > 8
    assert nat.last_path() == (nat.PATH_TENSORCORE if tc else nat.PATH_CUDACORE)
    want = ac.reference(c)
    ac.check("out", out, want["out"])
    ac.check("lse", lse, want["lse"])
    dq, dk, dv = attention_backward(c.dout, c.q, c.k, c.v, out, lse, kv_lengths=c.lengths)
    check_device_status()
    for name, got in (("dv", dv), ("dk", dk), ("dq", dq)):
        ac.check(name, got, want[name])
    again = attention_backward(c.dout, c.q, c.k, c.v, out, lse, kv_lengths=c.lengths)
    assert all(torch.equal(x, y) for x, y in zip((dq, dk, dv), again))
