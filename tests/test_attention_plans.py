"""CPU checks of the forward's plans for few query rows."""
import ctypes

import pytest

from reels_b200 import _native as nat
from reels_b200 import build as native_build


@pytest.mark.parametrize("rows", range(1, 9))
@pytest.mark.parametrize("kv_heads,D", [(1, 128), (12, 128), (24, 64), (40, 128)])
def test_key_splits_of_few_rows_run_at_once(rows, kv_heads, D):
    """Two blocks of the few-row kernel fit an SM with one or two rows, one
    with more: no split waits for another to end."""
    native_build.build()
    i3 = ctypes.c_int64 * 3
    q, k = i3(rows * kv_heads * D, kv_heads * D, D), i3(32760 * kv_heads * D, kv_heads * D, D)
    shape = nat.AttnShape(1, kv_heads, kv_heads, rows, 32760, D, q, k, k)
    info = (ctypes.c_int64 * 4)()
    assert nat.lib().reels_attention_plan(ctypes.byref(shape), nat.BF16, info) == nat.OK
    assert info[0] == nat.PATH_CUDACORE and info[1] * kv_heads <= 148 * (2 if rows <= 2 else 1)
