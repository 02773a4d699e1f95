"""Token counts whose last tile ends several 32-token chunks early: every row
of Y and dX is the product's, also the last whole chunk before the end, whose
output tile the chunks behind it must not write over."""
import pytest

pytestmark = pytest.mark.gpu


# 2048: the last 192-token tile of dX holds 128 tokens; the others leave one,
# two or three chunks of a tile's half, or all but one token of it, without tokens
@pytest.mark.parametrize("M,K,N,r", [(2048, 1536, 8960, 32), (2049, 1536, 8960, 32), (2015, 8960, 1536, 32),
                                     (4128, 1536, 8960, 8), (1184, 5120, 5120, 16)])
def test_rows_before_the_end(M, K, N, r):
    import torch

    import lora_case as lc
    from reels_b200 import check_device_status, lora_backward, lora_forward, saved_buffer

    c = lc.make_case(M, K, N, r, dtype="bf16", layout=0, seed=M)
    layer = lc.device_layer(torch, c)
    x = torch.from_numpy(c.X).cuda().bfloat16()
    dy = torch.from_numpy(c.dY).cuda().bfloat16()
    W = layer.weight.values.double() * layer.weight.scales.double()[:, None]
    A, B, s, t = layer.A.double(), layer.B.double(), layer.alpha / r, slice(M - 256, M)
    y_ref = x[t].double() @ W.t() + s * (x[t].double() @ A.t()) @ B.t()
    dx_ref = dy[t].double() @ W + s * (dy[t].double() @ B) @ A
    cold = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = None
    for _ in range(8):
        junk = [torch.full((M, n), float("nan"), dtype=torch.bfloat16, device="cuda") for n in (K, N)]
        del junk
        cold.zero_()
        torch.cuda.synchronize()
        saved = saved_buffer(layer, x)
        y = lora_forward(layer, x, saved=saved)
        dx = lora_backward(layer, x, dy, saved=saved).dx
        torch.cuda.synchronize()
        check_device_status()
        # a chunk of 32 rows and columns at a time, so that none hides behind the others;
        # twice the bound of a whole output, for the spread of 1024 values about it
        for got, ref in ((y[t], y_ref), (dx[t], dx_ref)):
            off = (got.double() - ref).square().view(8, 32, -1, 32).sum((1, 3))
            size = ref.square().view(8, 32, -1, 32).sum((1, 3))
            assert float((off / size).max().sqrt()) <= 2 * lc.TOL
        first = (y, dx) if first is None else first
        assert torch.equal(y, first[0]) and torch.equal(dx, first[1])
