"""GPU tests of attention's range: fp16 gradients of parts whose sizes lie far
apart, scores of -infinity, fp16 gradients of few queries over many keys."""
import math
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


@pytest.fixture(scope="module")
def reels(torch):
    import reels_b200
    return reels_b200


def _part(c, b=slice(None), h=slice(None), hk=slice(None), rows=slice(None)):
    """A part of a case whose outputs do not depend on the rest, so that no
    term of its bounds is taken over more than the part."""
    return types.SimpleNamespace(q=c.q[b, rows, h], k=c.k[b, :, hk], v=c.v[b, :, hk], dout=c.dout[b, rows, h],
                                 dtype=c.dtype, scale=c.scale, lengths=None if c.lengths is None else c.lengths[b])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("over", ["samples", "heads", "rows"])
def test_fp16_gradients_of_sizes_far_apart(torch, reels, over, D):
    """Gradients of the output, or values, that differ by 2^20 from sample to
    sample, from key head to key head and (for dq) from row to row: the small
    ones keep their bits."""
    B, S, H, HK = 2, 1500, 4, 2
    c = ac.Case(B, S, S, H, HK, D, torch.float16, [S, S - 7], seed=21, spread=0.5)
    size = torch.ones((B, S, H, 1), device="cuda")
    if over == "samples":
        size[1] = 2.0 ** -20
    elif over == "heads":
        size[:, :, :2] = 2.0 ** -20
        c.v[:, :, 1] *= 2.0 ** 6
    else:
        size[:, ::3] = 2.0 ** -20
    c.dout = (c.dout.float() * 2.0 ** 8 * size).half()
    out, lse = reels.attention(c.q, c.k, c.v, kv_lengths=c.lengths, return_lse=True)
    dq, dk, dv = reels.attention_backward(c.dout, c.q, c.k, c.v, out, lse, kv_lengths=c.lengths)
    reels.check_device_status()
    for b in range(B):
        for g in range(HK):
            s, h, hk = slice(b, b + 1), slice(2 * g, 2 * g + 2), slice(g, g + 1)
            for rows in ((slice(0, None, 3), slice(1, None, 3), slice(2, None, 3)) if over == "rows" else (slice(None),)):
                ac.check("dq", dq[s, rows, h], ac.reference(_part(c, s, h, hk, rows))["dq"])
            want = ac.reference(_part(c, s, h, hk))
            ac.check("dk", dk[s, :, hk], want["dk"])
            ac.check("dv", dv[s, :, hk], want["dv"])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("Sq,Sk,D", [(300, 700, 128), (300, 700, 64), (2, 700, 128), (130, 5000, 64)])
@pytest.mark.parametrize("first", [True, False])
def test_tiles_of_scores_of_minus_infinity(torch, reels, Sq, Sk, D, dtype, first):
    """200 keys whose scores are -infinity, ahead of or behind keys with scores
    of about -1000: they have no weight, and do not stand for a maximum of 0."""
    n = 200
    c = ac.Case(1, Sq, Sk, 2, 2, D, getattr(torch, dtype), seed=22, spread=0.5)
    c.q[..., 0], c.q[..., 1] = 1.0, 32.0
    c.k[..., 0], c.k[..., 1] = 0.0, -32.0 * D ** 0.5
    gone = slice(0, n) if first else slice(Sk - n, Sk)
    live = slice(n, Sk) if first else slice(0, Sk - n)
    c.k[:, gone, :, 0] = -math.inf
    out, lse = reels.attention(c.q, c.k, c.v, return_lse=True)
    reels.check_device_status()
    c.k, c.v = c.k[:, live], c.v[:, live]
    want = ac.reference(c, backward=False)
    ac.check("lse", lse, want["lse"])
    ac.check("out", out, want["out"])


def test_fp16_gradient_of_few_queries_over_many_keys(torch, reels):
    """What fp16 needs beside bf16, the sizes of the rows of v, is read by as
    many blocks as there are rows: 16 queries over 9000 keys take about the
    time that bf16 takes."""
    times = {}
    runs = {}
    for dtype in (torch.bfloat16, torch.float16):
        c = ac.Case(1, 16, 9000, 12, 12, 128, dtype, seed=23)
        out, lse = reels.attention(c.q, c.k, c.v, return_lse=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            reels.attention_backward(c.dout, c.q, c.k, c.v, out, lse)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                kept = [reels.attention_backward(c.dout, c.q, c.k, c.v, out, lse) for _ in range(10)]
        runs[dtype] = (g, c, out, lse, kept)
    torch.cuda.synchronize()
    for _ in range(10):  # in turn, and the best of each: another load on the GPU slows both
        for dtype, (g, *_) in runs.items():
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            g.replay()
            end.record()
            end.synchronize()
            times[dtype] = min(times.get(dtype, math.inf), start.elapsed_time(end))
    assert times[torch.float16] <= 1.5 * times[torch.bfloat16], times


def test_the_last_of_two_billion_keys(torch, reels):
    """Key splits whose lengths add up to more than 32 bits: the last one counts too."""
    Sk = 2 ** 31 - 257
    q = torch.full((1, 1, 1, 1), 0.5, device="cuda")
    k = torch.full((1, 1, 1, 1), 2.0, device="cuda").expand(1, Sk, 1, 1)
    out, lse = reels.attention(q, k, k, scale=1.0, return_lse=True)
    # equal scores of 1: sums of whole numbers below 2^24 in a split, then 592 of them to fp32's rounding
    assert float(out) == pytest.approx(2.0, rel=1e-5)
    assert float(lse) == pytest.approx(1.0 + math.log(Sk), rel=1e-6)
