"""The block's attention stretch, between the q/k/v projections and the
output projection: the norm of q and k with the video's rotary positions, and
softmax attention, forward and backward.

Activations are tokens-first like everywhere in this package.  The norm takes
what the projections return, ``(batch, tokens, heads * head_dim)``; attention
takes views of it by head, ``(batch, tokens, heads, head_dim)``, and reads
parts of a fused q/k/v projection in place.  All arithmetic runs in
libreels_lowvram.so on the GPU; sums, softmax statistics and norms are fp32
and every output is rounded once.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .lowvram import _check_numel, _dt, _ptr, _require_cuda

# These calls are a few microseconds of GPU work on small clips, so the host's
# way to the launch counts: the raw stream handle without a Stream object, and
# no view or copy of what is contiguous already.
_raw_stream = torch._C._cuda_getCurrentRawStream


def _stream(device) -> int:
    return _raw_stream(device.index)


# ------------------------------------------------------ norm and rotation
_ROPE_AXES = {}  # (sizes, dims, interleaved) -> table entries, head_dim, the C arrays


def _rope_axes(sizes, dims, interleaved):
    sizes, dims = [int(s) for s in sizes], [int(d) for d in dims]
    if len(sizes) != len(dims) or not 1 <= len(sizes) <= 3:
        raise ValueError("a rotary table has one to three axes, each with a size and a number of features")
    if min(sizes) <= 0 or min(dims) < 0 or any(d % 2 for d in dims):
        raise ValueError("a rotary axis needs a positive size and an even number of features")
    # fewer axes: the missing outer ones have one position and no features
    pad = 3 - len(sizes)
    i3 = ctypes.c_int32 * 3
    args = (i3(*([1] * pad), *sizes), i3(*([0] * pad), *dims),
            nat.ROPE_INTERLEAVED if interleaved else nat.ROPE_HALF)
    return sum(s * d // 2 for s, d in zip(sizes, dims)), sum(dims), args


class RopeTable:
    """Rotary positions of a video: ``table`` (entries, 2) holds (cos, sin) of
    the angles, axis after axis (time, height, width) as
    ``[sizes[a]][dims[a] / 2]`` rows, fp32 on the device.  ``dims`` are the
    features of a head that turn with each axis and sum to head_dim.
    ``interleaved`` pairs features (2i, 2i + 1) of a head, otherwise
    (i, i + head_dim / 2).  Build one with :func:`rope_table` and keep it for
    all blocks and steps of a resolution."""

    __slots__ = ("table", "sizes", "dims", "interleaved", "head_dim", "_args")

    def __init__(self, table: torch.Tensor, sizes: Sequence[int], dims: Sequence[int], interleaved: bool = True):
        key = (tuple(sizes), tuple(dims), bool(interleaved))
        known = _ROPE_AXES.get(key)
        if known is None:
            known = _rope_axes(*key)
            if len(_ROPE_AXES) >= 4096:
                _ROPE_AXES.clear()
            _ROPE_AXES[key] = known
        self.sizes, self.dims, self.interleaved = key
        entries, self.head_dim, self._args = known
        if table.dtype != torch.float32 or table.shape != (entries, 2) or not table.is_contiguous():
            raise ValueError(f"the rotary table must be contiguous fp32 of shape ({entries}, 2)")
        self.table = table


def rope_table(head_dim: int, sizes: Sequence[int], dims: Optional[Sequence[int]] = None, base: float = 10000.0,
               interleaved: bool = True, device=None) -> RopeTable:
    """(cos, sin) of ``position * base ** (-2i / dims[axis])``, computed in 64
    bits and rounded once.  ``sizes``: positions of each axis (time, height,
    width).  ``dims`` defaults to a third of the head's pairs for each of
    height and width and the rest for time (44, 42, 42 of 128)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if dims is None:
        if len(sizes) != 3:
            raise ValueError("dims are needed for other than three axes")
        side = 2 * (head_dim // 6)
        dims = (head_dim - 2 * side, side, side)
    if sum(dims) != head_dim:
        raise ValueError("the rotary axes' features must sum to head_dim")
    rows = []
    for size, dim in zip(sizes, dims):
        if dim < 0 or dim % 2:
            raise ValueError("a rotary axis needs a positive size and an even number of features")
        freq = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / max(dim, 1))
        angle = torch.arange(size, dtype=torch.float64, device=dev)[:, None] * freq
        rows.append(torch.stack((angle.cos(), angle.sin()), -1).reshape(-1, 2))
    return RopeTable(torch.cat(rows).float().contiguous(), sizes, dims, interleaved)


def _norm_rope_args(x, heads, weight, rope, tokens_per_sample, positions):
    _require_cuda(x, weight)
    C = x.shape[-1]
    heads = int(heads)
    if heads <= 0 or C == 0 or C % heads:
        raise ValueError("the features must be heads * head_dim")
    # (a weight has an entry for each feature, a table's axes sum to head_dim: they tell the two apart)
    if x.dim() == 4 and x.shape[-2] == heads > 1 and weight is None and rope is None and tokens_per_sample is None:
        raise ValueError("x looks like a view by head, but the norm spans all heads: pass (..., tokens, heads * "
                         "head_dim), or tokens_per_sample if these are tokens")
    xf = x if x.is_contiguous() else x.contiguous()
    M = x.numel() // C
    w, dt = weight, _dt(x.dtype)
    if w is not None:
        _check_numel(w, C, "norm weight", x.device)
        if w.dtype != x.dtype:  # fp32 holds what the other types hold
            w, dt = w.float(), dt | nat.NORM_WEIGHT_F32
        w = w.contiguous()
    if tokens_per_sample is None:
        tps = x.shape[-2] if x.dim() >= 2 else 1
    else:
        tps = int(tokens_per_sample)
        if tps <= 0:
            raise ValueError("tokens_per_sample must be positive")
    r, pos = None, None
    if rope is not None:
        if rope.head_dim != C // heads:
            raise ValueError("the rotary axes' features must sum to head_dim")
        if rope.table.device != x.device:
            raise ValueError(f"the rotary table is on {rope.table.device}, the input on {x.device}")
        if positions is not None:
            axes = len(rope.sizes)
            if positions.dtype not in (torch.int32, torch.int64) or positions.device != x.device:
                raise ValueError("positions must be integers on the input's device")
            if positions.shape[-1] != axes or positions.numel() != M * axes:
                raise ValueError(f"positions must have one row of {axes} for each of the {M} tokens")
            pos = positions.reshape(M, axes)
            if pos.dtype == torch.int64:  # what 32 bits do not hold stays outside every table
                pos = pos.clamp(-1, 2 ** 31 - 1).to(torch.int32)
            if axes < 3:  # the missing outer axes stand at their only position
                pos = torch.nn.functional.pad(pos, (3 - axes, 0))
            pos = pos.contiguous()
        sizes, dims, pairing = rope._args
        r = ctypes.byref(nat.Rope(rope.table.data_ptr(), _ptr(pos), sizes, dims, pairing))
    elif positions is not None:
        raise ValueError("positions need a rotary table")
    return xf, M, heads, C // heads, w, r, max(tps, 1), pos, dt


def rms_norm_rope(x: torch.Tensor, heads: int, weight: Optional[torch.Tensor] = None,
                  rope: Optional[RopeTable] = None, epsilon: float = 1e-6, tokens_per_sample: Optional[int] = None,
                  positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rotate(x / sqrt(mean(x ** 2) + epsilon) * weight)`` in one pass per
    token, the norm over all heads of ``x`` (..., tokens, heads * head_dim);
    a view by head is flattened first (``x.flatten(-2)``).

    ``weight`` may be of another type than x: it enters in fp32.
    ``rope=None`` is the norm alone (the cross-attention's q and k).  Tokens
    are at (t, h, w) of the table's sizes in raster order, starting again
    every ``tokens_per_sample`` tokens (default: x's tokens dimension), and
    tokens behind the grid are padding, normed and not turned.  With
    ``positions`` (..., tokens, axes), integers, each token is where its row
    says; a negative position marks padding.  A position behind its table
    leaves the token unturned and is reported by :func:`check_device_status`."""
    xf, M, heads, D, w, r, tps, pos, dt = _norm_rope_args(x, heads, weight, rope, tokens_per_sample, positions)
    out = torch.empty_like(xf)
    code = nat.lib().reels_rms_norm_rope(xf.data_ptr(), M, heads, D, _ptr(w), r, tps, float(epsilon), dt,
                                         out.data_ptr(), _stream(x.device))
    nat.check("rms_norm_rope", code)
    return out


def rms_norm_rope_backward(x: torch.Tensor, dout: torch.Tensor, heads: int, weight: Optional[torch.Tensor] = None,
                           rope: Optional[RopeTable] = None, epsilon: float = 1e-6,
                           tokens_per_sample: Optional[int] = None,
                           positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Pullback of :func:`rms_norm_rope`: dx.  The weight is frozen."""
    _require_cuda(dout)
    if dout.shape != x.shape or dout.dtype != x.dtype or dout.device != x.device:
        raise ValueError("dout must have the shape, dtype and device of x")
    xf, M, heads, D, w, r, tps, pos, dt = _norm_rope_args(x, heads, weight, rope, tokens_per_sample, positions)
    df = dout if dout.is_contiguous() else dout.contiguous()
    dx = torch.empty_like(xf)
    code = nat.lib().reels_rms_norm_rope_backward(xf.data_ptr(), df.data_ptr(), M, heads, D, _ptr(w), r, tps,
                                                  float(epsilon), dt, dx.data_ptr(), _stream(x.device))
    nat.check("rms_norm_rope_backward", code)
    return dx


class RMSNormRopeFunction(torch.autograd.Function):
    """Autograd rule of :func:`rms_norm_rope`: a gradient for x (the norm's
    weight is frozen: a backward pass that asks for its gradient raises)."""

    @staticmethod
    def forward(ctx, x, heads, weight=None, rope=None, epsilon=1e-6, tokens_per_sample=None, positions=None):
        ctx.save_for_backward(x, weight, positions)
        ctx.args = (heads, rope, epsilon, tokens_per_sample)
        return rms_norm_rope(x, heads, weight, rope, epsilon, tokens_per_sample, positions)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        if any(ctx.needs_input_grad[1:]):  # as long as the arguments that were given
            raise ValueError("the norm's weight is frozen and receives no gradient")
        x, weight, positions = ctx.saved_tensors
        heads, rope, epsilon, tps = ctx.args
        dx = rms_norm_rope_backward(x, dout.contiguous(), heads, weight, rope, epsilon, tps, positions)
        return dx, None, None, None, None, None, None


# ---------------------------------------------------------------- attention
def _readable(t: torch.Tensor) -> torch.Tensor:
    """``t`` if the kernels can follow its strides, else a contiguous copy:
    features contiguous, and for 16-bit types the strides TMA takes."""
    s, n = t.stride(), t.shape
    if n[3] > 1 and s[3] != 1:
        return t.contiguous()
    if t.dtype != torch.float32 and any(n[i] > 1 and (s[i] % 8 or s[i] <= 0) for i in range(3)):
        return t.contiguous()
    return t


_I3 = ctypes.c_int64 * 3
# Checked sizes, strides and types -> (head_dim ** -0.5, the C shape, scratch
# bytes forward and backward, whether the strides can be read): the host side
# of a call is mostly this, and a program repeats few of them.
_SHAPES = {}


def _attention_shape(q, k, v):
    key = (q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), q.dtype, k.dtype, v.dtype)
    hit = _SHAPES.get(key)
    if hit is not None:
        return hit
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k and v must be (batch, tokens, heads, head_dim)")
    B, Sq, H, D = q.shape
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    KB, Sk, HK, KD = k.shape
    if KB != B or KD != D:
        raise ValueError("q, k and v must agree in batch and head_dim")
    if HK == 0 or H % HK:
        raise ValueError("heads must be a multiple of kv_heads")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype")
    dt = _dt(q.dtype)
    shape = nat.AttnShape(B, H, HK, Sq, Sk, D, _I3(*q.stride()[:3]), _I3(*k.stride()[:3]), _I3(*v.stride()[:3]))
    ws = [nat.lib().reels_attention_workspace_bytes(ctypes.byref(shape), dt, p)
          for p in (nat.PASS_FORWARD, nat.PASS_BACKWARD)]
    hit = (D ** -0.5 if D else 1.0, shape, *ws, all(_readable(t) is t for t in (q, k, v)))
    if len(_SHAPES) >= 4096:
        _SHAPES.clear()
    _SHAPES[key] = hit
    return hit


def _attention_args(q, k, v, scale, kv_lengths):
    _require_cuda(q, k, v, kv_lengths)
    device = q.device
    if k.device != device or v.device != device:
        raise ValueError("q, k and v must be on the same device")
    known = _attention_shape(q, k, v)
    if not known[4]:
        q, k, v = _readable(q), _readable(k), _readable(v)
        known = _attention_shape(q, k, v)
    if kv_lengths is not None:
        if kv_lengths.dtype not in (torch.int32, torch.int64) or kv_lengths.shape != (q.shape[0],):
            raise ValueError("kv_lengths must be one integer per sample")
        if kv_lengths.device != device:
            raise ValueError(f"kv_lengths is on {kv_lengths.device}, the input on {device}")
        if kv_lengths.dtype == torch.int64:
            kv_lengths = kv_lengths.clamp(0, k.shape[1]).to(torch.int32)
        kv_lengths = kv_lengths.contiguous()
    return q, k, v, kv_lengths, known[0] if scale is None else float(scale), known


def _scratch(nbytes, device):
    """Scratch of one call, from the caching allocator: calls on different
    streams and captured graphs each have their own."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None,
              kv_lengths: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Softmax attention ``softmax(scale * q k') v`` over all keys of a sample.

    ``q`` (batch, tokens, heads, head_dim), ``k`` and ``v`` (batch, tokens,
    kv_heads, head_dim); heads is a multiple of kv_heads, and head_dim at
    most 256.  ``scale`` defaults to ``head_dim ** -0.5``.  ``kv_lengths``
    (batch,) integers on the device: keys at and behind a sample's length take
    no part, whatever they hold (a padded text); a sample of length 0 gives 0.

    Returns out (batch, tokens, heads, head_dim), contiguous, and with
    ``return_lse`` also the fp32 log-sum-exp (batch, heads, tokens) that
    :func:`attention_backward` needs."""
    q, k, v, lengths, scale, known = _attention_args(q, k, v, scale, kv_lengths)
    B, Sq, H, D = q.shape
    out = q.new_empty((B, Sq, H, D))
    lse = q.new_empty((B, H, Sq), dtype=torch.float32)
    ws = _scratch(known[2], q.device)
    code = nat.lib().reels_attention_forward(ctypes.byref(known[1]), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                             _ptr(lengths), scale, _dt(q.dtype), out.data_ptr(), lse.data_ptr(), _ptr(ws),
                                             0 if ws is None else ws.numel(), _stream(q.device))
    nat.check("attention", code)
    return (out, lse) if return_lse else out


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, scale: Optional[float] = None, kv_lengths: Optional[torch.Tensor] = None):
    """Pullback of :func:`attention`: ``(dq, dk, dv)``, contiguous, with the
    probabilities recomputed from q, k and ``lse``.  ``out`` and ``lse`` are
    the forward's.  Repeated calls give the same bits."""
    _require_cuda(dout, out, lse)
    q, k, v, lengths, scale, known = _attention_args(q, k, v, scale, kv_lengths)
    if out.shape != q.shape or dout.shape != q.shape:
        raise ValueError("out and dout must have the shape of q")
    if out.dtype != q.dtype or dout.dtype != q.dtype:
        raise ValueError("out and dout must have the dtype of q")
    if dout.device != q.device or out.device != q.device or lse.device != q.device:
        raise ValueError("dout, out and lse must be on q's device")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (q.shape[0], q.shape[2], q.shape[1]):
        raise ValueError("lse must be the forward's fp32 (batch, heads, tokens)")
    out, dout, lse = out.contiguous(), dout.contiguous(), lse.contiguous()
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), k.new_empty(k.shape)
    ws = _scratch(known[3], q.device)
    code = nat.lib().reels_attention_backward(ctypes.byref(known[1]), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                              out.data_ptr(), lse.data_ptr(), dout.data_ptr(), _ptr(lengths), scale,
                                              _dt(q.dtype), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ws),
                                              0 if ws is None else ws.numel(), _stream(q.device))
    nat.check("attention_backward", code)
    return dq, dk, dv


class AttentionFunction(torch.autograd.Function):
    """Autograd rule of :func:`attention`: gradients for q, k and v."""

    @staticmethod
    def forward(ctx, q, k, v, scale=None, kv_lengths=None):
        out, lse = attention(q, k, v, scale, kv_lengths, return_lse=True)
        ctx.save_for_backward(q, k, v, out, lse, kv_lengths)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, kv_lengths = ctx.saved_tensors
        return (*attention_backward(dout, q, k, v, out, lse, ctx.scale, kv_lengths), None, None)
