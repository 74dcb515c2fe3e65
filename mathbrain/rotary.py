"""Rotary positions of queries and keys on the gfx950 kernel of mb_apply_rotary.

``apply_rotary(q, k, cos, sin, start, layout)`` turns the channel pairs of every query and key
head by the angles of the row's position:

    y[a] = x[a] cos - x[b] sin,   y[b] = x[a] sin + x[b] cos

with pairs (2i, 2i + 1) (``layout="interleaved"``) or (i, i + d / 2) (``"half"``) of the first
d = 2 * cos.shape[1] channels; the others pass unchanged.  Evaluated in fp32, every product and sum
rounded by itself, and rounded to the inputs' dtype: with the interleaved layout and whole heads the
results are bit for bit those of baseline.rotate.  ``rotary_tables`` makes the tables, with the
frequencies rescaled for contexts longer than the trained ones.  One launch a direction; the
gradient is the rotation by the opposite angles.  CPU tensors raise NotImplementedError.
Registered for tracing as mathbrain::apply_rotary.
"""
import math
import operator
import struct
from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.MB_DTYPE_F32, torch.bfloat16: _lib.MB_DTYPE_BF16}
LAYOUTS = ("interleaved", "half")
_ARGS = struct.Struct("2P6q2PqP3q6q3q2P")   # mb_rotary (include/mathbrain_hip.h)


def rotary_tables(dim, positions, theta=10000.0, scaling=None, factor=1.0, trained=None, fast=32.0, slow=1.0,
                  device=None):
    """cos and sin [positions, dim / 2] fp32 of the angles t * theta^(-2i/dim), taken in 64 bits so that far
    positions keep their angles.

    ``scaling`` stretches them for contexts ``factor`` times as long as the trained ones: "linear" divides every
    angle by the factor; "ntk" raises theta by factor^(dim / (dim - 2)), which keeps the fastest pair and divides the
    slowest by the factor; "yarn" divides the angles of the pairs that turn less than ``slow`` times within the
    ``trained`` positions, keeps those that turn more than ``fast`` times, goes from one to the other linearly over the
    pairs between (the ends of that range rounded outwards to whole pairs; the range may end beyond the last pair, which
    is then divided in part), and multiplies both tables by 0.1 ln(factor) + 1."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_tables: dim={dim} (an even number of channels, at least 2)")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"rotary_tables: scaling={scaling!r} (None, 'linear', 'ntk' or 'yarn')")
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"rotary_tables: factor={factor} (1 or more)")
    if not (theta > 0.0 and math.isfinite(theta)):
        raise ValueError(f"rotary_tables: theta={theta} (above 0)")
    if scaling == "ntk":
        if dim < 4:
            raise ValueError("rotary_tables: 'ntk' wants dim of 4 or more")
        theta = theta * factor ** (dim / (dim - 2))
    rate = theta ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    size = 1.0
    if scaling == "linear":
        rate = rate / factor
    elif scaling == "yarn":
        if trained is None or trained < 1:
            raise ValueError("rotary_tables: 'yarn' wants the number of trained positions")
        if not (theta > 1.0 and fast >= slow > 0.0 and math.isfinite(fast)):
            raise ValueError(f"rotary_tables: theta={theta}, fast={fast}, slow={slow} ('yarn' wants theta above 1 and fast >= slow > 0)")
        # pair (dim / 2) log(trained / (2 pi n)) / log(theta) turns n times within the trained positions
        first, last = (dim / 2 * math.log(trained / (2 * math.pi * n)) / math.log(theta) for n in (fast, slow))
        first, last = max(math.floor(first), 0), min(math.ceil(last), dim - 1)
        pair = torch.arange(dim // 2, dtype=torch.float64, device=device)
        share = ((pair - first) / max(last - first, 1e-3)).clamp(0, 1)
        if last <= 0:      # the fastest pair, too, turns less than that
            share.fill_(1.0)
        rate = rate * (1 - share) + rate / factor * share
        size = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rate
    return (angle.cos() * size).float(), (angle.sin() * size).float()


def _fake(q, k, cos, sin, start_rows, start, half, inverse):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@_lib.traced_op("apply_rotary", _fake)
def rotary_op(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
              start_rows: Optional[torch.Tensor], start: int, half: bool,
              inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(q', k'), contiguous; ``inverse`` turns by the opposite angles."""
    B, L, H, hd = q.shape
    if q.stride(3) != 1:
        q = q.contiguous()
    if k.stride(3) != 1:
        k = k.contiguous()
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    rows = start_rows
    _lib.call_on(q.device, "mb_apply_rotary",
                 _ARGS.pack(q.data_ptr(), k.data_ptr(), *q.stride()[:3], *k.stride()[:3], cos.data_ptr(), sin.data_ptr(),
                            cos.shape[0], 0 if rows is None else rows.data_ptr(), 4 if rows is None else rows.element_size(),
                            0 if rows is None else rows.dim() == 2, start, B, L, H, k.shape[2], hd, 2 * cos.shape[1],
                            half, inverse, _DTYPES[q.dtype], qo.data_ptr(), ko.data_ptr()))
    return qo, ko


class RotaryFunction(torch.autograd.Function):
    """autograd for apply_rotary; its derivatives are rotations themselves, of any order and in both modes."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, start_rows, start, half, inverse):
        ctx.save_for_backward(cos, sin, start_rows)
        ctx.save_for_forward(cos, sin, start_rows)
        ctx.rest = (start, half, inverse, q.shape, k.shape, q.dtype, k.dtype)
        ctx.set_materialize_grads(False)
        return rotary_op(q, k, cos, sin, start_rows, start, half, inverse)

    @staticmethod
    def _turned(ctx, gq, gk, opposite):
        cos, sin, start_rows = ctx.saved_tensors
        start, half, inverse, q_shape, k_shape, q_type, k_type = ctx.rest
        if gq is None and gk is None:
            return None, None
        some = gq if gq is not None else gk
        # a side without a gradient takes no part: a tensor without heads
        q = some.new_empty((*q_shape[:2], 0, q_shape[3]), dtype=q_type) if gq is None else gq.to(q_type)
        k = some.new_empty((*k_shape[:2], 0, k_shape[3]), dtype=k_type) if gk is None else gk.to(k_type)
        args = (q, k, cos, sin, start_rows, start, half, inverse != opposite)
        dq, dk = RotaryFunction.apply(*args) if _lib.wants_derivatives(q, k) else rotary_op(*args)
        return dq if gq is not None else None, dk if gk is not None else None

    @staticmethod
    def backward(ctx, gq, gk):
        return (*RotaryFunction._turned(ctx, gq, gk, True), None, None, None, None, None, None)

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        tangents = RotaryFunction._turned(ctx, tq, tk, False)
        some = tq if tq is not None else tk      # forward mode wants a tangent of every output
        return tuple(some.new_zeros(shape, dtype=t) if x is None else x
                     for x, shape, t in zip(tangents, ctx.rest[3:5], ctx.rest[5:7]))


class TracedRotaryFunction(torch.autograd.Function):
    """RotaryFunction for torch.compile, which takes no function with a jvp of its own: the first derivative backwards."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, start_rows, start, half, inverse):
        ctx.save_for_backward(cos, sin, start_rows)
        ctx.rest = (start, half, inverse)
        return rotary_op(q, k, cos, sin, start_rows, start, half, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        start, half, inverse = ctx.rest
        return (*rotary_op(gq, gk, *ctx.saved_tensors, start, half, not inverse), None, None, None, None, None, None)


def _check(q, k, cos, sin, start, layout):
    what = "apply_rotary"
    rows = start if torch.is_tensor(start) else None
    at = q.get_device()
    if (at < 0 or k.get_device() != at or cos.get_device() != at or sin.get_device() != at
            or (rows is not None and rows.get_device() != at)):
        _lib.require_gpu(q, k, cos, sin, rows, what=what)
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or qs[:2] != ks[:2] or qs[3] != ks[3]:
        raise ValueError(f"{what}: q {tuple(qs)} and k {tuple(ks)} are not [B, L, H, hd] and [B, L, Hk, hd]")
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise ValueError(f"{what}: q {q.dtype} and k {k.dtype} (supported: both float32 or both bfloat16)")
    if layout not in LAYOUTS:
        raise ValueError(f"{what}: layout={layout!r} ('interleaved' or 'half')")
    if cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > qs[3]:
        raise ValueError(f"{what}: tables {tuple(cos.shape)}, {tuple(sin.shape)} are not [positions, d / 2] for d of up to "
                         f"{qs[3]} channels")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError(f"{what}: the tables must be contiguous float32")
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad) or _lib.has_tangent(cos, sin):
        raise ValueError(f"{what}: the tables get no derivative, and one of them wants it")
    if rows is None and not isinstance(start, (int, torch.SymInt)):
        try:
            start = operator.index(start)
        except TypeError:
            raise ValueError(f"{what}: start={start!r} is neither a whole number nor a tensor") from None
    if rows is None and type(start) is int and not -2**63 <= start < 2**63:
        raise ValueError(f"{what}: start={start} is no position")
    if rows is not None and (tuple(rows.shape) not in ((qs[0],), (qs[0], qs[1])) or rows.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"{what}: start {tuple(rows.shape)} {rows.dtype} is not one int32 or int64 for each of {qs[0]} rows, "
                         f"or for each of their {qs[1]} tokens")


def apply_rotary(q, k, cos, sin, start=0, layout="interleaved"):
    """Turns q [B, L, H, hd] and k [B, L, Hk, hd] (fp32 or bf16, any strides and head size) and returns them
    contiguous.  ``cos`` / ``sin`` [positions, d / 2] fp32, without gradients: the first d channels turn.  ``start``
    is the position of each row's first token, an int (checked against the tables) or an int32 / int64 tensor [B], or
    the position of every token, a tensor [B, L] (documents packed into rows); a position outside the tables gives NaN
    in the channels that turn."""
    _check(q, k, cos, sin, start, layout)
    rows = start.contiguous() if torch.is_tensor(start) else None
    args = (q, k, cos, sin, rows, 0 if rows is not None else int(start), layout == "half", False)
    if _lib.wants_derivatives(q, k):
        return (TracedRotaryFunction if torch.compiler.is_compiling() else RotaryFunction).apply(*args)
    return rotary_op(*args)
