"""RMS norm of every query and key head with the position rotation, on the gfx950 kernels of
mb_qk_norm_rotary_fwd / mb_qk_norm_rotary_bwd.

``qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, eps, start)`` computes, for each head's
row x of q and k,

    y = weight * x * rsqrt(mean(x^2) + eps),  then turns the pairs (y[2i], y[2i+1]) by the
    angle of the row's position (``cos`` / ``sin`` as baseline.rotary_tables makes them),

evaluated in fp32 and rounded once to the inputs' dtype, with gradients for q, k and both
weights.  One launch forward, two backward; the weight gradients are summed in a fixed order.
CPU tensors raise NotImplementedError: there is no CPU path.  Both directions are registered
as torch ops (mathbrain::qk_norm_rotary_fwd / _bwd) for tracing.
"""
import struct
from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.MB_DTYPE_F32, torch.bfloat16: _lib.MB_DTYPE_BF16}
# mb_qk_norm_rotary (include/mathbrain_hip.h): the forward's fields, then the backward's
_ARGS = struct.Struct("2P6q4PqP2q5qqd2P" + "2P6q4PPq")
_NO_BACKWARD = (0,) * 14


def _rows16(x):
    """x with the head's channels next to each other and rows at multiples of 16 bytes."""
    sb, sl, sh, sd = x.stride()
    if sd == 1 and not (x.data_ptr() | (sb | sl | sh) * x.element_size()) & 15:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _like(x):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _weight(w):
    return w if w.dtype is torch.float32 and w.stride(0) == 1 else w.float().contiguous()


def _inputs(q, k, wq, wk, cos, sin, eps, start_rows, start):
    """The struct's fields up to eps."""
    B, L, H, hd = q.shape
    return (q.data_ptr(), k.data_ptr(), *q.stride()[:3], *k.stride()[:3], wq.data_ptr(), wk.data_ptr(), cos.data_ptr(),
            sin.data_ptr(), cos.shape[0], 0 if start_rows is None else start_rows.data_ptr(),
            4 if start_rows is None else start_rows.element_size(), start, B, L, H, k.shape[2], hd, _DTYPES[q.dtype], eps)


def _fwd_fake(q, k, q_weight, k_weight, cos, sin, eps, start_rows, start):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@_lib.traced_op("qk_norm_rotary_fwd", _fwd_fake)
def qk_norm_rotary_fwd(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                       cos: torch.Tensor, sin: torch.Tensor, eps: float, start_rows: Optional[torch.Tensor],
                       start: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(q', k'), contiguous."""
    q, k, wq, wk = _rows16(q), _rows16(k), _weight(q_weight), _weight(k_weight)
    qo, ko = _like(q), _like(k)
    _lib.call_on(q.device, "mb_qk_norm_rotary_fwd",
                 _ARGS.pack(*_inputs(q, k, wq, wk, cos, sin, eps, start_rows, start), qo.data_ptr(), ko.data_ptr(),
                            *_NO_BACKWARD))
    return qo, ko


def _bwd_fake(q, k, q_weight, k_weight, cos, sin, dq_out, dk_out, eps, start_rows, start):
    return (q.new_empty(q.shape), k.new_empty(k.shape), q_weight.new_empty(q_weight.shape),
            k_weight.new_empty(k_weight.shape))


@_lib.traced_op("qk_norm_rotary_bwd", _bwd_fake)
def qk_norm_rotary_bwd(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                       cos: torch.Tensor, sin: torch.Tensor, dq_out: torch.Tensor, dk_out: torch.Tensor,
                       eps: float, start_rows: Optional[torch.Tensor], start: int
                       ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dq_weight, dk_weight) of qk_norm_rotary_fwd for the output gradients."""
    dev = q.device
    B, L, H, hd = q.shape
    q, k, wq, wk = _rows16(q), _rows16(k), _weight(q_weight), _weight(k_weight)
    gq = _rows16(dq_out if dq_out.dtype is q.dtype else dq_out.to(q.dtype))
    gk = _rows16(dk_out if dk_out.dtype is q.dtype else dk_out.to(q.dtype))
    dq, dk, dwq, dwk = _like(q), _like(k), torch.empty_like(wq), torch.empty_like(wk)
    nbytes = _lib.workspace_bytes("mb_qk_norm_rotary_bwd_workspace", B, L, hd)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _lib.call_on(dev, "mb_qk_norm_rotary_bwd",
                 _ARGS.pack(*_inputs(q, k, wq, wk, cos, sin, eps, start_rows, start), 0, 0, gq.data_ptr(), gk.data_ptr(),
                            *gq.stride()[:3], *gk.stride()[:3], dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(),
                            dwk.data_ptr(), ws.data_ptr(), nbytes))
    if q_weight.dtype is not torch.float32 or k_weight.dtype is not torch.float32:
        dwq, dwk = dwq.to(q_weight.dtype), dwk.to(k_weight.dtype)
    return dq, dk, dwq, dwk


class QKNormRotaryFunction(torch.autograd.Function):
    """autograd for qk_norm_rotary: gradients for q, k and the two weights."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, eps, start_rows, start):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, start_rows)
        ctx.rest = (eps, start)
        return qk_norm_rotary_fwd(q, k, q_weight, k_weight, cos, sin, eps, start_rows, start)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin, start_rows = ctx.saved_tensors
        eps, start = ctx.rest
        grads = qk_norm_rotary_bwd(q, k, q_weight, k_weight, cos, sin, dq_out, dk_out, eps, start_rows, start)
        return (*grads, None, None, None, None, None)


def _check(q, k, q_weight, k_weight, cos, sin, start):
    what = "qk_norm_rotary"
    rows = start if torch.is_tensor(start) else None
    at = q.get_device()
    if (at < 0 or k.get_device() != at or q_weight.get_device() != at or k_weight.get_device() != at
            or cos.get_device() != at or sin.get_device() != at or (rows is not None and rows.get_device() != at)):
        _lib.require_gpu(q, k, q_weight, k_weight, cos, sin, rows, what=what)
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or qs[:2] != ks[:2] or qs[3] != ks[3]:
        raise ValueError(f"{what}: q {tuple(qs)} and k {tuple(ks)} are not [B, L, H, hd] and [B, L, Hk, hd]")
    hd = qs[3]
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise ValueError(f"{what}: q {q.dtype} and k {k.dtype} (supported: both float32 or both bfloat16)")
    if q_weight.shape != (hd,) or k_weight.shape != (hd,):
        raise ValueError(f"{what}: weights {tuple(q_weight.shape)}, {tuple(k_weight.shape)} do not match head_dim {hd}")
    if cos.dim() != 2 or cos.shape[1] * 2 != hd or cos.shape != sin.shape:
        raise ValueError(f"{what}: tables {tuple(cos.shape)}, {tuple(sin.shape)} are not [positions, {hd // 2}]")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError(f"{what}: the tables must be contiguous float32")
    if (cos.requires_grad or sin.requires_grad) and torch.is_grad_enabled():
        raise ValueError(f"{what}: the tables get no gradient, and one of them requires it")
    if rows is not None and (rows.shape != qs[:1] or rows.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"{what}: start {tuple(rows.shape)} {rows.dtype} is not one int32 or int64 for each of "
                         f"{qs[0]} rows")


def qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, eps=1e-6, start=0):
    """Normalises and rotates q [B, L, H, hd] and k [B, L, Hk, hd] (fp32 or bf16, any strides);
    weights [hd]; ``cos`` / ``sin`` [positions, hd / 2] fp32, without gradients.  ``start`` is the position of each
    row's first token: an int (checked against the tables), or an int32 / int64 tensor [B], as a
    step that appends one token to sequences of different lengths has it; a position outside the
    tables gives NaN rows there.  head_dim 32, 64 or 128."""
    _check(q, k, q_weight, k_weight, cos, sin, start)
    rows = start.contiguous() if torch.is_tensor(start) else None
    args = (q, k, q_weight, k_weight, cos, sin, float(eps), rows, 0 if rows is not None else int(start))
    if _lib.wants_derivatives(q, k, q_weight, k_weight):
        return QKNormRotaryFunction.apply(*args)
    return qk_norm_rotary_fwd(*args)
