"""Softmax cross entropy of a linear layer's outputs without the outputs, on the gfx950 kernels of
mb_linear_ce_fwd / mb_linear_ce_bwd.

``linear_cross_entropy(hidden, weight, target)`` is F.cross_entropy(F.linear(hidden, weight), target)
with gradients for hidden and weight, for the tied output matrix over a vocabulary of any size: the
scores exist a tile at a time, and in the backward pass a piece of the vocabulary at a time (about
512 MiB, in fp32 twice that), where F.cross_entropy keeps [rows, vocabulary] several times.  fp32 and
bf16; scores, maxima, sums and both gradients' sums are fp32 or more, the scores are never rounded to
bf16, and the loss is fp32.  The gradients' products take softmax - onehot, and the rows of hidden times
their gradients, in 11 bits for bf16 tensors: a word whose probability is below 2^-40 in every row
has no gradient there, one below 2^-32 fewer than bf16's 8 bits, and rows (times their gradients) or words
below 2^-31 of the largest lose bits in the same way.  For fp32 tensors all operands have 24 bits
down to 2^-16 of their own row's largest value (or of the largest term of the row's or word's sum).
Sums have a fixed order.  CPU tensors raise NotImplementedError.  Both directions
are registered as torch ops (mathbrain::linear_ce_fwd / linear_ce_bwd) for tracing.
"""
import functools
import struct

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.MB_DTYPE_F32, torch.bfloat16: _lib.MB_DTYPE_BF16}
REDUCTIONS = ("none", "mean", "sum")
_ARGS = struct.Struct("2P2qP2q4qq3PP2PPq")   # mb_linear_ce (include/mathbrain_hip.h)
_ANY = 1 << 20                               # an aligned address that nothing is done with


def _rows(x):
    """x [rows, D] with the elements of a row next to each other and rows no closer than D."""
    if x.stride(1) == 1 and (x.shape[0] == 1 or x.shape[1] <= x.stride(0) <= 1 << 22):
        return x
    return x.contiguous()


@functools.lru_cache(maxsize=256)
def _workspace(backward, follows, h_at, w_at, h_ld, w_ld, N, V, D, dtype):
    """The library's workspace for these sizes, row distances and addresses modulo 16; whether a backward follows."""
    nbytes = _lib.lib().mb_linear_ce_workspace(
        _ARGS.pack(_ANY + h_at, _ANY + w_at, h_ld, w_ld, _ANY, 8, 0, N, V, D, dtype, 0, _ANY, _ANY, _ANY, _ANY if follows else 0, 0, 0, 0, 0),
        backward)
    if nbytes < 0:
        raise _lib.HipKernelError(_lib.lib().mb_last_error().decode(errors="replace"))
    return nbytes


def _call(name, backward, hidden, weight, target, ignore_index, reduction, loss, stats, dloss, dh=None, dw=None):
    N, D = hidden.shape
    V = weight.shape[0]
    h, w, t = hidden.data_ptr(), weight.data_ptr(), _DTYPES[hidden.dtype]
    h_ld, w_ld = hidden.stride(0) if N > 1 else D, weight.stride(0) if V > 1 else D
    nbytes = _workspace(backward, dloss is not None, h % 16, w % 16, h_ld, w_ld, N, V, D, t)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=hidden.device)
    lse = stats.data_ptr()
    _lib.call_on(hidden.device, name,
                 _ARGS.pack(h, w, h_ld, w_ld, target.data_ptr(), target.element_size(), ignore_index, N, V, D, t, reduction,
                            0 if loss is None else loss.data_ptr(), lse, lse + 8 * N, 0 if dloss is None else dloss.data_ptr(),
                            0 if dh is None else dh.data_ptr(), 0 if dw is None else dw.data_ptr(), ws.data_ptr(), nbytes))


def _fwd_fake(hidden, weight, target, ignore_index, reduction, follows=True):
    N = hidden.shape[0]
    return (hidden.new_empty((N,) if reduction == 0 else (), dtype=torch.float32),
            hidden.new_empty((2 * N + 1,), dtype=torch.float32))


@_lib.traced_op("linear_ce_fwd", _fwd_fake)
def linear_ce_fwd(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int,
                  reduction: int, follows: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss, what the backward wants of the rows: their maxima, logarithms of sums and how many count [2 N + 1]);
    ``follows``: whether a backward may follow, which wants the scores of its own kernels."""
    loss, stats = _fwd_fake(hidden, weight, target, ignore_index, reduction)
    if hidden.shape[0] == 0:
        return loss.fill_(float("nan") if reduction == 1 else 0.0), stats.zero_()
    _call("mb_linear_ce_fwd", 0, _rows(hidden), _rows(weight), target, ignore_index, reduction, loss, stats,
          stats if follows else None)
    return loss, stats


def _bwd_fake(hidden, weight, target, stats, dloss, ignore_index, reduction, wants_hidden, wants_weight):
    return (hidden.new_empty(hidden.shape if wants_hidden else (0,)),
            weight.new_empty(weight.shape if wants_weight else (0,)))


@_lib.traced_op("linear_ce_bwd", _bwd_fake)
def linear_ce_bwd(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, stats: torch.Tensor, dloss: torch.Tensor,
                  ignore_index: int, reduction: int, wants_hidden: bool, wants_weight: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(dhidden, dweight), contiguous, of linear_ce_fwd's inputs and results; an empty tensor for one that is not wanted."""
    dh, dw = _bwd_fake(hidden, weight, target, stats, dloss, ignore_index, reduction, wants_hidden, wants_weight)
    if hidden.shape[0] == 0:
        return dh, dw.zero_()
    dloss = dloss.to(torch.float32).contiguous()
    _call("mb_linear_ce_bwd", 1, _rows(hidden), _rows(weight), target, ignore_index, reduction, None, stats, dloss,
          dh if wants_hidden else None, dw if wants_weight else None)
    return dh, dw


class LinearCrossEntropyFunction(torch.autograd.Function):
    """autograd for linear_cross_entropy: gradients for hidden and weight."""

    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction):
        loss, stats = linear_ce_fwd(hidden, weight, target, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, target, stats)
        ctx.rest = (ignore_index, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        hidden, weight, target, stats = ctx.saved_tensors
        wants_h, wants_w = ctx.needs_input_grad[:2]
        dh, dw = linear_ce_bwd(hidden, weight, target, stats, dloss, *ctx.rest, wants_h, wants_w)
        return dh if wants_h else None, dw if wants_w else None, None, None, None


def linear_cross_entropy(hidden, weight, target, ignore_index=-100, reduction="mean"):
    """The cross entropy of F.linear(hidden, weight) against ``target``: hidden [..., D], weight [V, D] (both fp32 or
    both bf16, any strides; under torch.autocast both are cast as nn.Linear casts them), target [...] int32 or int64.
    ``reduction`` "mean" (over the rows whose target is not ``ignore_index``; NaN where there is none), "sum" or "none"
    (the losses [...], 0 for ignored rows); fp32.  A target outside the vocabulary that is not ``ignore_index`` gives
    NaN in the loss and in the gradients that it reaches."""
    what = "linear_cross_entropy"
    at = hidden.get_device()
    if at < 0 or weight.get_device() != at or target.get_device() != at:
        _lib.require_gpu(hidden, weight, target, what=what)
    if torch.is_autocast_enabled("cuda"):
        t = torch.get_autocast_dtype("cuda")
        hidden, weight = (x if x.dtype is torch.float64 else x.to(t) for x in (hidden, weight))
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise ValueError(f"{what}: hidden {hidden.dtype} and weight {weight.dtype} (supported: both float32 or both bfloat16)")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"{what}: hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} are not [..., D] and [V, D]")
    if target.shape != hidden.shape[:-1] or target.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: target {tuple(target.shape)} {target.dtype} is not one int32 or int64 for each row of "
                         f"hidden {tuple(hidden.shape)}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"{what}: reduction={reduction!r} ('none', 'mean' or 'sum')")
    args = (hidden.reshape(-1, hidden.shape[-1]), weight, target.reshape(-1).contiguous(), int(ignore_index),
            REDUCTIONS.index(reduction))
    loss = LinearCrossEntropyFunction.apply(*args) if _lib.wants_derivatives(hidden, weight) else linear_ce_fwd(*args, False)[0]
    return loss.view(target.shape) if reduction == "none" else loss
