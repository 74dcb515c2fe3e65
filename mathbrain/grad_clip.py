"""The global gradient norm over many tensors, and clipping, on the gfx950 kernels of mb_grad_clip.

``clip_grad_norm_(parameters, max_norm)`` has torch.nn.utils.clip_grad_norm_'s arguments and
result for the 2-norm (train.py's training step calls it): the gradients are scaled in place
by min(1, max_norm / (norm + 1e-6)), and the norm before that is returned as a 0-dim fp32
tensor on the device, without a synchronisation.  ``clip_gradients(grads, max_norm, out)``
takes the tensors themselves and can write the clipped values elsewhere, for instance bf16
gradients into the fp32 buffer that an optimiser with fp32 master weights reads.

Two launches for every 120 tensors, squares summed in 64 bits in a fixed order, so that the
same gradients always give the same norm.  Where the factor is 1 an in-place call writes
nothing.  fp32 and bf16 tensors, mixed as they come; CPU tensors raise NotImplementedError.
"""
import array
import bisect
import math

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.MB_DTYPE_F32, torch.bfloat16: _lib.MB_DTYPE_BF16}


def _dense(t):
    """True if t's elements fill one stretch of memory, in whatever order."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _codes(tensors, device, what):
    """(the tensors' element types, whether all are contiguous): they have to be on one GPU, of one of
    this library's types each, dense.  Whole lists are compared, tensor by tensor only to name the one that fails: with
    many small tensors the host's time is the call's."""
    codes = [_DTYPES.get(t.dtype, -1) for t in tensors]
    try:
        contiguous = False not in list(map(torch.Tensor.is_contiguous, tensors))
    except RuntimeError:    # some sparse layouts' answer; others say False
        contiguous = False
    if -1 in codes or not contiguous and any(t.layout is not torch.strided for t in tensors):
        t = next(t for t, c in zip(tensors, codes) if c < 0 or t.layout is not torch.strided)
        raise ValueError(f"{what}: a {t.layout} tensor of {t.dtype} (supported: dense float32 and bfloat16)")
    index = device.index if device.type == "cuda" else -2
    if list(map(torch.Tensor.get_device, tensors)).count(index) != len(codes):
        _lib.require_gpu(torch.empty(0, device=device), *tensors, what=what)
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: forward-mode tangents are not scaled with their tensors")
    return array.array("i", codes), contiguous


def _stretch(t):
    """The addresses of a tensor's first byte and of the one behind its last."""
    at = t.data_ptr()
    return at, at + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()


def _refuse_overwritten(grads, out, what):
    """The library sees copies of the gradients that are not contiguous: their own memory must not be
    an output's.  (Outputs that share memory among them are refused there.)"""
    written = sorted(_stretch(o) for o in out if o.numel())
    starts = [first for first, _ in written]
    for g in grads:
        if g.numel() and not g.is_contiguous():
            first, end = _stretch(g)
            i = bisect.bisect_left(starts, end) - 1
            if i >= 0 and written[i][1] > first:
                raise _lib.HipKernelError(f"{what}: tensors share memory that the call writes")


def _clip(src, codes, dst, dst_codes, max_norm, device):
    """The norm of src (element types: codes) as a 0-dim fp32 tensor; dst (None: no scaling) gets
    the scaled values."""
    n = len(src)
    sizes = array.array("q", map(torch.Tensor.numel, src))
    srcs = array.array("Q", map(torch.Tensor.data_ptr, src))
    dsts = srcs if dst is src else dst and array.array("Q", map(torch.Tensor.data_ptr, dst))
    at = [a and a.buffer_info()[0] for a in (srcs, codes, dsts, dst_codes, sizes)]
    nbytes = _lib.lib().mb_grad_clip_workspace(n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    _lib.call_on(device, "mb_grad_clip", *at, n, max_norm, norm.data_ptr(), ws.data_ptr(), nbytes)
    if dst:
        torch.autograd.graph.increment_version(dst)   # a graph that saved one of them says so in its backward
    return norm


@torch.no_grad()
def grad_norm(grads):
    """The 2-norm of all tensors together, a 0-dim fp32 tensor; nothing is scaled."""
    grads = list(grads)
    if not grads:
        return torch.tensor(0.0)
    device = grads[0].device
    codes, contiguous = _codes(grads, device, "grad_norm")
    return _clip(grads if contiguous else [g if _dense(g) else g.contiguous() for g in grads], codes, None, None, math.inf,
                 device)


@torch.no_grad()
def clip_gradients(grads, max_norm, out=None):
    """Scales ``grads`` by min(1, max_norm / (norm + 1e-6)) and returns the norm before that.

    ``out`` None: in place; the tensors must fill their memory without gaps (any order of the
    dimensions).  Otherwise one contiguous tensor of the same shape for each gradient, fp32 or
    bf16, which gets the scaled values; ``grads`` are left as they are.  No written tensor may
    share memory with another tensor of the call (a gradient with gaps counts with them), and no
    tensor may be listed twice where it is written; such calls raise HipKernelError before anything
    is launched."""
    what = "clip_gradients"
    grads = list(grads)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"{what}: max_norm={max_norm}")
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"{what}: {len(out)} outputs for {len(grads)} gradients")
    if not grads:
        return torch.tensor(0.0)
    device = grads[0].device
    codes, contiguous = _codes(grads, device, what)
    if out is None:
        for g in () if contiguous else grads:
            if not _dense(g):
                raise ValueError(f"{what}: a gradient of shape {tuple(g.shape)} and strides {g.stride()} has gaps or "
                                 "shares its own elements, and cannot be scaled in place")
        return _clip(grads, codes, grads, codes, max_norm, device)
    out_codes, whole = _codes(out, device, what)
    if not whole or False in list(map(torch.Tensor.is_same_size, out, grads)):
        g, o = next((g, o) for g, o in zip(grads, out) if o.shape != g.shape or not o.is_contiguous())
        raise ValueError(f"{what}: an output of shape {tuple(o.shape)}, strides {o.stride()} for a gradient "
                         f"of shape {tuple(g.shape)}: contiguous tensors of the same shape are wanted")
    if not contiguous:
        _refuse_overwritten(grads, out, what)
        grads = [g.contiguous() for g in grads]
    return _clip(grads, codes, out, out_codes, max_norm, device)


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ for the 2-norm, on one GPU: scales the parameters' gradients
    in place and returns their norm before that.  Parameters without a gradient are passed over; one
    that is listed twice is refused (HipKernelError), as are gradients that share memory.
    ``error_if_nonfinite`` raises RuntimeError, before anything is scaled, where the norm is not
    finite (that reads the norm back to the host).  ``foreach`` is accepted and has no effect."""
    if float(norm_type) != 2.0:
        raise ValueError(f"clip_grad_norm_: norm_type={norm_type} (supported: 2)")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite and grads:
        norm = grad_norm(grads)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"clip_grad_norm_: the gradients' norm is {float(norm)}, and cannot be used for clipping")
    return clip_gradients(grads, max_norm)
