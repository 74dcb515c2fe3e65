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
import ctypes
import math

import torch

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


def _code(t, what):
    code = _DTYPES.get(t.dtype)
    if code is None or t.layout is not torch.strided:
        raise ValueError(f"{what}: a {t.layout} tensor of {t.dtype} (supported: dense float32 and bfloat16)")
    return code


def _clip(src, codes, dst, max_norm, what):
    """The norm of src (element types: codes) as a 0-dim fp32 tensor; dst (None: no scaling) gets
    the scaled values."""
    n = len(src)
    dev = src[0].device
    codes = (ctypes.c_int32 * n)(*codes)
    _lib.require_gpu(*src, what=what)
    sizes = (ctypes.c_int64 * n)(*[t.numel() for t in src])
    srcs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in src])
    if dst is None or dst is src:
        dsts, dst_codes = (None, None) if dst is None else (srcs, codes)
    else:
        dst_codes = (ctypes.c_int32 * n)(*[_code(t, what) for t in dst])
        dsts = (ctypes.c_void_p * n)(*[t.data_ptr() for t in dst])
    nbytes = _lib.lib().mb_grad_clip_workspace(n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.call("mb_grad_clip", srcs, codes, dsts, dst_codes, sizes, n, max_norm, norm.data_ptr(),
                  ws.data_ptr(), nbytes, _lib.stream(dev))
    return norm


@torch.no_grad()
def grad_norm(grads):
    """The 2-norm of all tensors together, a 0-dim fp32 tensor; nothing is scaled."""
    grads = list(grads)
    codes = [_code(g, "grad_norm") for g in grads]
    if not grads:
        return torch.tensor(0.0)
    return _clip([g if _dense(g) else g.contiguous() for g in grads], codes, None, math.inf, "grad_norm")


@torch.no_grad()
def clip_gradients(grads, max_norm, out=None):
    """Scales ``grads`` by min(1, max_norm / (norm + 1e-6)) and returns the norm before that.

    ``out`` None: in place; the tensors must fill their memory without gaps (any order of the
    dimensions).  Otherwise one contiguous tensor of the same shape for each gradient, fp32 or
    bf16, which gets the scaled values; ``grads`` are left as they are.  No written tensor may
    share memory with another tensor of the call, and no tensor may be listed twice where it is
    written; such calls raise HipKernelError before anything is launched."""
    what = "clip_gradients"
    grads = list(grads)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"{what}: max_norm={max_norm}")
    codes = [_code(g, what) for g in grads]
    if out is None:
        for g in grads:
            if not _dense(g):
                raise ValueError(f"{what}: a gradient of shape {tuple(g.shape)} and strides {g.stride()} has gaps or "
                                 "shares its own elements, and cannot be scaled in place")
        dst = grads
    else:
        dst = list(out)
        if len(dst) != len(grads):
            raise ValueError(f"{what}: {len(dst)} outputs for {len(grads)} gradients")
        for g, o in zip(grads, dst):
            if o.shape != g.shape or not o.is_contiguous():
                raise ValueError(f"{what}: an output of shape {tuple(o.shape)}, strides {o.stride()} for a gradient "
                                 f"of shape {tuple(g.shape)}: contiguous tensors of the same shape are wanted")
        if dst:
            _lib.require_gpu(grads[0], *dst, what=what)
        grads = [g.contiguous() for g in grads]
    if not grads:
        return torch.tensor(0.0)
    return _clip(grads, codes, dst, max_norm, what)


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ for the 2-norm, on one GPU: scales the parameters' gradients
    in place and returns their norm before that.  Parameters without a gradient are passed over.
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
