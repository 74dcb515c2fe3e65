"""Orthogonalised updates of weight matrices and the optimiser that applies them, on the gfx950 kernels of mb_muon_run.

``orthogonalize(matrices)`` brings the singular values of every matrix near 1 by Newton-Schulz products:
X = G / (|G| + eps), then ``steps`` times A = X X^T, X <- a X + (b A + c A^2) X (on the side with fewer rows).
``muon_step`` is the optimiser's step with it for lists of tensors, in place: momentum, the orthogonalised
update and the decayed weights; ``Muon`` is the torch.optim.Optimizer of it, for the weight matrices of a model
(its embeddings, norms and other vectors belong to another optimiser).

All matrices of a call, of whatever shapes, go through every launch together, as far as a workspace of 4 GiB holds them
(some 200 million elements; one matrix at least).  The products are those of fp32 values
whatever the inputs' type (two fp16 planes a matrix, 24 bits; a single 16-bit plane would leave errors of the first
iterations multiplied by some hundreds).  fp32 and bf16, mixed as they come; no gradients.  CPU tensors raise
NotImplementedError.
"""
import ctypes
import functools
import math
import struct

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.MB_DTYPE_F32, torch.bfloat16: _lib.MB_DTYPE_BF16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # a, b, c: singular values from 1 down to a few thousandths come to 0.7 .. 1.2 in 5 steps
_MATRIX = struct.Struct("3P2q3qd")         # mb_muon_matrix (include/mathbrain_hip.h)
_ARGS = struct.Struct("P4q4d3q3dPq")       # mb_muon


@functools.lru_cache(maxsize=64)
def _exponents(steps, coefficients):
    """Powers of two for the planes of X, A and b A + c A^2 from bounds on their singular values: X's are at most 1 at
    first, and after each step at most the polynomial's largest value on the interval so far."""
    a, b, c = coefficients
    top, most = 1.0, [1.0, 1.0, 0.0]
    for _ in range(steps):
        s = torch.linspace(0.0, top, 20001, dtype=torch.float64, device="cpu")
        gram = s * s
        second = b * gram + c * gram * gram
        most = [max(most[0], top), max(most[1], top * top), max(most[2], float(second.abs().max()))]
        top = 1.01 * float((s * (a + second)).abs().max())     # between the points, and roundings
        if not top < 64.0:
            raise ValueError(f"orthogonalize: with coefficients {coefficients} the iterates grow beyond 64 in {steps} steps")
    return tuple(min(15, math.floor(math.log2(32768.0 / max(1.05 * m, 2.0**-10)))) for m in most)


def _check(tensors, what, device, contiguous):
    for t in tensors:
        if t.dtype not in _DTYPES or t.layout is not torch.strided:
            raise ValueError(f"{what}: a {t.layout} tensor of {t.dtype} (supported: dense float32 and bfloat16)")
        if t.dim() != 2:
            raise ValueError(f"{what}: a tensor of shape {tuple(t.shape)} is not a matrix")
        if contiguous and not t.is_contiguous():
            raise ValueError(f"{what}: a tensor of shape {tuple(t.shape)} and strides {t.stride()} that is written has to be contiguous")
    if device.type != "cuda" or any(t.device != device for t in tensors):
        _lib.require_gpu(torch.empty(0, device=device), *tensors, what=what)
    if _lib.has_tangent(*tensors):
        raise NotImplementedError(f"{what}: forward-mode tangents are not carried along")


def _run(src, dst, momenta, rates, steps, coefficients, eps, step=None):
    """mb_muon_run; ``step``: (lr, momentum, nesterov, weight_decay) of an optimiser's step."""
    device = dst[0].device
    lr, mu, nesterov, decay = step or (0.0, 0.0, False, 0.0)
    table = bytearray(_MATRIX.size * len(src))
    for i, (x, y) in enumerate(zip(src, dst)):
        m = momenta[i] if step else None
        _MATRIX.pack_into(table, i * _MATRIX.size, x.data_ptr(), y.data_ptr(), m.data_ptr() if step else 0, *y.shape, _DTYPES[x.dtype],
                          _DTYPES[y.dtype], _DTYPES[m.dtype] if step else 0, rates[i] if rates else 1.0)
    held = (ctypes.c_char * len(table)).from_buffer(table)
    head = (ctypes.addressof(held), len(src), steps, step is not None, nesterov, *coefficients, eps,
            *_exponents(steps, coefficients), lr, mu, decay)
    nbytes = _lib.lib().mb_muon_workspace(_ARGS.pack(*head, 0, 0))
    if nbytes < 0:
        raise _lib.HipKernelError(_lib.lib().mb_last_error().decode(errors="replace"))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _lib.call_on(device, "mb_muon_run", _ARGS.pack(*head, ws.data_ptr(), nbytes))


def _settings(what, steps, coefficients, eps):
    coefficients = tuple(float(x) for x in coefficients)
    if len(coefficients) != 3 or not all(map(math.isfinite, coefficients)):
        raise ValueError(f"{what}: coefficients {coefficients} are not three finite numbers")
    if not 1 <= int(steps) <= 100:
        raise ValueError(f"{what}: steps={steps} (1 to 100)")
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"{what}: eps={eps}")
    return int(steps), coefficients, float(eps)


@torch.no_grad()
def orthogonalize(matrices, steps=5, coefficients=COEFFICIENTS, eps=1e-7, dtype=None):
    """The orthogonalised matrices, contiguous, of ``dtype`` (their own): ``matrices`` is a list of [rows, cols] tensors of
    any shapes (a list comes back) or one tensor [..., rows, cols].  A matrix of zeros stays zero (with eps = 0 it is 0 / 0, NaN); a NaN or an infinity in a
    matrix makes all of it NaN."""
    what = "orthogonalize"
    steps, coefficients, eps = _settings(what, steps, coefficients, eps)
    if torch.is_tensor(matrices):
        if matrices.dim() < 2 or matrices.layout is not torch.strided:
            raise ValueError(f"{what}: a {matrices.layout} tensor of shape {tuple(matrices.shape)} is not a dense [..., rows, cols]")
        each = matrices[None] if matrices.dim() == 2 else matrices.flatten(0, -3)
        out = torch.empty(matrices.shape, dtype=dtype or matrices.dtype, device=matrices.device)
        src, dst = list(each.unbind()), list(out.view(each.shape).unbind())
    else:
        src = list(matrices)
        dst = out = [torch.empty(x.shape, dtype=dtype or x.dtype, device=x.device) for x in src]
    if not src:
        return out
    _check(src, what, src[0].device, False)
    _check(dst, what, src[0].device, True)
    _run([x.contiguous() for x in src], dst, None, None, steps, coefficients, eps)
    return out


@torch.no_grad()
def muon_step(params, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS,
              eps=1e-7):
    """One step for lists of matrices, in place: with g a gradient and m its momentum,

        m <- momentum * m + g,   u = g + momentum * m (nesterov) or m,
        p <- p (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) orthogonalize(u)

    in fp32, rounded to the tensors' types (fp32 or bf16 each).  ``params`` and ``momenta`` have to be contiguous and share no
    memory with another tensor of the call (HipKernelError)."""
    what = "muon_step"
    steps, coefficients, eps = _settings(what, steps, coefficients, eps)
    params, grads, momenta = list(params), list(grads), list(momenta)
    lr, momentum, weight_decay = float(lr), float(momentum), float(weight_decay)
    if not (math.isfinite(lr) and math.isfinite(momentum) and math.isfinite(weight_decay)):
        raise ValueError(f"{what}: lr={lr}, momentum={momentum}, weight_decay={weight_decay}")
    if not len(params) == len(grads) == len(momenta) or any(not p.shape == g.shape == m.shape for p, g, m in zip(params, grads, momenta)):
        raise ValueError(f"{what}: {len(params)} parameters, {len(grads)} gradients and {len(momenta)} momenta do not match in number "
                         "or shape")
    if not params:
        return
    device = params[0].device
    _check(params, what, device, True)
    _check(momenta, what, device, True)
    _check(grads, what, device, False)
    rates = [math.sqrt(max(1.0, p.shape[0] / p.shape[1])) if p.numel() else 1.0 for p in params]
    _run([g.contiguous() for g in grads], params, momenta, rates, steps, coefficients, eps, (lr, momentum, bool(nesterov), weight_decay))
    torch.autograd.graph.increment_version(params + momenta)   # a graph that saved one of them says so in its backward


class Muon(torch.optim.Optimizer):
    """muon_step as an optimizer for matrices; parameters of another number of dimensions are refused."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
        if not lr >= 0 or not 0 <= momentum < 1 or not weight_decay >= 0:
            raise ValueError(f"Muon: lr={lr}, momentum={momentum}, weight_decay={weight_decay}")
        _exponents(*_settings("Muon", steps, coefficients, eps)[:2])
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"Muon: a parameter of shape {tuple(p.shape)} is not a matrix")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            for p in params:
                if "momentum_buffer" not in self.state[p]:
                    self.state[p]["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            muon_step(params, [p.grad for p in params], [self.state[p]["momentum_buffer"] for p in params], group["lr"],
                      group["momentum"], group["nesterov"], group["weight_decay"], group["steps"], group["coefficients"], group["eps"])
        return loss
