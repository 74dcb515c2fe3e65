"""Attention with a learned relative position bias by distance buckets, on the gfx950 kernels of
mb_bias_attn_fwd / mb_bias_attn_bwd.

``relative_bias_attention(q, k, v, bias, ...)`` computes

    softmax_j(scale q_i . k_j + bias[bucket(i - j), h]) v_j

without the scores, the bias or their gradients ever being in memory, with gradients for q, k,
v and the bias table.  torch's scaled_dot_product_attention takes such a bias only as a tensor
of one value for each pair, and gives its gradient as another one.

Buckets (``bucket_starts``): a distance n = i - j >= 0 below half of the buckets has one of its
own; the others grow by the same factor each up to ``max_distance``, and the last one takes
everything beyond.  Without ``causal`` the lower half of the table serves keys at or before the
query and the upper half, by the same rule, keys after it.

CPU tensors raise NotImplementedError: there is no CPU path.  Both directions are registered as
torch ops (mathbrain::bias_attn_fwd / _bwd) for tracing.
"""
import ctypes
import functools
import math
import struct
from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.MB_DTYPE_F32, torch.bfloat16: _lib.MB_DTYPE_BF16}
# mb_bias_attn (include/mathbrain_hip.h): the inputs, o and lse, the backward's tensors, the workspace
_ARGS = struct.Struct("3P9qPP2qPqP2q6qq2qd" + "P3qP" + "P3q3P9qP" + "Pq")
_NO_BACKWARD = (0,) * 17
MAX_BUCKETS = 128     # in one direction
MAX_DISTANCE = 1024


@functools.lru_cache(maxsize=64)
def bucket_starts(num_buckets, max_distance):
    """The first distance of each of a direction's buckets, as a tuple: 0, 1, ..., e for e =
    num_buckets // 2, then the smallest n with
    floor(log(n / e) / log(max_distance / e) (num_buckets - e)) >= k for k = 1, 2, ...,
    found by whole numbers (n^m >= max_distance^k e^(m-k)), so that no border depends on how a
    logarithm is rounded."""
    e = num_buckets // 2
    if e == 0:
        return (0,)
    m = num_buckets - e
    starts = list(range(e + 1))
    n = e
    for k in range(1, m):
        border = max_distance ** k * e ** (m - k)
        while n ** m < border:
            n += 1
        starts.append(n)
    return tuple(starts)


@functools.lru_cache(maxsize=64)
def _starts_array(num_buckets, max_distance, causal):
    """(array, its address, its length): a caller keeps the array while it uses the address."""
    starts = bucket_starts(num_buckets if causal else num_buckets // 2, max_distance)
    array = (ctypes.c_int32 * len(starts))(*starts)
    return array, ctypes.addressof(array), len(starts)


def _rows16(x):
    """x with the channels next to each other and rows at multiples of 16 bytes, at most 16 MiB apart."""
    sb, sh, sl, sd = x.stride()
    size = x.element_size()
    if sd == 1 and not (x.data_ptr() | (sb | sh | sl) * size) & 15 and sl * size <= 1 << 24:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _heads_last(B, H, L, hd, like):
    """[B, H, L, hd] over memory [B, L, H, hd], so that the projections around it need no copy."""
    return torch.empty_strided((B, H, L, hd), (L * H * hd, hd, H * hd, 1), dtype=like.dtype, device=like.device)


def _inputs(q, k, v, bias, starts, causal, scale, lengths, start_rows, start):
    """The struct's fields up to scale."""
    B, H, Lq, hd = q.shape
    return (q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], bias.data_ptr(),
            starts[1], bias.shape[0], starts[2], 0 if lengths is None else lengths.data_ptr(),
            4 if lengths is None else lengths.element_size(), 0 if start_rows is None else start_rows.data_ptr(),
            4 if start_rows is None else start_rows.element_size(), start, B, H, k.shape[1], Lq, k.shape[2], hd, causal,
            _DTYPES[q.dtype], _DTYPES[bias.dtype], scale)


def _fwd_fake(q, k, v, bias, max_distance, causal, scale, lengths, start_rows, start, want_lse):
    B, H, Lq, hd = q.shape
    return (q.new_empty((B, Lq, H, hd)).transpose(1, 2),
            q.new_empty((B, H, Lq) if want_lse else (0,), dtype=torch.float32))


@_lib.traced_op("bias_attn_fwd", _fwd_fake)
def bias_attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bias: torch.Tensor, max_distance: int,
                  causal: bool, scale: float, lengths: Optional[torch.Tensor], start_rows: Optional[torch.Tensor],
                  start: int, want_lse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(o, lse): lse [B, H, Lq] = log2 of the row's softmax denominator (inf without keys, NaN from NaN) for the
    backward, empty unless wanted."""
    dev = q.device
    B, H, Lq, hd = q.shape
    q, k, v, bias = _rows16(q), _rows16(k), _rows16(v), bias.contiguous()
    o = _heads_last(B, H, Lq, hd, q)
    lse = torch.empty((B, H, Lq) if want_lse else (0,), dtype=torch.float32, device=dev)
    nbytes = _lib.workspace_bytes("mb_bias_attn_fwd_workspace", B, H, k.shape[1], Lq, k.shape[2], hd, causal,
                                  _DTYPES[q.dtype])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    starts = _starts_array(bias.shape[0], max_distance, causal)
    _lib.call_on(dev, "mb_bias_attn_fwd",
                 _ARGS.pack(*_inputs(q, k, v, bias, starts, causal, scale, lengths, start_rows, start),
                            o.data_ptr(), *o.stride()[:3], lse.data_ptr() if want_lse else 0, *_NO_BACKWARD,
                            ws.data_ptr() if nbytes else 0, nbytes))
    return o, lse


def _bwd_fake(q, k, v, bias, o, d_o, lse, max_distance, causal, scale, lengths, start_rows, start, want_dbias):
    def like(x):
        B, H, L, hd = x.shape
        return x.new_empty((B, L, H, hd)).transpose(1, 2)
    return like(q), like(k), like(v), bias.new_empty(bias.shape if want_dbias else (0,))


@_lib.traced_op("bias_attn_bwd", _bwd_fake)
def bias_attn_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bias: torch.Tensor, o: torch.Tensor,
                  d_o: torch.Tensor, lse: torch.Tensor, max_distance: int, causal: bool, scale: float,
                  lengths: Optional[torch.Tensor], start_rows: Optional[torch.Tensor], start: int,
                  want_dbias: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv, dbias) of bias_attn_fwd for the output gradient d_o; dbias is empty unless wanted."""
    dev = q.device
    B, H, Lq, hd = q.shape
    Hk, Lk = k.shape[1:3]
    q, k, v, o, d_o = _rows16(q), _rows16(k), _rows16(v), _rows16(o), _rows16(d_o if d_o.dtype is q.dtype else d_o.to(q.dtype))
    bias = bias.contiguous()
    dq, dk, dv = _heads_last(B, H, Lq, hd, q), _heads_last(B, Hk, Lk, hd, k), _heads_last(B, Hk, Lk, hd, v)
    dbias = torch.empty(bias.shape if want_dbias else (0,), dtype=bias.dtype, device=dev)
    nbytes = _lib.workspace_bytes("mb_bias_attn_bwd_workspace", B, H, Hk, Lq, Lk, hd, causal,
                                  _DTYPES[q.dtype], bias.shape[0])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    starts = _starts_array(bias.shape[0], max_distance, causal)
    _lib.call_on(dev, "mb_bias_attn_bwd",
                 _ARGS.pack(*_inputs(q, k, v, bias, starts, causal, scale, lengths, start_rows, start),
                            o.data_ptr(), *o.stride()[:3], lse.data_ptr(), d_o.data_ptr(), *d_o.stride()[:3],
                            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *dq.stride()[:3], *dk.stride()[:3],
                            *dv.stride()[:3], dbias.data_ptr() if want_dbias else 0, ws.data_ptr(), nbytes))
    return dq, dk, dv, dbias


class RelativeBiasAttentionFunction(torch.autograd.Function):
    """autograd for relative_bias_attention: gradients for q, k, v and the bias table."""

    @staticmethod
    def forward(ctx, q, k, v, bias, max_distance, causal, scale, lengths, start_rows, start):
        o, lse = bias_attn_fwd(q, k, v, bias, max_distance, causal, scale, lengths, start_rows, start, True)
        ctx.save_for_backward(q, k, v, bias, o, lse, lengths, start_rows)
        ctx.rest = (max_distance, causal, scale, start)
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o):
        q, k, v, bias, o, lse, lengths, start_rows = ctx.saved_tensors
        max_distance, causal, scale, start = ctx.rest
        want = ctx.needs_input_grad[3]
        dq, dk, dv, dbias = bias_attn_bwd(q, k, v, bias, o, d_o, lse, max_distance, causal, scale, lengths, start_rows,
                                          start, want)
        return dq, dk, dv, dbias if want else None, None, None, None, None, None, None


def _check(q, k, v, bias, max_distance, causal, lengths, q_start):
    what = "relative_bias_attention"
    rows = q_start if torch.is_tensor(q_start) else None
    at = q.get_device()
    if (at < 0 or k.get_device() != at or v.get_device() != at or bias.get_device() != at
            or (lengths is not None and lengths.get_device() != at) or (rows is not None and rows.get_device() != at)):
        _lib.require_gpu(q, k, v, bias, lengths, rows, what=what)
    qs, ks, bs = q.shape, k.shape, bias.shape
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape or qs[0] != ks[0] or qs[3] != ks[3]:
        raise ValueError(f"{what}: q {tuple(qs)}, k {tuple(ks)}, v {tuple(v.shape)} are not [B, H, Lq, hd] "
                         "and twice [B, Hk, Lk, hd]")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q {q.dtype}, k {k.dtype}, v {v.dtype} (supported: all float32 or all bfloat16)")
    if len(bs) != 2 or bs[1] != qs[1] or bias.dtype not in _DTYPES:
        raise ValueError(f"{what}: bias {tuple(bs)} {bias.dtype} is not [buckets, {qs[1]}] in float32 or bfloat16")
    buckets = bs[0]
    if buckets < 1 or (not causal and buckets % 2):
        raise ValueError(f"{what}: {buckets} buckets (at least one, and an even number without causal)")
    side = buckets if causal else buckets // 2
    if side > MAX_BUCKETS or not side // 2 < max_distance <= MAX_DISTANCE:
        raise ValueError(f"{what}: {side} buckets in a direction up to distance {max_distance} (supported: at most "
                         f"{MAX_BUCKETS}, and a distance above half of them, at most {MAX_DISTANCE})")
    for name, t in (("lengths", lengths), ("q_start", rows)):
        if t is not None and (t.shape != qs[:1] or t.dtype not in (torch.int32, torch.int64)):
            raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype} is not one int32 or int64 for each of "
                             f"{qs[0]} rows")


def relative_bias_attention(q, k, v, bias, max_distance=128, causal=True, scale=None, lengths=None, q_start=None):
    """Attention of q [B, H, Lq, hd] over k, v [B, Hk, Lk, hd] (Hk divides H: key heads shared by
    H / Hk query heads each), fp32 or bf16, any strides, head_dim 32, 64 or 128, with ``bias``
    [buckets, H] (fp32 or bf16) added to the scores by distance.  Returns [B, H, Lq, hd].

    ``q_start``: the position of each row's first query among the keys, an int or an int32 / int64
    tensor [B] (within +-2^29); None: Lk - Lq, so that the last query stands at the last key.
    ``causal``: a query sees the keys up to its position.  ``lengths``: an int32 / int64 tensor [B];
    keys from there on are not seen (values in 0 .. Lk; others are taken as the nearest of these).
    Rows of k and v behind these ends, and with ``causal`` behind the last query's position, may hold
    anything; other values of q, k and v have to be finite (NaN there, or in the bias, comes out as
    NaN in the rows that it reaches).  A bias below -65536 (-inf, or its type's lowest value) hides the
    pairs of its bucket; where all of a head's lie there, the largest is taken off them first.  A query that sees no key gets zeros, and passes on
    no gradient.  ``scale``: 1 / sqrt(hd) by default, otherwise 1e-20 to 1e20.

    In bf16 the probabilities and the scores' gradients are rounded to bf16 for the products that
    they enter; all sums are in fp32.  Gradients come out the same each time."""
    causal, max_distance = bool(causal), int(max_distance)
    _check(q, k, v, bias, max_distance, causal, lengths, q_start)
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    rows = q_start.contiguous() if torch.is_tensor(q_start) else None
    start = k.shape[2] - q.shape[2] if q_start is None else 0 if rows is not None else int(q_start)
    lengths = None if lengths is None else lengths.contiguous()
    args = (q, k, v, bias, max_distance, causal, scale, lengths, rows, start)
    if _lib.wants_derivatives(q, k, v, bias):
        return RelativeBiasAttentionFunction.apply(*args)
    return bias_attn_fwd(*args, False)[0]
