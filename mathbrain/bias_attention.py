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
from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.MB_DTYPE_F32, torch.bfloat16: _lib.MB_DTYPE_BF16}
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
    starts = bucket_starts(num_buckets if causal else num_buckets // 2, max_distance)
    return (ctypes.c_int32 * len(starts))(*starts), len(starts)


def _rows16(x):
    """x with the channels next to each other and rows at multiples of 16 bytes, at most 16 MiB apart."""
    sb, sh, sl, sd = x.stride()
    if sd == 1 and not (x.data_ptr() | (sb | sh | sl) * x.element_size()) & 15 and sl * x.element_size() <= 1 << 24:
        return x
    return x.contiguous() if not x.is_contiguous() else x.clone()


def _st(x):
    return (ctypes.c_int64 * 3)(*x.stride()[:3])


def _per_row(rows, value=0):
    """(pointer, bytes of an element, value) of an optional int tensor [B]."""
    return (None, 4, value) if rows is None else (rows.data_ptr(), rows.element_size(), 0)


def _heads_last(B, H, L, hd, like):
    """[B, H, L, hd] over memory [B, L, H, hd], so that the projections around it need no copy."""
    return torch.empty((B, L, H, hd), dtype=like.dtype, device=like.device).transpose(1, 2)


def _inputs(q, k, v, bias, max_distance, causal, scale, lengths, start_rows, start):
    """The arguments that both directions begin with."""
    B, H, Lq, hd = q.shape
    starts, n_starts = _starts_array(bias.shape[0], max_distance, causal)
    at, at_bytes, first = _per_row(start_rows, start)
    return (q.data_ptr(), _st(q), k.data_ptr(), _st(k), v.data_ptr(), _st(v), bias.data_ptr(), _DTYPES[bias.dtype],
            bias.shape[0], starts, n_starts, *_per_row(lengths)[:2], at, at_bytes, first, B, H, k.shape[1], Lq,
            k.shape[2], hd, scale, int(causal), _DTYPES[q.dtype])


def _fwd_fake(q, k, v, bias, max_distance, causal, scale, lengths, start_rows, start, want_lse):
    B, H, Lq, hd = q.shape
    return (q.new_empty((B, Lq, H, hd)).transpose(1, 2),
            q.new_empty((B, H, Lq) if want_lse else (0,), dtype=torch.float32))


@_lib.traced_op("bias_attn_fwd", _fwd_fake)
def bias_attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bias: torch.Tensor, max_distance: int,
                  causal: bool, scale: float, lengths: Optional[torch.Tensor], start_rows: Optional[torch.Tensor],
                  start: int, want_lse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(o, lse): lse [B, H, Lq] = log2 of the row's softmax denominator (inf without keys) for the
    backward, empty unless wanted."""
    dev = q.device
    B, H, Lq, hd = q.shape
    q, k, v, bias = _rows16(q), _rows16(k), _rows16(v), bias.contiguous()
    o = _heads_last(B, H, Lq, hd, q)
    lse = torch.empty((B, H, Lq) if want_lse else (0,), dtype=torch.float32, device=dev)
    nbytes = _lib.lib().mb_bias_attn_fwd_workspace(B, H, k.shape[1], Lq, k.shape[2], hd, int(causal))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _lib.call_on(dev, "mb_bias_attn_fwd",
                 *_inputs(q, k, v, bias, max_distance, causal, scale, lengths, start_rows, start),
                 o.data_ptr(), _st(o), lse.data_ptr() if want_lse else None, ws.data_ptr() if nbytes else None, nbytes)
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
    q, k, v, o, d_o = _rows16(q), _rows16(k), _rows16(v), _rows16(o), _rows16(d_o.to(q.dtype))
    bias = bias.contiguous()
    dq, dk, dv = _heads_last(B, H, Lq, hd, q), _heads_last(B, Hk, Lk, hd, k), _heads_last(B, Hk, Lk, hd, v)
    dbias = torch.empty(bias.shape if want_dbias else (0,), dtype=bias.dtype, device=dev)
    nbytes = _lib.lib().mb_bias_attn_bwd_workspace(B, H, Lq, bias.shape[0])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _lib.call_on(dev, "mb_bias_attn_bwd",
                 *_inputs(q, k, v, bias, max_distance, causal, scale, lengths, start_rows, start),
                 o.data_ptr(), _st(o), d_o.data_ptr(), _st(d_o), lse.data_ptr(), dq.data_ptr(), _st(dq),
                 dk.data_ptr(), _st(dk), dv.data_ptr(), _st(dv), dbias.data_ptr() if want_dbias else None,
                 ws.data_ptr(), nbytes)
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
    _lib.require_gpu(q, k, v, bias, lengths, rows, what=what)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} are not [B, H, Lq, hd] "
                         "and twice [B, Hk, Lk, hd]")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q {q.dtype}, k {k.dtype}, v {v.dtype} (supported: all float32 or all bfloat16)")
    if bias.dim() != 2 or bias.shape[1] != q.shape[1] or bias.dtype not in _DTYPES:
        raise ValueError(f"{what}: bias {tuple(bias.shape)} {bias.dtype} is not [buckets, {q.shape[1]}] in float32 or "
                         "bfloat16")
    buckets = bias.shape[0]
    if buckets < 1 or (not causal and buckets % 2):
        raise ValueError(f"{what}: {buckets} buckets (at least one, and an even number without causal)")
    side = buckets if causal else buckets // 2
    if side > MAX_BUCKETS or not side // 2 < max_distance <= MAX_DISTANCE:
        raise ValueError(f"{what}: {side} buckets in a direction up to distance {max_distance} (supported: at most "
                         f"{MAX_BUCKETS}, and a distance above half of them, at most {MAX_DISTANCE})")
    for name, t in (("lengths", lengths), ("q_start", rows)):
        if t is not None and (t.shape != (q.shape[0],) or t.dtype not in (torch.int32, torch.int64)):
            raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype} is not one int32 or int64 for each of "
                             f"{q.shape[0]} rows")


def relative_bias_attention(q, k, v, bias, max_distance=128, causal=True, scale=None, lengths=None, q_start=None):
    """Attention of q [B, H, Lq, hd] over k, v [B, Hk, Lk, hd] (Hk divides H: key heads shared by
    H / Hk query heads each), fp32 or bf16, any strides, head_dim 32, 64 or 128, with ``bias``
    [buckets, H] (fp32 or bf16) added to the scores by distance.  Returns [B, H, Lq, hd].

    ``q_start``: the position of each row's first query among the keys, an int or an int32 / int64
    tensor [B] (within +-2^30); None: Lk - Lq, so that the last query stands at the last key.
    ``causal``: a query sees the keys up to its position.  ``lengths``: an int32 / int64 tensor [B];
    keys from there on are not seen, whatever their rows hold (values in 0 .. Lk; others are taken
    as the nearest of these).  A query that sees no key gets zeros, and passes on no gradient.
    Other values have to be finite.  ``scale``: 1 / sqrt(hd) by default.

    In bf16 the probabilities and the scores' gradients are rounded to bf16 for the products that
    they enter; all sums are in fp32.  Gradients come out the same each time."""
    causal, max_distance = bool(causal), int(max_distance)
    _check(q, k, v, bias, max_distance, causal, lengths, q_start)
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    rows = q_start.contiguous() if torch.is_tensor(q_start) else None
    start = k.shape[2] - q.shape[2] if q_start is None else 0 if rows is not None else int(q_start)
    lengths = None if lengths is None else lengths.contiguous()
    args = (q, k, v, bias, max_distance, causal, scale, lengths, rows, start)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or bias.requires_grad):
        return RelativeBiasAttentionFunction.apply(*args)
    return bias_attn_fwd(*args, False)[0]
