"""RoPE transformer baseline (the comparison model train.py builds with --model rope).

Not on the Per-Slot EMA path: it exists so that train.py's ``from mathbrain.baseline
import RoPETransformerLM`` (train.py:43) resolves and a run can switch models.  The
module tree and parameter names follow mathbrain/baseline.py:31-129 (checkpoints load
by name); the blocks reuse this package's RMSNorm and SwiGLU (one HIP pass per
direction) and torch's scaled_dot_product_attention.  The rotary embedding rotates the
channel pairs (2i, 2i+1) of each head by t * theta^(-2i/hd), written with real cos/sin
tables instead of the reference's complex multiply (the same rotation).

``qk_norm=True`` (not in the reference) norms every query and key head before the rotation,
in the rotation's own pass (``qk_norm_rotary``).  ``rel_buckets=n`` (not in the reference)
adds a learned bias by distance buckets to every layer's scores, one table [n, heads] for all
layers, in the attention that reads it (``relative_bias_attention``, which replaces torch's
there; its probabilities are not dropped out, the block's output is).  The rotation without head
norms is one launch a direction (``apply_rotary``); ``rope_layout``, ``rope_dims`` and ``rope_scaling``
(not in the reference) choose its pairs, the part of each head that turns, and tables for longer
contexts.
"""
import warnings

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib
from .bias_attention import relative_bias_attention
from .model import RMSNorm, SwiGLU, head_loss
from .qk_norm import qk_norm_rotary
from .rotary import LAYOUTS, apply_rotary
from .rotary import rotary_tables as scaled_rotary_tables


def rotary_tables(head_dim, max_len, theta=10000.0):
    """cos and sin [max_len, head_dim / 2] of the angles t * theta^(-2i/head_dim)."""
    inv = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float32) / head_dim)
    ang = torch.arange(max_len, dtype=torch.float32)[:, None] * inv[None, :]
    return ang.cos(), ang.sin()


def rotate(x, cos, sin):
    """Rotates the pairs (x[..., 2i], x[..., 2i+1]) of x [B, L, H, hd] by the step's angles
    (computed in fp32, returned in x's dtype)."""
    xf = x.float().unflatten(-1, (-1, 2))
    a, b = xf[..., 0], xf[..., 1]
    c = cos[None, :, None, :]
    s = sin[None, :, None, :]
    return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2).type_as(x)


def _on_the_kernel(q, cos, sin):
    """Whether apply_rotary takes the rotation of q by these tables: plain GPU tensors in fp32 or bf16, tables of fp32 at most
    that get no derivative and have a row for every position, and no torch.func transform.  Everything else goes through
    ``rotate``'s tensor operations."""
    return (q.is_cuda and q.dtype in (torch.float32, torch.bfloat16)
            and all(t.dtype is not torch.float64 and t.shape[0] >= q.shape[1] and not (t.requires_grad and torch.is_grad_enabled())
                    for t in (cos, sin))
            and (torch.compiler.is_compiling()
                 or (type(q) is torch.Tensor and torch._C._functorch.peek_interpreter_stack() is None and not _lib.has_tangent(cos, sin))))


class CausalSelfAttention(nn.Module):
    """baseline.py:31-70."""

    def __init__(self, d_model: int, n_heads: int, dropout: float = 0.0, qk_norm: bool = False,
                 rope_layout: str = "interleaved"):
        super().__init__()
        assert d_model % n_heads == 0
        self.rope_layout = rope_layout
        self.d_model = d_model
        self.n_heads = n_heads
        self.head_dim = d_model // n_heads
        self.wq = nn.Linear(d_model, d_model, bias=False)
        self.wk = nn.Linear(d_model, d_model, bias=False)
        self.wv = nn.Linear(d_model, d_model, bias=False)
        self.wo = nn.Linear(d_model, d_model, bias=False)
        self.resid_dropout = nn.Dropout(dropout)
        if qk_norm:
            # their weights and eps; the norms run in the rotation's pass
            self.q_norm = RMSNorm(self.head_dim)
            self.k_norm = RMSNorm(self.head_dim)
        self.qk_norm = qk_norm

    def forward(self, x, cos, sin, rel_bias=None, rel_max_distance=128):
        B, L, D = x.shape
        shape = (B, L, self.n_heads, self.head_dim)
        q, k = self.wq(x).view(shape), self.wk(x).view(shape)
        if self.qk_norm:
            q, k = qk_norm_rotary(q, k, self.q_norm.weight, self.k_norm.weight, cos.float(), sin.float(),
                                  self.q_norm.eps)
        elif _on_the_kernel(q, cos, sin):
            q, k = apply_rotary(q, k, cos.float().contiguous(), sin.float().contiguous(), layout=self.rope_layout)
        else:
            if self.rope_layout != "interleaved" or 2 * cos.shape[1] != self.head_dim:
                raise ValueError("CausalSelfAttention: rope_layout and rope_dims take float32 or bfloat16 on the GPU, tables without "
                                 f"gradients and no torch.func transform (got {q.dtype} on {q.device})")
            q, k = rotate(q, cos, sin), rotate(k, cos, sin)
        q, k = q.transpose(1, 2), k.transpose(1, 2)
        v = self.wv(x).view(shape).transpose(1, 2)
        if rel_bias is not None:
            out = relative_bias_attention(q, k, v, rel_bias, rel_max_distance)
        else:
            out = F.scaled_dot_product_attention(q, k, v, is_causal=True,
                                                 dropout_p=self.resid_dropout.p if self.training else 0.0)
        return self.resid_dropout(self.wo(out.transpose(1, 2).reshape(B, L, D)))


class RoPETransformerBlock(nn.Module):
    """baseline.py:72-84."""

    def __init__(self, d_model: int, n_heads: int, d_ff: int, dropout: float = 0.0, qk_norm: bool = False,
                 rope_layout: str = "interleaved"):
        super().__init__()
        self.attn_norm = RMSNorm(d_model)
        self.attn = CausalSelfAttention(d_model, n_heads, dropout, qk_norm, rope_layout)
        self.ffn_norm = RMSNorm(d_model)
        self.ffn = SwiGLU(d_model, d_ff)

    def forward(self, x, cos, sin, rel_bias=None, rel_max_distance=128):
        x = x + self.attn(self.attn_norm(x), cos, sin, rel_bias, rel_max_distance)
        return x + self.ffn(self.ffn_norm(x))


class RoPETransformerLM(nn.Module):
    """baseline.py:86-129: RoPETransformerLM(vocab_size, d_model, n_layers, n_heads,
    max_seq_len=4096, dropout=0.1); forward(x [B, L]) -> logits [B, L, vocab_size].
    ``qk_norm``: RMS norms of every query and key head.  ``rel_buckets``: a learned bias by that
    many distance buckets, up to ``rel_max_distance`` (0: none); the probabilities are not dropped
    out then, and a ``dropout`` above 0 warns of it.  Both take head_dim 32, 64 or 128; the bias
    starts as zeros.  ``rope_layout``: "interleaved" (the reference's) or "half"; ``rope_dims``: the first channels of
    each head that turn (all); ``rope_scaling``: keyword arguments of rotary.rotary_tables for longer contexts, such as
    dict(scaling="yarn", factor=4, trained=4096).  With ``qk_norm`` whole heads turn, interleaved.

    forward(x, targets) is the mean cross entropy over the targets that are not ``ignore_index``, without the logits
    (``linear_cross_entropy`` with lm_head's weight)."""

    def __init__(self, vocab_size: int, d_model: int, n_layers: int, n_heads: int,
                 max_seq_len: int = 4096, dropout: float = 0.1, qk_norm: bool = False,
                 rel_buckets: int = 0, rel_max_distance: int = 128, rope_layout: str = "interleaved", rope_dims=None,
                 rope_scaling=None):
        super().__init__()
        head_dim = d_model // n_heads
        if rope_layout not in LAYOUTS:
            raise ValueError(f"RoPETransformerLM: rope_layout={rope_layout!r} ('interleaved' or 'half')")
        if rope_dims is not None and not (0 < rope_dims <= head_dim and rope_dims % 2 == 0):
            raise ValueError(f"RoPETransformerLM: rope_dims={rope_dims} (an even number, at most head_dim {head_dim})")
        if qk_norm and (rope_layout != "interleaved" or rope_dims not in (None, head_dim)):
            raise ValueError("RoPETransformerLM: qk_norm turns whole heads, interleaved")
        if rel_buckets and dropout:
            warnings.warn(f"RoPETransformerLM: with rel_buckets the attention's probabilities are not dropped out; "
                          f"dropout={dropout} is that of the blocks' outputs alone", stacklevel=2)
        self.vocab_size = vocab_size
        self.d_model = d_model
        self.embed = nn.Embedding(vocab_size, d_model)
        d_ff = 256 * ((int(8 * d_model / 3) + 255) // 256)
        self.layers = nn.ModuleList([RoPETransformerBlock(d_model, n_heads, d_ff, dropout, qk_norm, rope_layout)
                                     for _ in range(n_layers)])
        self.final_norm = RMSNorm(d_model)
        self.lm_head = nn.Linear(d_model, vocab_size, bias=False)
        self.lm_head.weight = self.embed.weight
        self.rel_bias = nn.Parameter(torch.zeros(rel_buckets, n_heads)) if rel_buckets else None
        self.rel_max_distance = rel_max_distance
        if rope_dims is None and rope_scaling is None:
            cos, sin = rotary_tables(head_dim, max_seq_len)
        else:
            cos, sin = scaled_rotary_tables(rope_dims or head_dim, max_seq_len, **(rope_scaling or {}))
        self.register_buffer("rope_cos", cos, persistent=False)
        self.register_buffer("rope_sin", sin, persistent=False)

    def forward(self, x, targets=None, ignore_index=-1):
        L = x.shape[1]
        cos, sin = self.rope_cos[:L], self.rope_sin[:L]
        h = self.embed(x)
        for layer in self.layers:
            h = layer(h, cos, sin, self.rel_bias, self.rel_max_distance)
        h = self.final_norm(h)
        if targets is not None:
            return head_loss(self.lm_head, h, targets, ignore_index)
        return self.lm_head(h)
