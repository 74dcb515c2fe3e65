"""RoPETransformerLM with its options (query/key norms, a learned bias by distance buckets) and
clip_grad_norm_, run together as a training program runs them, against the same model written in
float64 on the CPU; and what the options leave as it was.

Tolerance of the fp32 model: norm-wise, 2e-5 for logits and 1e-4 for gradients.  A layer's products
sum at most 256 terms in fp32 (256 * 2^-24 = 1.5e-5 of the terms' sizes in the worst order, a
tenth of that in a blocked one) and two layers with their norms pass about ten of them on."""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

V, D, HEADS, LAYERS = 97, 128, 4, 2
OPTIONS = [dict(qk_norm=True), dict(rel_buckets=16, rel_max_distance=40), dict(qk_norm=True, rel_buckets=16, rel_max_distance=40)]


def model(**options):
    from mathbrain.baseline import RoPETransformerLM
    torch.manual_seed(0)
    m = RoPETransformerLM(V, D, LAYERS, HEADS, max_seq_len=256, dropout=0.0, **options)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if "rel_bias" in name:
                p.copy_(torch.randn(p.shape, generator=g))
            elif p.dim() == 1:
                p.add_(0.2 * torch.randn(p.shape, generator=g))
    return m.cuda()


def norm(x, w):
    return w * x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()


def definition(m, p, x, options):
    """The model's logits in float64 from the parameters p."""
    from mathbrain.bias_attention import bucket_starts
    B, L = x.shape
    hd = D // HEADS
    cos, sin = (t[:L].cpu().double()[:, None] for t in (m.rope_cos, m.rope_sin))
    h = p["embed.weight"][x]
    i = torch.arange(L)
    dist = i[:, None] - i
    for n in range(LAYERS):
        w = {k[len(f"layers.{n}."):]: v for k, v in p.items() if k.startswith(f"layers.{n}.")}
        y = norm(h, w["attn_norm.weight"])
        q, k, v = ((y @ w[f"attn.w{c}.weight"].T).view(B, L, HEADS, hd) for c in "qkv")
        if options.get("qk_norm"):
            q, k = norm(q, w["attn.q_norm.weight"]), norm(k, w["attn.k_norm.weight"])
        q, k = (torch.stack((t[..., 0::2] * cos - t[..., 1::2] * sin, t[..., 0::2] * sin + t[..., 1::2] * cos), -1).flatten(-2)
                for t in (q, k))
        s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(hd)
        if options.get("rel_buckets"):
            starts = bucket_starts(options["rel_buckets"], options["rel_max_distance"])
            bucket = sum((dist >= s0).long() for s0 in starts) - 1
            s = s + p["rel_bias"][bucket.clamp(min=0)].permute(2, 0, 1)
        a = s.masked_fill(dist < 0, -math.inf).softmax(-1)
        h = h + torch.einsum("bhij,bjhd->bihd", a, v).reshape(B, L, D) @ w["attn.wo.weight"].T
        y = norm(h, w["ffn_norm.weight"])
        h = h + (F.silu(y @ w["ffn.w1.weight"].T) * (y @ w["ffn.w3.weight"].T)) @ w["ffn.w2.weight"].T
    return norm(h, p["final_norm.weight"]) @ p["embed.weight"].T


def off(a, b):
    return float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm().clamp(min=1e-30))


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("L", [1, 63, 200])
def test_a_training_step_against_float64(options, L):
    from mathbrain.grad_clip import clip_grad_norm_
    m = model(**options)
    x = torch.randint(0, V, (3, L), generator=torch.Generator().manual_seed(2))
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in m.named_parameters()}
    want = definition(m, p, x, options)
    logits = m(x.cuda())
    assert off(logits, want) < 2e-5
    target = torch.randint(0, V, (3 * L,), generator=torch.Generator().manual_seed(3))
    F.cross_entropy(want.view(-1, V), target).backward()
    F.cross_entropy(logits.view(-1, V), target.cuda()).backward()
    total = math.sqrt(sum(float(t.grad.square().sum()) for t in p.values()))
    worst = {k: float((v.grad.cpu().double() - p[k].grad).norm()) / total for k, v in m.named_parameters()}
    assert max(worst.values()) < 1e-4, worst
    got = clip_grad_norm_(m.parameters(), 0.5 * total)
    assert abs(float(got) - total) < 1e-4 * total
    for k, v in m.named_parameters():
        assert float((v.grad.cpu().double() - 0.5 * p[k].grad).norm()) < 1e-4 * total, k


def test_steps_under_bf16_autocast():
    """The options train under autocast: finite losses and gradients, of the parameters' types, and the
    bf16 logits within bf16's steps of the fp32 ones (2 layers, about 20 roundings of 2^-8 norm-wise
    and independent: sqrt(20) * 2^-8 < 2e-2; held to 5e-2)."""
    from mathbrain.grad_clip import clip_grad_norm_
    m = model(qk_norm=True, rel_buckets=32)
    x = torch.randint(0, V, (4, 130), device="cuda")
    opt = torch.optim.AdamW(m.parameters(), lr=1e-3)
    with torch.no_grad():
        full = m(x)
    for step in range(3):
        opt.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            logits = m(x)
            loss = F.cross_entropy(logits.view(-1, V), x.view(-1))
        if step == 0:
            assert off(logits.float(), full.cpu().double()) < 5e-2
        loss.backward()
        norm_ = clip_grad_norm_(m.parameters(), 1.0, error_if_nonfinite=True)
        assert torch.isfinite(loss) and float(norm_) > 0
        for k, v in m.named_parameters():
            assert v.grad is not None and v.grad.dtype == v.dtype and torch.isfinite(v.grad).all(), k
        assert m.rel_bias.grad.abs().sum() > 0
        opt.step()


def test_a_model_in_bf16_throughout():
    """model.bfloat16(): weights, tables and bias in bf16; finite losses and gradients of that type, and
    logits within bf16's steps of the fp32 model's (as under autocast, and the tables' and weights'
    roundings: held to 1e-1)."""
    m = model(qk_norm=True, rel_buckets=32)
    x = torch.randint(0, V, (4, 130), device="cuda")
    with torch.no_grad():
        full = m(x)
    m = m.bfloat16()
    logits = m(x)
    assert logits.dtype == torch.bfloat16 and off(logits.float(), full.cpu().double()) < 1e-1
    F.cross_entropy(logits.view(-1, V).float(), x.view(-1)).backward()
    for k, v in m.named_parameters():
        assert v.grad.dtype == torch.bfloat16 and torch.isfinite(v.grad).all(), k


def test_the_model_without_options_is_what_it_was():
    m = model()
    assert not any("norm.weight" in k and ("q_norm" in k or "k_norm" in k) or "rel_bias" in k for k in m.state_dict())
    x = torch.randint(0, V, (2, 50), device="cuda")
    plain = copy.deepcopy(m)
    assert torch.equal(m(x), plain(x))
    p = {k: v.detach().cpu().double() for k, v in m.named_parameters()}
    assert off(m(x), definition(m, p, x.cpu(), {})) < 2e-5


def test_traced_without_breaks():
    m = model(qk_norm=True, rel_buckets=16)
    x = torch.randint(0, V, (2, 40), device="cuda")
    assert torch._dynamo.explain(m)(x).graph_break_count == 0
    compiled = torch.compile(m, backend="aot_eager")
    a, b = m(x), compiled(x)
    assert torch.equal(a, b)
    ga = torch.autograd.grad(a.square().sum(), list(m.parameters()))
    gb = torch.autograd.grad(b.square().sum(), list(m.parameters()))
    for u, v in zip(ga, gb):
        assert torch.allclose(u, v, rtol=1e-4, atol=1e-4 * float(u.abs().max()))


def test_tokens_one_by_one_agree_with_the_whole_sequence():
    """Prompts of different lengths read into caches, then a token at a time, against each sequence
    read at once.  Both sides are off from the exact output by at most dp |v| with (in units of 2^-24)
    dp = 2 (hd + 8) (|q||k| / sqrt(hd) + |bias|) + 2 n + 16 for n keys, where normed rows with weights
    of 1 have |q||k| <= hd: 144 (8 + 4) + 156 = 1884, 1.2e-4 each; the rotated rows' own error of
    2e-6 moves a score by 4e-6 * 8 at most, p by 7e-5.  Together under 4e-4 of the largest |v|."""
    from mathbrain.baseline import rotary_tables
    from mathbrain.bias_attention import relative_bias_attention
    from mathbrain.qk_norm import qk_norm_rotary
    B, H, Hk, hd, room, steps = 3, 4, 2, 64, 70, 6
    g = torch.Generator().manual_seed(9)
    prompts = [5, 17, 40]
    x = [torch.randn(B, room, n, hd, generator=g).cuda() for n in (H, Hk, Hk)]
    bias = torch.randn(32, H, generator=g).clamp(-4, 4).cuda()
    w = torch.ones(hd, device="cuda")
    cos, sin = (t.cuda() for t in rotary_tables(hd, room))

    def layer(b, upto):
        q, k = qk_norm_rotary(x[0][b:b + 1, :upto], x[1][b:b + 1, :upto], w, w, cos, sin)
        return relative_bias_attention(q.transpose(1, 2), k.transpose(1, 2), x[2][b:b + 1, :upto].transpose(1, 2), bias)
    caches = [torch.full((B, room, Hk, hd), float("nan"), device="cuda") for _ in range(2)]
    most = max(prompts)
    lengths = torch.tensor(prompts, device="cuda")
    # the padded batch of prompts; what stands behind a prompt's end is written over token by token
    q, k = qk_norm_rotary(x[0][:, :most], x[1][:, :most], w, w, cos, sin)
    caches[0][:, :most], caches[1][:, :most] = k, x[2][:, :most]
    out = relative_bias_attention(q.transpose(1, 2), *(c.transpose(1, 2) for c in caches), bias, lengths=lengths, q_start=0)
    bound = 4e-4 * float(x[2].abs().max())
    for b, n in enumerate(prompts):
        assert float((out[b, :, :n] - layer(b, n)[0]).abs().max()) <= bound
    rows = torch.arange(B, device="cuda")
    for _ in range(steps):
        q, k = qk_norm_rotary(x[0][rows, lengths][:, None], x[1][rows, lengths][:, None], w, w, cos, sin, start=lengths)
        caches[0][rows, lengths], caches[1][rows, lengths] = k[:, 0], x[2][rows, lengths]
        lengths = lengths + 1
        out = relative_bias_attention(q.transpose(1, 2), *(c.transpose(1, 2) for c in caches), bias, lengths=lengths,
                                      q_start=lengths - 1)
        for b, n in enumerate(lengths.tolist()):
            assert float((out[b, :, 0] - layer(b, n)[0, :, -1]).abs().max()) <= bound, (b, n)
