"""apply_rotary and its tables (mathbrain/rotary.py) against the rotation by complex numbers in 64 bits.

Roundings: fp32 products and sums round to 2^-24 of values up to |x| (|c|, |s| <= 1): out is within
3 * 2^-24 * (|a| + |b|) of the exact one; bf16 adds its own half step, 2^-9 of the result's binade,
at most 2^-8 relative."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def tables(d, n, seed=0):
    from mathbrain.rotary import rotary_tables
    return tuple(t.cuda() for t in rotary_tables(d, n))


def want(x, cos, sin, at, layout, inverse=False):
    """x [B, L, H, hd] turned in 64 bits; `at` [B, L]."""
    d = 2 * cos.shape[1]
    y = x.double().clone()
    spin = torch.complex(cos.double(), sin.double())[at][:, :, None, :]
    spin = spin.conj() if inverse else spin
    i = torch.arange(d // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + d // 2)
    z = torch.complex(y[..., a], y[..., b]) * spin
    y[..., a], y[..., b] = z.real, z.imag
    return y


def check(got, exact, x, t):
    assert got.dtype == t and got.is_contiguous() and got.shape == x.shape
    size = x.double().abs().amax(-1, keepdim=True)
    room = 6 * 2.0**-24 * size + (2.0**-8 * exact.abs() if t == torch.bfloat16 else 0.0)
    assert ((got.double() - exact).abs() <= room).all()


CASES = [  # B, L, H, Hk, hd, turned
    (1, 1, 1, 1, 64, 64), (2, 5, 8, 8, 64, 64), (3, 33, 4, 2, 128, 64), (2, 17, 3, 1, 32, 16), (1, 70, 5, 5, 80, 20),
    (2, 9, 2, 1, 96, 96), (1, 3, 1, 1, 2, 2), (2, 4, 3, 3, 30, 30), (1, 6, 2, 2, 33, 10), (4, 1, 16, 4, 256, 64), (2, 3, 2, 2, 64, 0)]


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,L,H,Hk,hd,d", CASES)
def test_forward_and_gradients(B, L, H, Hk, hd, d, layout, t):
    from mathbrain.rotary import apply_rotary
    g = torch.Generator("cuda").manual_seed(B * L + hd)
    q, k, gq, gk = (torch.randn(B, L, n, hd, generator=g, device="cuda").to(t) for n in (H, Hk, H, Hk))
    q.requires_grad_(), k.requires_grad_()
    cos, sin = tables(d, 100) if d else (torch.empty(100, 0, device="cuda"),) * 2
    for start in (0, 7, torch.randint(0, 100 - L + 1, (B,), generator=g, device="cuda"),
                  torch.randint(0, 100, (B, L), generator=g, device="cuda", dtype=torch.int32)):
        at = torch.arange(L, device="cuda").expand(B, L)
        at = start.long() if torch.is_tensor(start) and start.dim() == 2 else at + (start[:, None] if torch.is_tensor(start) else start)
        qo, ko = apply_rotary(q, k, cos, sin, start, layout)
        dq, dk = torch.autograd.grad([qo, ko], [q, k], [gq, gk])
        for got, x, inverse in ((qo, q, False), (ko, k, False), (dq, gq, True), (dk, gk, True)):
            check(got, want(x.detach(), cos, sin, at, layout, inverse), x.detach(), t)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_bit_for_bit_as_rotate(t):
    from mathbrain import baseline
    from mathbrain.rotary import apply_rotary
    q, k = (torch.randn(3, 50, n, 64, device="cuda").to(t).requires_grad_() for n in (8, 4))
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    cos, sin = (x.cuda() for x in baseline.rotary_tables(64, 50))
    got = apply_rotary(q, k, cos, sin)
    old = baseline.rotate(q, cos, sin), baseline.rotate(k, cos, sin)
    for a, b in zip((*got, *torch.autograd.grad(got, [q, k], [gq, gk])), (*old, *torch.autograd.grad(old, [q, k], [gq, gk]))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_strides_and_offsets(layout):
    from mathbrain.rotary import apply_rotary
    cos, sin = tables(64, 40)
    at = torch.arange(9, device="cuda").expand(2, 9)
    base = torch.randn(2, 9, 3 * 4 * 64 + 3, device="cuda").bfloat16()
    views = [base[..., :768].view(2, 9, 12, 64)[:, :, :4], base[..., 1:257].unflatten(-1, (4, 64)),       # odd addresses
             torch.randn(2, 4, 9, 64, device="cuda").bfloat16().transpose(1, 2),                            # heads first
             torch.randn(2, 9, 64, 4, device="cuda").bfloat16().transpose(2, 3),                            # channels apart
             torch.randn(2, 1, 4, 64, device="cuda").bfloat16().expand(2, 9, 4, 64)]                        # one row for all
    for q in views:
        for k in (views[0], views[1]):
            for got, x in zip(apply_rotary(q, k, cos, sin, layout=layout), (q, k)):
                check(got, want(x, cos, sin, at, layout), x, torch.bfloat16)


def test_positions_outside_the_tables():
    from mathbrain.rotary import apply_rotary
    cos, sin = tables(32, 10)
    q = torch.randn(3, 2, 2, 64, device="cuda")
    start = torch.tensor([-1, 9, 2**40], device="cuda")
    qo, ko = apply_rotary(q, q, cos, sin, start)
    bad = torch.tensor([[True, False], [False, True], [True, True]], device="cuda")
    assert torch.equal(qo[..., :32].isnan().all(-1).all(-1), bad) and torch.equal(qo[..., :32].isnan().any(-1).any(-1), bad)
    assert torch.equal(qo[..., 32:], q[..., 32:]) and torch.equal(qo.nan_to_num(), ko.nan_to_num())


def test_special_values_stay_in_their_pairs():
    from mathbrain.rotary import apply_rotary
    cos, sin = tables(64, 8)
    q = torch.randn(1, 8, 2, 64, device="cuda")
    q[0, 3, 1, 10] = math.nan
    q[0, 5, 0, 0] = math.inf
    qo, _ = apply_rotary(q, q, cos, sin)
    assert (~qo.isfinite()).sum() == 4 and not qo[0, 3, 1, 10:12].isfinite().any() and not qo[0, 5, 0, :2].isfinite().any()


def test_empty_and_one_sided_calls():
    from mathbrain.rotary import apply_rotary
    cos, sin = tables(64, 8)
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        a, b = apply_rotary(x, x, cos, sin)
        (a.sum() + b.sum()).backward()
        assert a.shape == shape and x.grad.shape == shape
    q, k = (torch.randn(2, 4, n, 64, device="cuda", requires_grad=True) for n in (2, 1))
    qo, ko = apply_rotary(q, k, cos, sin)
    dk, = torch.autograd.grad(ko.sum(), k)                   # nothing arrives at q's side
    at = torch.arange(4, device="cuda").expand(2, 4)
    check(dk, want(torch.ones_like(k), cos, sin, at, "interleaved", True), torch.ones_like(k), torch.float32)
    nothing = q[:, :, :0].detach()
    check(apply_rotary(q.detach(), nothing, cos, sin)[0], want(q.detach(), cos, sin, at, "interleaved"), q.detach(), torch.float32)


def test_higher_derivatives_and_forward_mode():
    import torch.autograd.forward_ad as fwad
    from mathbrain.rotary import apply_rotary
    cos, sin = tables(32, 8)
    q, k, tq = (torch.randn(1, 3, 2, 64, device="cuda") for _ in range(3))
    q.requires_grad_()
    g = torch.randn_like(q).requires_grad_()
    dq, = torch.autograd.grad(apply_rotary(q, k, cos, sin)[0], q, g, create_graph=True)
    back, = torch.autograd.grad(dq, g, tq)                   # the rotation's own derivative is the rotation
    assert torch.equal(back, apply_rotary(tq, k, cos, sin)[0])
    with fwad.dual_level():
        qo, ko = apply_rotary(fwad.make_dual(q.detach(), tq), k, cos, sin, layout="half")
        assert torch.equal(fwad.unpack_dual(qo).tangent, apply_rotary(tq, k, cos, sin, layout="half")[0])
        with pytest.raises(ValueError, match="derivative"):
            apply_rotary(k, k, fwad.make_dual(cos, cos), sin)


def test_gradient_against_differences():
    from mathbrain.rotary import apply_rotary
    cos, sin = tables(8, 6)
    q = torch.randn(1, 6, 1, 12, device="cuda", requires_grad=True)
    w = torch.randn(1, 6, 1, 12, device="cuda")
    f = lambda x: float((apply_rotary(x, x, cos, sin, layout="half")[0].double() * w).sum())
    dq, = torch.autograd.grad((apply_rotary(q, q, cos, sin, layout="half")[0] * w).sum(), q)
    for i in (0, 5, 13, 40, 71):
        e = torch.zeros(72, device="cuda")
        e[i] = 0.5                                            # linear: a large step costs nothing
        e = e.view_as(q)
        x = q.detach()
        assert abs((f(x + e) - f(x - e)) - float(dq.flatten()[i])) < 72 * 4 * 2.0**-24 * float(x.abs().max() + 1) * 4


def test_captured_and_on_another_stream():
    from mathbrain.rotary import apply_rotary
    cos, sin = tables(64, 64)
    q, k = (torch.randn(2, 8, 4, 64, device="cuda").bfloat16() for _ in range(2))
    start = torch.tensor([3, 9], device="cuda")
    apply_rotary(q, k, cos, sin, start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_rotary(q, k, cos, sin, start)
    for step in range(3):
        start += step
        q.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, apply_rotary(q, k, cos, sin, start)):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = apply_rotary(q, k, cos, sin, start)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there[0], out[0])


def test_many_tokens():
    """Positions and offsets of a tensor beyond 2^31 elements (bf16, 4.3 GB): its ends against a small call."""
    from mathbrain.rotary import apply_rotary
    cos, sin = tables(64, 2100)
    B, L = 16500, 2050
    q = torch.empty(B, L, 1, 64, device="cuda", dtype=torch.bfloat16)
    q[0], q[-1] = torch.randn(2, L, 1, 64, device="cuda").bfloat16()
    k = q[:, :, :0]
    out, _ = apply_rotary(q, k, cos, sin)
    ends = apply_rotary(q[[0, -1]], k[[0, -1]], cos, sin)[0]
    assert torch.equal(out[0], ends[0]) and torch.equal(out[-1], ends[1])


def test_refusals():
    from mathbrain import _lib
    from mathbrain.rotary import apply_rotary, rotary_tables
    cos, sin = tables(64, 8)
    q = torch.randn(2, 4, 2, 64, device="cuda")
    for bad in (dict(k=q[:, :3]), dict(k=q.bfloat16()), dict(cos=cos[:, :16]), dict(cos=cos.double()), dict(layout="other"),
                dict(start=torch.zeros(3, device="cuda", dtype=torch.int32)), dict(start=torch.zeros(2, device="cuda")),
                dict(cos=cos.clone().requires_grad_()), dict(q=q.half(), k=q.half()), dict(q=q[..., :32], k=q[..., :32]),
                dict(cos=cos.t().contiguous().t())):
        with pytest.raises(ValueError):
            apply_rotary(**(dict(q=q, k=q, cos=cos, sin=sin) | bad))
    with pytest.raises(NotImplementedError):
        apply_rotary(q.cpu(), q.cpu(), cos.cpu(), sin.cpu())
    for start in (-1, 5):
        with pytest.raises(_lib.HipKernelError, match="pass the table"):
            apply_rotary(q, q, cos, sin, start)


def test_the_model_turns_as_it_did_and_with_options():
    import torch.nn.functional as F
    from mathbrain import baseline
    torch.manual_seed(0)
    m = baseline.RoPETransformerLM(300, 128, 2, 2, max_seq_len=64, dropout=0.0).cuda()
    x = torch.randint(0, 300, (2, 50), device="cuda")
    logits = m(x)
    saved = baseline.apply_rotary
    baseline.apply_rotary = lambda q, k, cos, sin, layout: (baseline.rotate(q, cos, sin), baseline.rotate(k, cos, sin))
    try:
        assert torch.equal(m(x), logits)
    finally:
        baseline.apply_rotary = saved
    torch.manual_seed(0)
    half = baseline.RoPETransformerLM(300, 128, 2, 2, max_seq_len=64, dropout=0.0, rope_layout="half").cuda()
    # the halves' pairs are the neighbours' of heads whose projections have their rows in that order
    order = torch.arange(128).view(2, 32, 2).transpose(1, 2).reshape(-1).cuda()
    for a, b in zip(half.layers, m.layers):
        a.attn.wq.weight.data.copy_(b.attn.wq.weight[order])
        a.attn.wk.weight.data.copy_(b.attn.wk.weight[order])
    assert (half(x) - logits).abs().max() < 1e-4 * logits.abs().max()
    part = baseline.RoPETransformerLM(300, 128, 2, 2, max_seq_len=64, dropout=0.0, rope_dims=16,
                                      rope_scaling=dict(scaling="yarn", factor=4.0, trained=16)).cuda()
    F.cross_entropy(part(x).view(-1, 300), x.view(-1)).backward()
    assert all(p.grad.isfinite().all() for p in part.parameters()) and part.rope_cos.shape == (64, 8)
    for bad in (dict(rope_layout="x"), dict(rope_dims=7), dict(rope_dims=66), dict(qk_norm=True, rope_dims=16)):
        with pytest.raises(ValueError):
            baseline.RoPETransformerLM(300, 128, 2, 2, **bad)


@pytest.mark.parametrize("options", [{}, dict(rope_layout="half", rope_dims=16), dict(rel_buckets=8)])
@pytest.mark.parametrize("targets", [False, True])
def test_the_model_traces_into_one_graph(options, targets):
    """torch.compile of the training step makes one graph of the model, with the eager step's results.  The traced step
    calls the same kernels in the same order; sums of shared gradients may be taken in another one: 2^-24 of the terms each."""
    from mathbrain.baseline import RoPETransformerLM
    torch.manual_seed(3)
    m = RoPETransformerLM(400, 128, 2, 4, max_seq_len=64, dropout=0.0, **options).cuda()
    args = [torch.randint(0, 400, (2, 48), device="cuda") for _ in range(1 + targets)]
    torch._dynamo.reset()
    assert torch._dynamo.explain(m)(*args).graph_break_count == 0
    torch._dynamo.reset()
    compiled = torch.compile(m, backend="aot_eager", fullgraph=True)
    a, b = m(*args), compiled(*args)
    assert torch.equal(a, b)
    ga, gb = (torch.autograd.grad(x.square().mean(), list(m.parameters())) for x in (a, b))
    for u, v in zip(ga, gb):
        assert torch.allclose(u, v, rtol=1e-4, atol=1e-4 * float(u.abs().max()))


@pytest.mark.parametrize("sides", ["both", "q", "k"])
@pytest.mark.parametrize("start", ["int", "rows", "tokens"])
def test_traced_gradients(start, sides):
    """The same function compiled and not, with a gradient for both results or one of them."""
    from mathbrain.rotary import apply_rotary, rotary_tables
    torch.manual_seed(4)
    q, k = torch.randn(3, 5, 4, 32, device="cuda"), torch.randn(3, 5, 2, 32, device="cuda")
    cos, sin = rotary_tables(32, 40, device="cuda")
    at = {"int": 3, "rows": torch.tensor([0, 30, 7], device="cuda"),
          "tokens": torch.randint(0, 40, (3, 5), device="cuda", dtype=torch.int32)}[start]

    def run(f):
        x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
        a, b = f(x, y)
        loss = sum((t * t * t).sum() for side, t in (("q", a), ("k", b)) if sides in ("both", side))
        return a, b, *torch.autograd.grad(loss, [x, y], materialize_grads=True)

    torch._dynamo.reset()
    eager = run(lambda x, y: apply_rotary(x, y, cos, sin, at, "half"))
    traced = run(torch.compile(lambda x, y: apply_rotary(x, y, cos, sin, at, "half"), backend="aot_eager", fullgraph=True))
    assert all(torch.equal(a, b) for a, b in zip(eager, traced))
