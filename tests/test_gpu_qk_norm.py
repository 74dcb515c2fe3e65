"""qk_norm_rotary (mathbrain/qk_norm.py) against its definition in float64 on the CPU: outputs and
the gradients of q, k and both weights, at every head width and type, odd lengths and head
counts, strided views, positions per row, and the refused calls.

Tolerances, element by element.  An output in bf16 is off by its rounding, half a step
(finfo.eps / 2 of the value).  The fp32 evaluation before it adds at most about 12 roundings to
the row's factor and 4 to the rotation's two terms: 16 * 2^-24 < 1e-6 of the terms' sizes, held
to 2e-6.  dx adds the mean over the row, whose terms are bounded by rs (|w g| + |n| mean|w g n|):
24 roundings, 1.5e-6, held to 4e-6 of that.  A weight's gradient is a sum in which a term goes
through at most 64 additions in these tests: 64 * 2^-24 = 4e-6 and 1e-6 of the term itself,
held to 1e-5 of the sum of the terms' sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-6


def tables(hd, n):
    from mathbrain.baseline import rotary_tables
    return rotary_tables(hd, n)


def turn(x, c, s):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def definition(x, w, c, s, dy):
    """y, dx, dw in float64, and the sizes that their errors are measured by."""
    x, w, dy, c, s = (t.double() for t in (x, w, dy, c, s))
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = x * r
    y = turn(n * w, c, s)
    g = turn(dy, c, -s)
    gw = g * w
    dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
    ysize = turn((n * w).abs(), c.abs(), -s.abs()).abs() + turn((n * w).abs(), c.abs(), s.abs()).abs()
    gsize = (turn(dy.abs(), c.abs(), s.abs()).abs() + turn(dy.abs(), c.abs(), -s.abs()).abs())
    dxsize = r * (gsize * w.abs() + n.abs() * (gsize * w.abs() * n.abs()).mean(-1, keepdim=True))
    return y, dx, (g * n).sum((0, 1, 2)), ysize, dxsize, (gsize * n.abs()).sum((0, 1, 2))


def close(got, want, size, mul, what):
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype == torch.bfloat16 else 0.0
    off = (got.double() - want).abs() - half * want.abs() - mul * (1 + half) * size
    assert torch.isfinite(got).all() and float(off.max()) <= 0, (what, float(off.max()))


def check(q, k, start, hd, seed, n=300):
    """q, k: GPU views; runs both directions against the definition."""
    from mathbrain.qk_norm import qk_norm_rotary
    g = torch.Generator().manual_seed(seed)
    B, L = q.shape[:2]
    cos, sin = tables(hd, n)
    w = [(1 + 0.3 * torch.randn(hd, generator=g)) for _ in range(2)]
    dy = [torch.randn(t.shape, generator=g).to(t.dtype) for t in (q, k)]
    leaves = [q.detach().requires_grad_(), k.detach().requires_grad_(), w[0].cuda().requires_grad_(),
              w[1].cuda().requires_grad_()]
    out = qk_norm_rotary(*leaves, cos.cuda(), sin.cuda(), EPS, start)
    grads = torch.autograd.grad(out, leaves, [d.cuda() for d in dy])
    at = (start.cpu().long()[:, None] if torch.is_tensor(start) else start) + torch.arange(L).expand(B, L)
    c, s = cos[at][:, :, None], sin[at][:, :, None]
    for i, x in enumerate((q, k)):
        y, dx, dw, ysize, dxsize, dwsize = definition(x.cpu(), w[i], c, s, dy[i])
        assert out[i].shape == x.shape and out[i].dtype == x.dtype and out[i].is_contiguous()
        close(out[i], y, ysize, 2e-6, f"out {i}")
        close(grads[i], dx, dxsize, 4e-6, f"dx {i}")
        close(grads[2 + i], dw, dwsize, 1e-5, f"dw {i}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("B,L,H,Hk", [(1, 1, 1, 1), (3, 17, 8, 8), (2, 33, 10, 5), (2, 7, 5, 1), (1, 130, 3, 3)])
def test_matches_the_definition(dtype, hd, B, L, H, Hk):
    g = torch.Generator().manual_seed(B * 1000 + L + hd)
    q = (2 * torch.randn(B, L, H, hd, generator=g)).to(dtype).cuda()
    k = (0.5 * torch.randn(B, L, Hk, hd, generator=g)).to(dtype).cuda()
    check(q, k, 0, hd, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_positions_for_each_row(dtype):
    g = torch.Generator().manual_seed(3)
    q = torch.randn(5, 4, 6, 64, generator=g).to(dtype).cuda()
    k = torch.randn(5, 4, 2, 64, generator=g).to(dtype).cuda()
    for t in (torch.int32, torch.int64):
        check(q, k, torch.tensor([0, 7, 296, 100, 13], dtype=t, device="cuda"), 64, 4)
    check(q, k, 296, 64, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_views_and_misaligned_rows(dtype):
    g = torch.Generator().manual_seed(6)
    both = torch.randn(2, 9, 3, 4, 64, generator=g).to(dtype).cuda()   # a fused projection's parts
    check(both[:, :, 0], both[:, :, 1], 0, 64, 7)
    heads_first = torch.randn(2, 4, 9, 64, generator=g).to(dtype).cuda().transpose(1, 2)
    check(heads_first, heads_first, 0, 64, 8)
    odd = torch.randn(2 * 9 * 4 * 64 + 1, generator=g).to(dtype).cuda()[1:].view(2, 9, 4, 64)
    check(odd, odd, 0, 64, 9)                                          # rows off the 16 bytes
    channels = torch.randn(2, 9, 4, 128, generator=g).to(dtype).cuda()[..., ::2]
    check(channels, channels, 0, 64, 10)
    one = torch.randn(2, 1, 1, 64, generator=g).to(dtype).cuda().expand(2, 9, 4, 64)
    check(one, one, 0, 64, 11)                                         # broadcast inputs


def test_more_tokens_than_the_backward_has_waves():
    g = torch.Generator().manual_seed(12)
    q = torch.randn(40, 250, 2, 32, generator=g).bfloat16().cuda()
    check(q, q, 0, 32, 13)


def test_more_tokens_than_a_launch_takes():
    from mathbrain.qk_norm import qk_norm_rotary
    n = (1 << 25) + 5
    cos, sin = (t.cuda() for t in tables(32, 1))
    w = torch.rand(32, device="cuda")
    q = torch.randn(n, 1, 1, 32, device="cuda", dtype=torch.bfloat16)
    got = qk_norm_rotary(q, q, w, w, cos, sin)
    for part in (slice(0, 9), slice(n - 9, n)):
        for x, y in zip(got, qk_norm_rotary(q[part], q[part], w, w, cos, sin)):
            assert torch.equal(x[part], y)


def test_zero_rows_and_empty_batches():
    from mathbrain.qk_norm import qk_norm_rotary
    cos, sin = (t.cuda() for t in tables(64, 16))
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.zeros(2, 3, 2, 64, device="cuda", requires_grad=True)
    q, k = qk_norm_rotary(x, x, w, w, cos, sin)
    dx, dw = torch.autograd.grad([q, k], [x, w], [torch.ones_like(q), torch.ones_like(k)])
    assert not q.any() and not k.any() and not dw.any() and torch.isfinite(dx).all()
    for shape in ((0, 3, 2, 64), (2, 0, 2, 64)):
        e = torch.zeros(shape, device="cuda", requires_grad=True)
        q, k = qk_norm_rotary(e, e, w, w, cos, sin)
        de, dw = torch.autograd.grad([q, k], [e, w], [torch.ones_like(q), torch.ones_like(k)])
        assert q.shape == shape and de.shape == shape and not dw.any()


def test_positions_outside_the_tables_give_nan_there_alone():
    from mathbrain.qk_norm import qk_norm_rotary
    cos, sin = (t.cuda() for t in tables(32, 8))
    w = torch.ones(32, device="cuda")
    x = torch.randn(4, 2, 3, 32, device="cuda")
    start = torch.tensor([0, 7, -1, 1 << 40], device="cuda")
    q, k = qk_norm_rotary(x, x, w, w, cos, sin, EPS, start)
    bad = torch.tensor([[0, 0], [0, 1], [1, 0], [1, 1]], dtype=torch.bool)
    for y in (q, k):
        assert torch.equal(torch.isnan(y).all(-1).all(-1).cpu(), bad)
        assert torch.equal(torch.isnan(y).any(-1).any(-1).cpu(), bad)


def test_same_bits_each_time_and_on_another_stream():
    from mathbrain.qk_norm import qk_norm_rotary
    cos, sin = (t.cuda() for t in tables(64, 512))
    q = torch.randn(8, 200, 8, 64, device="cuda").bfloat16().requires_grad_()
    k = torch.randn(8, 200, 8, 64, device="cuda").bfloat16().requires_grad_()
    w = torch.rand(64, device="cuda").requires_grad_()
    dy = torch.randn_like(q)

    def once():
        out = qk_norm_rotary(q, k, w, w, cos, sin)
        return [*out, *torch.autograd.grad(out, [q, k, w], [dy, dy])]
    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = once()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    from mathbrain.qk_norm import qk_norm_rotary
    cos, sin = (t.cuda() for t in tables(64, 64))
    q = torch.randn(4, 1, 8, 64, device="cuda").bfloat16()
    k = torch.randn(4, 1, 2, 64, device="cuda").bfloat16()
    w = torch.rand(64, device="cuda")
    start = torch.zeros(4, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        qk_norm_rotary(q, k, w, w, cos, sin, EPS, start)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qk_norm_rotary(q, k, w, w, cos, sin, EPS, start)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        start.fill_(i * 3)
        graph.replay()
        want = qk_norm_rotary(q, k, w, w, cos, sin, EPS, start)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_refusals():
    from mathbrain import _lib
    from mathbrain.qk_norm import qk_norm_rotary
    cos, sin = (t.cuda() for t in tables(64, 16))
    x = torch.randn(2, 4, 3, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    with pytest.raises(NotImplementedError):
        qk_norm_rotary(x.cpu(), x.cpu(), w.cpu(), w.cpu(), cos.cpu(), sin.cpu())
    for bad in (dict(q=x.half(), k=x.half()), dict(q=x.bfloat16()), dict(k=x[:, :2]), dict(k=x[0]),
                dict(q_weight=w[:32]), dict(cos=cos[:, :16]), dict(sin=sin[:8]), dict(cos=cos.double()),
                dict(cos=cos.t().contiguous().t()), dict(start=torch.zeros(3, dtype=torch.int32, device="cuda")),
                dict(start=torch.zeros(2, device="cuda"))):
        args = dict(q=x, k=x, q_weight=w, k_weight=w, cos=cos, sin=sin) | bad
        with pytest.raises(ValueError, match="qk_norm_rotary"):
            qk_norm_rotary(**args)
    for start in (-1, 13):
        with pytest.raises(_lib.HipKernelError, match="pass the table"):
            qk_norm_rotary(x, x, w, w, cos, sin, EPS, start)
    x48 = torch.randn(2, 4, 3, 48, device="cuda")
    c48, s48 = (t.cuda() for t in tables(48, 16))
    with pytest.raises(_lib.HipKernelError, match="head_dim=48"):
        qk_norm_rotary(x48, x48, w[:48], w[:48], c48, s48)


def test_differences_agree_with_the_gradient():
    """Central differences of sum(out * dy) in float32 along a random direction: the step's error is
    h^2 of the third derivative and 2^-24 of the sum's size over h; with h = 1e-2 and 384 terms of
    size about 1 both stay under 1e-3 of the directional derivative's scale (its norm, about 20)."""
    from mathbrain.qk_norm import qk_norm_rotary
    cos, sin = (t.cuda() for t in tables(32, 16))
    g = torch.Generator().manual_seed(20)
    q, k, w, u, dy, dq, dk = (torch.randn(s, generator=g).cuda() for s in
                              ((2, 3, 2, 32), (2, 3, 2, 32), (32,), (32,), (2, 3, 2, 32), (2, 3, 2, 32), (2, 3, 2, 32)))
    leaves = [t.requires_grad_() for t in (q, k, w)]

    def value(q, k, w):
        a, b = qk_norm_rotary(q, k, w, u, cos, sin)
        return (a.double() * dy.double()).sum() + (b.double() * dy.double()).sum()
    grads = torch.autograd.grad(value(*leaves), leaves)
    dw = torch.randn(32, generator=g).cuda()
    h = 1e-2
    with torch.no_grad():
        diff = (value(q + h * dq, k + h * dk, w + h * dw) - value(q - h * dq, k - h * dk, w - h * dw)) / (2 * h)
    along = sum((a.double() * b.double()).sum() for a, b in zip(grads, (dq, dk, dw)))
    assert abs(float(diff - along)) < 2e-2, (float(diff), float(along))


def test_forward_mode_derivatives_are_refused():
    """A dual tensor asks for a tangent without requiring a gradient; an output without one would be
    a derivative of zero."""
    import torch.autograd.forward_ad as fw
    from mathbrain.qk_norm import qk_norm_rotary
    cos, sin = (t.cuda() for t in tables(32, 8))
    w = torch.rand(32, device="cuda")
    x = torch.randn(2, 3, 2, 32, device="cuda")
    want = qk_norm_rotary(x, x, w, w, cos, sin)
    with fw.dual_level():
        for i in range(4):
            args = [x, x, w, w]
            args[i] = fw.make_dual(args[i].clone(), torch.ones_like(args[i]))
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(NotImplementedError, match="jvp"):
                    qk_norm_rotary(*args, cos, sin)
        assert all(torch.equal(a, b) for a, b in zip(qk_norm_rotary(x, x, w, w, cos, sin), want))


def test_tables_that_require_a_gradient_are_refused():
    """They would get none."""
    from mathbrain.qk_norm import qk_norm_rotary
    cos, sin = (t.cuda() for t in tables(32, 8))
    w = torch.rand(32, device="cuda", requires_grad=True)
    x = torch.randn(2, 3, 2, 32, device="cuda")
    want = qk_norm_rotary(x, x, w, w, cos, sin)
    for c, s in ((cos.clone().requires_grad_(), sin), (cos, sin.clone().requires_grad_())):
        for weight in (w, w.detach()):
            with pytest.raises(ValueError, match="get no gradient"):
                qk_norm_rotary(x, x, weight, weight, c, s)
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(qk_norm_rotary(x, x, w, w, c, s), want))
