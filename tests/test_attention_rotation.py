"""baseline.CausalSelfAttention where the rotation's kernel does not apply: on the CPU, under torch.func, with tables that want
a gradient or that are broadcast.  The rotation is ``rotate``'s tensor operations there."""
import math

import pytest
import torch


def module(D=32, heads=2, **options):
    from mathbrain.baseline import CausalSelfAttention
    torch.manual_seed(0)
    return CausalSelfAttention(D, heads, **options)


def definition(m, x, cos, sin):
    """In float64, with the rotation by complex numbers."""
    B, L, D = x.shape
    q, k, v = ((x.double() @ w.weight.double().T).view(B, L, m.n_heads, m.head_dim).transpose(1, 2) for w in (m.wq, m.wk, m.wv))
    spin = torch.complex(cos.double(), sin.double())
    turn = lambda t: torch.view_as_real(torch.view_as_complex(t.unflatten(-1, (-1, 2)).contiguous()) * spin).flatten(-2)
    s = turn(q) @ turn(k).transpose(-1, -2) / math.sqrt(m.head_dim)
    s = s.masked_fill(torch.ones(L, L, dtype=torch.bool, device=x.device).triu(1), -math.inf)
    return (s.softmax(-1) @ v).transpose(1, 2).reshape(B, L, D) @ m.wo.weight.double().T


def run_everywhere(dev):
    from mathbrain.baseline import rotary_tables
    m = module().to(dev)
    x = torch.randn(3, 7, 32, device=dev)
    cos, sin = (t.to(dev) for t in rotary_tables(16, 7))
    want = definition(m, x, cos, sin)
    near = lambda a, b: float((a.double() - b).abs().max()) < 1e-5 * float(b.abs().max())   # 32 products and sums of 2^-24 each, five in a row
    assert near(m(x, cos, sin), want)
    # each row by itself under vmap, and gradients of each row
    assert near(torch.func.vmap(lambda r: m(r[None], cos, sin)[0])(x), want)
    f = lambda r: m(r[None], cos, sin).square().sum()
    each = torch.func.vmap(torch.func.grad(f))(x)
    y = x.clone().requires_grad_()
    whole, = torch.autograd.grad(m(y, cos, sin).square().sum(), y)
    assert float((each - whole).abs().max()) < 1e-4 * float(whole.abs().max())
    # tables with gradients
    c, s = cos.clone().requires_grad_(), sin.clone().requires_grad_()
    gc, gs = torch.autograd.grad(m(x, c, s).square().sum(), [c, s])
    c64, s64 = cos.double().requires_grad_(), sin.double().requires_grad_()
    wc, ws = torch.autograd.grad(definition(m, x, c64, s64).square().sum(), [c64, s64])
    assert float((gc - wc).abs().max()) < 1e-4 * float(wc.abs().max()) and float((gs - ws).abs().max()) < 1e-4 * float(ws.abs().max())
    # one row of angles for all positions; tables in 64 bits; strided ones
    assert near(m(x, cos[3:4], sin[3:4]), definition(m, x, cos[3:4], sin[3:4]))
    assert near(m(x, cos.double(), sin.double()), want)
    wide = torch.stack((cos, sin), -1)
    assert near(m(x, wide[..., 0], wide[..., 1]), want)
    with pytest.raises(RuntimeError):                      # more positions than the tables have
        m(x, cos[:5], sin[:5])


def test_on_the_cpu():
    run_everywhere("cpu")


@pytest.mark.gpu
def test_on_the_gpu():
    run_everywhere("cuda")


def test_options_of_the_kernel_are_refused_elsewhere():
    from mathbrain.rotary import rotary_tables
    x = torch.randn(1, 4, 32)
    for m, d in ((module(rope_layout="half"), 16), (module(), 8)):
        with pytest.raises(ValueError, match="rope_layout and rope_dims"):
            m(x, *rotary_tables(d, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, dict(rope_layout="half")])
@pytest.mark.parametrize("strict", [True, False])
def test_exported(options, strict):
    """An exported attention holds the rotation's op and gives the eager results."""
    from mathbrain.baseline import rotary_tables
    m = module(**options).cuda().eval()
    x = torch.randn(2, 6, 32, device="cuda")
    args = (x, *(t.cuda() for t in rotary_tables(16, 6)))
    with torch.no_grad():
        program = torch.export.export(m, args, strict=strict)
        assert any("apply_rotary" in str(n.target) for n in program.graph.nodes)
        assert torch.equal(program.module()(*args), m(*args))
