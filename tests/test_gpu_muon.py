"""orthogonalize, muon_step and Muon (mathbrain/muon.py) against their definition in 64 bits.

Tolerances.  Two planes round a value by 2^-23, a product's fp32 sums by a few 2^-24 of it; an iteration multiplies an
error of X by at most the polynomial's steepest slope, below 4 (3.4445 at 0, 3.9 at 1.2).  Five steps leave at most
4^5 of the first one's error and as much again of the later ones' together: 2 * 4^steps * 4 * 2^-23 of max(1, |X|) in the
Frobenius norm (|X| is 1 at first), to which the result's own rounding adds half a step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
COEF = (3.4445, -4.7750, 2.0315)


def definition(g, steps=5, coef=COEF, eps=1e-7):
    x = g.double()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (x.norm() + eps)
    a, b, c = coef
    for _ in range(steps):
        y = x @ x.t()
        x = a * x + (b * y + c * y @ y) @ x
    return x.t() if flip else x


def half_step(t):
    return {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}[t]


def check(got, want, steps=5, what=""):
    size = float(want.norm())
    room = 2 * 4.0**steps * 4 * 2.0**-23 * max(1.0, size) + half_step(got.dtype) * size
    assert got.shape == want.shape and got.is_contiguous(), what
    assert float((got.double() - want).norm()) <= room, (what, float((got.double() - want).norm()), room)


SHAPES = [(1, 1), (1, 7), (9, 1), (8, 8), (31, 33), (64, 64), (128, 128), (129, 65), (100, 300), (257, 130), (512, 64), (96, 1500),
          (700, 513)]


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_all_shapes_together_and_alone(t):
    from mathbrain.muon import orthogonalize
    g = torch.Generator("cuda").manual_seed(3)
    mats = [(torch.randn(s, generator=g, device="cuda") * 10.0**(i % 5 - 2)).to(t) for i, s in enumerate(SHAPES)]
    got = orthogonalize(mats)
    assert all(x.dtype == t for x in got)
    for x, y in zip(got, mats):
        check(x, definition(y), what=tuple(y.shape))
        check(orthogonalize([y])[0], definition(y), what=tuple(y.shape))       # small ones alone have a kernel of their own
    for x, y in zip(orthogonalize(mats, dtype=torch.float32), mats):
        check(x, definition(y), what=tuple(y.shape))


def test_spectra():
    from mathbrain.muon import orthogonalize
    g = torch.Generator("cuda").manual_seed(4)
    u = torch.linalg.qr(torch.randn(160, 160, generator=g, device="cuda", dtype=torch.float64))[0]
    v = torch.linalg.qr(torch.randn(200, 160, generator=g, device="cuda", dtype=torch.float64))[0].t()
    for s in (torch.ones(160), 2.0**-torch.linspace(0, 20, 160), torch.cat((torch.ones(1), torch.zeros(159))),
              torch.cat((torch.full((80,), 1e-4), torch.ones(80)))):
        x = ((u * s.cuda().double()) @ v).float()
        check(orthogonalize(x), definition(x), what=s[:3])
    x = (u * torch.linspace(0.5, 1, 160, device="cuda", dtype=torch.float64)).float()   # well conditioned: all near 1
    s = torch.linalg.svdvals(orthogonalize(x).double())
    assert s.min() > 0.6 and s.max() < 1.25


@pytest.mark.parametrize("steps,coef", [(1, COEF), (2, (1.5, -0.5, 0.0)), (8, (1.875, -1.25, 0.375)), (3, (2.0, 0.0, 0.0)), (30, (1.5, -0.5, 0.0))])
def test_steps_and_coefficients(steps, coef):
    from mathbrain.muon import orthogonalize
    x = torch.randn(70, 100, device="cuda")
    want = definition(x, steps, coef)
    # slopes: at most a; 1.5^30 would be of no use, but singular values near 1 have slope 0 and the rest have grown to there
    check(orthogonalize(x, steps=steps, coefficients=coef), want, min(steps, 6))


def test_sizes_from_tiny_to_huge_and_zeros():
    from mathbrain.muon import orthogonalize
    x = torch.randn(40, 50, device="cuda")
    for scale in (1e-36, 1e-20, 1e20, 1e36):
        check(orthogonalize(x * scale, eps=0.0), definition(x * scale, eps=0.0), what=scale)
        check(orthogonalize((x * scale).bfloat16(), eps=0.0), definition((x * scale).bfloat16(), eps=0.0), what=scale)
    check(orthogonalize(x * 1e-8), definition(x * 1e-8))                    # eps counts
    assert not orthogonalize(torch.zeros(5, 9, device="cuda")).any()
    for bad in (math.nan, math.inf):
        y = x.clone()
        y[3, 4] = bad
        a, b = orthogonalize([y, x])
        assert a.isnan().all()
        check(b, definition(x))


def test_forms_of_the_input():
    from mathbrain.muon import orthogonalize
    x = torch.randn(3, 2, 40, 70, device="cuda")
    got = orthogonalize(x)
    assert got.shape == x.shape
    for i in range(3):
        for j in range(2):
            check(got[i, j], definition(x[i, j]))
    view = torch.randn(80, 90, device="cuda")[::2, 3:60]
    assert torch.equal(orthogonalize(view), orthogonalize(view.contiguous()))
    assert torch.equal(orthogonalize(view.t()), orthogonalize(view.t().contiguous()))
    assert orthogonalize([]) == [] and orthogonalize(x[:, :0]).shape == (3, 0, 40, 70) and orthogonalize(x[..., :0]).shape == (3, 2, 40, 0)
    a, b, c = orthogonalize([x[0, 0], torch.empty(0, 5, device="cuda"), x[0, 1]])     # (all of them small)
    assert b.shape == (0, 5) and torch.equal(a, got[0, 0]) and torch.equal(c, got[0, 1])
    assert torch.equal(orthogonalize([x[0, 0], x[0, 0]])[1], got[0, 0])      # the same tensor twice is read twice
    w = torch.nn.Parameter(x[0, 0])
    assert not orthogonalize(w).requires_grad
    mixed = orthogonalize([x[0, 0], x[0, 1].bfloat16()])
    assert mixed[0].dtype == torch.float32 and mixed[1].dtype == torch.bfloat16


def test_small_matrices_alone():
    """Up to what a CU's LDS holds, and just beyond: rows, columns, both ways round, every type, steps and decay."""
    from mathbrain.muon import muon_step, orthogonalize
    g = torch.Generator("cuda").manual_seed(8)
    for shape in ((1, 1), (64, 64), (65, 64), (128, 128), (128, 192), (192, 128), (128, 193), (64, 570), (570, 64), (64, 577), (1, 570),
                  (33, 300), (129, 5), (100, 190), (17, 63)):
        for t in (torch.float32, torch.bfloat16):
            x = (torch.randn(shape, generator=g, device="cuda") * 3).to(t)
            check(orthogonalize(x), definition(x), what=shape)
            check(orthogonalize(x, steps=2), definition(x, 2), 2, what=shape)
            p, m = torch.zeros_like(x), torch.randn(shape, generator=g, device="cuda").to(t)
            want_m = 0.9 * m.double() + x.double()
            muon_step([p], [x], [m], 1.0, momentum=0.9, nesterov=False)
            check(-p / math.sqrt(max(1.0, shape[0] / shape[1])), definition(want_m), what=shape)
            assert ((m.double() - want_m).abs() <= half_step(t) * want_m.abs() + 2.0**-22 * (want_m.abs() + 30)).all()


def test_many_matrices():
    """More than one launch's arguments hold, and more than a wave looks through at once."""
    from mathbrain.muon import orthogonalize
    g = torch.Generator("cuda").manual_seed(5)
    mats = [torch.randn(1 + i % 37, 1 + (7 * i) % 41, generator=g, device="cuda") for i in range(150)]
    for x, y in zip(orthogonalize(mats), mats):
        check(x, definition(y), what=tuple(y.shape))


def test_tall_long_and_large():
    from mathbrain.muon import orthogonalize
    for shape in ((20000, 48), (48, 20000), (2100, 1030)):
        x = torch.randn(shape, device="cuda")
        check(orthogonalize(x), definition(x), what=shape)


def step_definition(p, g, m, lr, mu, nesterov, decay):
    m = mu * m.double() + g.double()
    u = g.double() + mu * m if nesterov else m
    scale = math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
    return p.double() * (1 - lr * decay) - lr * scale * definition(u), m


@pytest.mark.parametrize("tp,tg,tm", [(torch.float32,) * 3, (torch.bfloat16,) * 3, (torch.bfloat16, torch.bfloat16, torch.float32),
                                      (torch.float32, torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_step(tp, tg, tm, nesterov):
    from mathbrain.muon import muon_step
    g = torch.Generator("cuda").manual_seed(6)
    shapes = [(64, 64), (130, 33), (33, 130), (1, 5), (256, 100)]
    make = lambda t: [torch.randn(s, generator=g, device="cuda").to(t) for s in shapes]
    params, grads, momenta = make(tp), make(tg), make(tm)
    keep = [g.clone() for g in grads]
    for _ in range(3):
        want = [step_definition(p, x, m, 0.1, 0.9, nesterov, 0.2) for p, x, m in zip(params, grads, momenta)]
        versions = [p._version for p in params]
        muon_step(params, grads, momenta, 0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.2)
        assert all(p._version > v for p, v in zip(params, versions))
        for p, m, (p_, m_) in zip(params, momenta, want):
            assert ((m.double() - m_).abs() <= half_step(tm) * m_.abs() + 4 * 2.0**-24 * (m_.abs() + 4)).all()
            # the update's own room (as above), and the sums' rounding
            scale = math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
            size = max(1.0, math.sqrt(min(p.shape)) * 1.25)
            room = 0.1 * scale * 2 * 4.0**5 * 4 * 2.0**-23 * size + (half_step(tp) + 2.0**-22) * float(p_.norm() + 0.1 * scale * size)
            assert float((p.double() - p_).norm()) <= room
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))


def test_optimizer():
    from mathbrain.muon import Muon, muon_step
    torch.manual_seed(0)
    ws = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((30, 40), (70, 20), (5, 5))]
    twins = [w.detach().clone() for w in ws]
    momenta = [torch.zeros_like(w) for w in twins]
    opt = Muon([dict(params=ws[:2]), dict(params=ws[2:], lr=0.3)], lr=0.05, weight_decay=0.1)
    for i in range(3):
        opt.zero_grad()
        x = torch.randn(8, 30, device="cuda")
        ((x @ ws[0]).square().sum() + (ws[1] ** 3).sum() + (ws[2].sum() if i != 1 else 0)).backward()
        for sel, lr in (((0, 1), 0.05), ((2,), 0.3)):
            sel = [j for j in sel if ws[j].grad is not None]
            muon_step([twins[j] for j in sel], [ws[j].grad for j in sel], [momenta[j] for j in sel], lr, weight_decay=0.1)
        opt.step()
        assert all(torch.equal(a.detach(), b) for a, b in zip(ws, twins))
    again = Muon([dict(params=ws[:2]), dict(params=ws[2:])])
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[ws[0]]["momentum_buffer"], momenta[0]) and again.param_groups[1]["lr"] == 0.3
    assert opt.step(lambda: 7.0) == 7.0
    with pytest.raises(ValueError, match="not a matrix"):
        Muon([torch.nn.Parameter(torch.zeros(3, device="cuda"))])


def test_captured_and_on_another_stream():
    from mathbrain.muon import muon_step, orthogonalize
    x = [torch.randn(s, device="cuda") for s in ((40, 70), (130, 129))]
    want = orthogonalize(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = orthogonalize(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, there))
    p, m = [torch.randn_like(y) for y in x], [torch.zeros_like(y) for y in x]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step(p, x, m, 0.1)
    for _ in range(3):
        [y.mul_(1.3).add_(0.1) for y in x]
        twin_p, twin_m = [y.clone() for y in p], [y.clone() for y in m]
        graph.replay()
        torch.cuda.synchronize()
        muon_step(twin_p, x, twin_m, 0.1)
        assert all(torch.equal(a, b) for a, b in zip(p + m, twin_p + twin_m))


def test_refusals():
    import torch.autograd.forward_ad as fwad
    from mathbrain import _lib
    from mathbrain.muon import muon_step, orthogonalize
    x = torch.randn(20, 30, device="cuda")
    for bad in (x.half(), x[0], [x, x[0]], x.to_sparse()):
        with pytest.raises(ValueError):
            orthogonalize(bad)
    for kw in (dict(steps=0), dict(steps=101), dict(coefficients=(1, 2)), dict(coefficients=(100.0, 0.0, 0.0)), dict(eps=-1.0),
               dict(dtype=torch.half), dict(coefficients=(math.nan, 0, 0))):
        with pytest.raises(ValueError):
            orthogonalize(x, **kw)
    with pytest.raises(NotImplementedError):
        orthogonalize([x, x.cpu()])
    with pytest.raises(NotImplementedError):
        orthogonalize(x.cpu())
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        orthogonalize(fwad.make_dual(x, x))
    y, z, keep = torch.randn_like(x), torch.randn_like(x), x.clone()
    for p, g, m, err in (([x], [y], [], ValueError), ([x], [y.t()], [z], ValueError), ([x.t()], [y.t()], [z.t()], ValueError),
                         ([x, x], [y, y], [z, torch.zeros_like(z)], _lib.HipKernelError), ([x], [y], [x], _lib.HipKernelError),
                         ([x], [x], [z], _lib.HipKernelError), ([x], [y], [y], _lib.HipKernelError)):
        with pytest.raises(err):
            muon_step(p, g, m, 0.1)
    with pytest.raises(ValueError):
        muon_step([x], [y], [z], math.nan)
    assert torch.equal(x, keep)
    muon_step([], [], [], 0.1)


@pytest.mark.parametrize("shapes", [[(4096, 1024)], [(640, 4000)], [(48, 20000)], [(129, 1300)], [(130, 1023), (1023, 130)],
                                    [(300, 2500), (65, 66), (200, 1), (640, 700)], [(1400, 1400)]])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_few_matrices_with_long_sums(shapes, t):
    """Few matrices, whose first products are shared out along their sums; with short matrices among them, which have fewer
    steps than there are shares; the same twice; and a step of the optimiser."""
    from mathbrain.muon import muon_step, orthogonalize
    g = torch.Generator("cuda").manual_seed(11)
    mats = [torch.randn(s, generator=g, device="cuda").to(t) for s in shapes]
    got, again = orthogonalize(mats), orthogonalize(mats)
    for x, y, z in zip(got, mats, again):
        check(x, definition(y), what=tuple(y.shape))
        assert torch.equal(x, z)
    params, momenta = [torch.zeros_like(x) for x in mats], [torch.zeros_like(x) for x in mats]
    muon_step(params, mats, momenta, 1.0, momentum=0.9, nesterov=False)
    for p, x in zip(params, mats):
        check(-p / math.sqrt(max(1.0, x.shape[0] / x.shape[1])), definition(x), what=tuple(x.shape))


def test_few_long_matrices_captured():
    from mathbrain.muon import orthogonalize
    x = torch.randn(300, 2500, device="cuda")
    orthogonalize(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = orthogonalize(x)
    for i in range(3):
        x.copy_(torch.randn(300, 2500, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, orthogonalize(x))
