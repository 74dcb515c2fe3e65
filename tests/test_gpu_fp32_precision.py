"""The digits of the fp32 paths that hold values as two fp16 planes: the cross entropy and the orthogonalised matrices, to bounds that
a single plane anywhere does not meet (which the tests here without a GPU show).

Cross entropy.  For random rows a partial sum of a score is about |h| |w| / sqrt(D) times sqrt(k / D), so D roundings of 2^-25 of them
are 2^-25 |h| |w| / sqrt(2) together, and the planes' (2^-23 of each factor) less: 8 2^-24 |h| |w| is over ten of that.  A single plane's
2^-12 of each product is 2^-12 sqrt(2 / D) |h| |w|: 60 to 15 times the bound at D = 512 to 2048 for the largest of the scores.

Orthogonalised matrices.  A step's roundings are a few 2^-24 of |X|, and the polynomial multiplies what lies in small directions by
3.4445 a step, as it does those directions themselves: from |X| = 1 at first to the end 3.4445^5 = 485.  Four sources in five steps, sqrt(20) of
them if independent: 4 * 485 * 2^-24 in the Frobenius norm, whatever the result's."""
import math

import pytest
import torch

SIZES = [(64, 5000, 512), (128, 127, 2048), (8, 515, 1024), (17, 131, 2048), (2, 259, 2047), (200, 3000, 1024), (1500, 2000, 512)]
SHAPES = [(64, 64), (128, 128), (129, 65), (100, 300), (512, 64), (96, 1500), (700, 513), (640, 1400)]
COEF = (3.4445, -4.7750, 2.0315)


def make(N, V, D, dev):
    g = torch.Generator(dev).manual_seed(N + V + D)
    w = torch.randn(V, D, generator=g, device=dev) / math.sqrt(D)
    target = torch.randint(0, V, (N,), generator=g, device=dev)
    h = torch.randn(N, D, generator=g, device=dev) + 4 * torch.rand(N, 1, generator=g, device=dev) * w[target]
    return h, w, target, 0.2 + torch.rand(N, generator=g, device=dev)


def loss_and_rooms(h, w, target, g):
    from test_gpu_linear_ce_ranges import expected
    return expected(h, w, target, g, spread=8.0)


def off(got, want, room):
    d = (got.double() - want).abs() if want.dim() == 1 else (got.double() - want).norm(dim=1)
    return float((d / room).max())


def one_plane(x):
    """Rows scaled to a largest value of 2^14 .. 2^15, rounded to fp16."""
    x = x.double()
    s = torch.exp2(14 - torch.floor(torch.log2(x.abs().amax(1, keepdim=True).clamp(min=1e-300))))
    return (x * s).half().double() / s


@pytest.mark.parametrize("N,V,D", SIZES)
def test_a_single_plane_would_show_in_the_loss(N, V, D):
    h, w, target, g = make(N, V, D, "cpu")
    loss, dh, dw, loss_room, dh_room, dw_room = loss_and_rooms(h, w, target, g)
    for a, b in ((one_plane(h), w.double()), (h.double(), one_plane(w))):
        s = a @ b.t()
        # (a few rows' errors may be small by chance; the scores of all words count in the gradients)
        p = torch.softmax(s, 1)
        u = (p - torch.nn.functional.one_hot(target, V)) * g.double()[:, None]
        seen = [off(torch.logsumexp(s, 1) - s.gather(1, target[:, None])[:, 0], loss, loss_room), off(u @ w.double(), dh, dh_room),
                off(u.t() @ h.double(), dw, dw_room)]
        assert max(seen) > 2, seen
    p = torch.softmax(h.double() @ w.double().t(), 1)
    u = (p - torch.nn.functional.one_hot(target, V)) * g.double()[:, None]
    assert off(one_plane(u) @ w.double(), dh, dh_room) > 2 and off(u @ one_plane(w), dh, dh_room) > 2
    assert off(one_plane(u.t()) @ h.double(), dw, dw_room) > 2 and off(u.t() @ one_plane(h), dw, dw_room) > 2


@pytest.mark.gpu
@pytest.mark.parametrize("N,V,D", SIZES)
def test_loss_and_gradients(N, V, D):
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    h, w, target, g = make(N, V, D, "cuda")
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    each = linear_cross_entropy(a, b, target, reduction="none")
    da, db = torch.autograd.grad(each, [a, b], g)
    loss, dh, dw, loss_room, dh_room, dw_room = loss_and_rooms(h, w, target, g)
    seen = off(each.detach(), loss, loss_room), off(da, dh, dh_room), off(db, dw, dw_room)
    assert max(seen) <= 1, seen


def orthogonal(g, plain=lambda what: False):
    """The definition in 64 bits; plain(what) takes the operands of a product, in every step, from single planes."""
    x = g.double()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (x.norm() + 1e-7)
    a, b, c = COEF

    def product(y, z, what):
        if plain(what):
            y, z = ((t * 2.0**14).half().double() / 2.0**14 for t in (y, z))
        return y @ z

    for _ in range(5):
        y = product(x, x.t(), "A")
        second = b * y + c * product(y, y, "B")
        x = a * x + product(second, x, "X")
    return x.t() if flip else x


ROOM = 4 * 3.4445**5 * 2.0**-24


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("what", ["A", "B", "X"])
def test_a_single_plane_would_show_in_any_product(shape, what):
    g = torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape)))
    want = orthogonal(g)
    got = orthogonal(g, lambda w: w == what)
    assert float((got - want).norm()) > 10 * ROOM, float((got - want).norm()) / ROOM


@pytest.mark.gpu
@pytest.mark.parametrize("together", [False, True])
def test_orthogonalize(together):
    from mathbrain.muon import orthogonalize
    mats = [torch.randn(s, generator=torch.Generator("cuda").manual_seed(sum(s)), device="cuda") for s in SHAPES]
    got = orthogonalize(mats) if together else [orthogonalize(x) for x in mats]
    for x, y in zip(got, mats):
        want = orthogonal(y)
        assert float((x.double() - want).norm()) <= ROOM + 2.0**-24 * float(want.norm()), (tuple(y.shape), float((x.double() - want).norm()) / ROOM)
