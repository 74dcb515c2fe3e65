"""linear_cross_entropy in fp32, row by row: words that are improbable in every row, and rows of hidden or of the weights
beside one of another size, keep the digits that fp32 operations would keep.

Tolerances, to first order, for each row and word by itself.  A score of D products of values with 24 bits (two planes: 2^-23 of
each factor and 2^-24 of the product left out) summed in fp32 is off by e = (2 sqrt(D) + 8) 2^-24 |h_n| |w_v| (the roundings of
the sum are independent), and by 2^-23 of itself and of the row's maximum in units of log 2.  A probability moves by
p_v [(1 - p_v) e_v + sum of the others' p e], and by 2^-22 of itself; U = p - [v = t] by 2^-24 more at the target.  The
sums' operands are off by 2^-22 of each term, their fp32 sum of K terms by sqrt(K) 2^-24 of the absolute sum, the result by 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
IGN = -100


def expected(h, w, target, g, spread=None):
    """loss, dh, dw of sum_n g_n loss_n in 64 bits, and how far each row of them may be off, with scores off by `spread`
    (2 sqrt(D) + 8) of 2^-24 |h_n| |w_v|."""
    h, w, g = h.double(), w.double(), g.double()
    N, D = h.shape
    use = target != IGN
    t = torch.where(use, target, 0)
    s = h @ w.t()
    p = torch.softmax(s, 1)
    lse = torch.logsumexp(s, 1, keepdim=True)
    loss = torch.where(use, (lse - s.gather(1, t[:, None]))[:, 0], 0.0)
    e = (spread or 2 * math.sqrt(D) + 8) * 2.0**-24 * h.norm(dim=1)[:, None] * w.norm(dim=1) + 2.0**-23 * (s.abs() + lse.abs())
    pe = (p * e).sum(1, keepdim=True)
    onehot = torch.nn.functional.one_hot(t, w.shape[0])
    pt, et = p.gather(1, t[:, None]), e.gather(1, t[:, None])
    room = (pe - pt * et + (1 - pt) * et)[:, 0]          # of d loss = sum_v p_v ds_v - ds_t
    loss_room = torch.where(use, room + 2.0**-22 * (loss + 1), 0.0)
    du = p * ((1 - p) * e + (pe - p * e)) + 2.0**-22 * p + 2.0**-23 * onehot
    gg = torch.where(use, g, 0.0)[:, None]
    u, du = (p - onehot) * gg, du * gg.abs()
    each = lambda k: 2.0**-22 + math.sqrt(k) * 2.0**-24
    hn, wn = h.norm(dim=1, keepdim=True), w.norm(dim=1, keepdim=True)
    dh, dw = u @ w, u.t() @ h
    dh_room = (du @ wn + each(w.shape[0]) * (u.abs() @ wn))[:, 0] + 2.0**-24 * dh.norm(dim=1)
    dw_room = (du.t() @ hn + each(N) * (u.abs().t() @ hn))[:, 0] + 2.0**-24 * dw.norm(dim=1)
    return loss, dh, dw, loss_room, dh_room, dw_room


def check(h, w, target, g, what=""):
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
    each = linear_cross_entropy(a, b, target, IGN, "none")
    got = torch.autograd.grad(each, [a, b], g)
    loss, dh, dw, loss_room, dh_room, dw_room = expected(h, w, target, g)
    tiny = 1e-37          # below fp32's normal numbers digits are lost to everybody
    off = ((each.detach().double() - loss).abs() / (loss_room + tiny)).max()
    off_h = ((got[0].double() - dh).norm(dim=1) / (dh_room + tiny)).max()
    off_w = ((got[1].double() - dw).norm(dim=1) / (dw_room + tiny)).max()
    assert off <= 1 and off_h <= 1 and off_w <= 1, (what, float(off), float(off_h), float(off_w))
    return got


def make(N, V, D, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + N + V + D)
    w = torch.randn(V, D, generator=g, device="cuda") / math.sqrt(D)
    target = torch.randint(0, V, (N,), generator=g, device="cuda")
    h = torch.randn(N, D, generator=g, device="cuda") + 5 * torch.rand(N, 1, generator=g, device="cuda") * w[target]
    return h, w, target, 0.2 + torch.rand(N, generator=g, device="cuda")


ROWS = [5, 16, 40, 64, 200, 1300]      # each of the ways through the kernels


@pytest.mark.parametrize("N", ROWS)
def test_improbable_words(N):
    """Words whose scores lie 8 to 60 below the others in every row: their rows of dweight, from 1e-4 to 1e-26 of the others'."""
    h, w, target, g = make(N, 700, 64)
    h[:, 0] = 8.0
    far = torch.arange(700, device="cuda") % 3 == 1
    w[far, 0] = -torch.linspace(1.0, 7.5, int(far.sum()), device="cuda")
    target = torch.where(far[target], target - target % 3, target)
    _, dw = check(h, w, target, g)
    size = dw.double().norm(dim=1)
    assert size[far].min() < 1e-24 * size.max() and size[far].min() > 0


@pytest.mark.parametrize("N", ROWS)
@pytest.mark.parametrize("up", [2.0**24, 2.0**-24, 2.0**40])
def test_a_row_of_another_size(N, up):
    h, w, target, g = make(N, 700, 64, seed=1)
    h[3] *= up
    check(h, w, target, g)


@pytest.mark.parametrize("N", ROWS)
@pytest.mark.parametrize("up", [2.0**24, 2.0**-24, 2.0**40])
def test_a_word_of_another_size(N, up):
    h, w, target, g = make(N, 700, 64, seed=2)
    w[11] *= up
    target[target == 11] = 12
    check(h, w, target, g)


@pytest.mark.parametrize("N", ROWS)
def test_gradients_of_another_size(N):
    """Rows whose losses' gradients are far apart: each word's row is as exact as its largest term allows."""
    h, w, target, g = make(N, 700, 64, seed=3)
    g[0] *= 2.0**30
    g[1] *= 2.0**-60
    g[2] = 0.0
    got = check(h, w, target, g)
    assert not got[0][2].any()
    g *= 2.0**-40             # a row without a gradient says nothing about the others' size
    g[:2] = 0.0
    check(h, w, target, g)


@pytest.mark.parametrize("N", ROWS)
@pytest.mark.parametrize("a,b,c", [(2.0**80, 2.0**-80, 1.0), (2.0**-80, 2.0**80, 1.0), (1.0, 1.0, 2.0**90), (1.0, 1.0, 2.0**-90)])
def test_very_large_and_small_values(N, a, b, c):
    h, w, target, g = make(N, 700, 64, seed=4)
    check(h * a, w * b, target, g * c, (a, b, c))


def test_many_blocks_of_both_sums():
    """More blocks of the vocabulary and of the rows than wait in LDS at a time, and several pieces of the vocabulary."""
    h, w, target, g = make(17000, 2600, 32, seed=5)
    target[::5] = IGN
    check(h, w, target, g)
    h, w, target, g = make(70, 70001, 32, seed=6)
    check(h, w, target, g)
    h, w, target, g = make(6000, 15001, 32, seed=7)
    check(h, w, target, g)


@pytest.mark.parametrize("N,V,D", [(17000, 8000, 2048), (4000, 20000, 2048)])
def test_long_runs_of_blocks_of_different_sizes(N, V, D):
    """Sums over rows (or words) that one workgroup takes from end to end, so that the exponents in LDS are replaced on the way (after 64
    blocks of 128), of blocks whose terms lie up to 2^150 apart."""
    h, w, target, g = make(N, V, D, seed=8)
    at = torch.arange(N, device="cuda") // 128
    g *= torch.exp2(((at * 37) % 25 - 12).float() * 6)
    words = torch.arange(V, device="cuda") // 128
    h[:, 0] = 8.0
    w[:, 0] -= ((words * 29) % 11).float() * 0.5
    check(h, w, target, g)
