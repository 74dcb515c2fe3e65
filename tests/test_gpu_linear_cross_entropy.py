"""linear_cross_entropy (mathbrain/linear_cross_entropy.py) against its definition in 64 bits.

Tolerances.  A score of D products accumulated in fp32 is off by at most e = (D + 4) 2^-24 |h|.|w| (fp32 operands as two
planes add 2^-22 |h|.|w|), in units of log 2 by another 2 * 2^-24 of itself; a loss by 2 e and the rounding of its own
parts, a few 2^-24 of |max| + log V.  A probability p is off by the relative 2 e and by 2^-22 of its exponent's rounding:
that is an error of p (2 e + ...) in U = p - [v = t], however near to 0 U is at a confident row's target (as in the
difference of an fp32 softmax and 1), so it counts on the products with p, not with |U|.  U's plane rounds by 2^-12 relative in bf16's case (fp16) and 2^-23 in fp32's, never by more than 2^-40 absolutely; the
sums over K add sqrt(K) 2^-24 of the absolute sum (their roundings are independent; in the norm of the whole result),
and the output's rounding is half a step: 2^-8 (bf16), 2^-24 (fp32)."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
IGN = -100


def make(N, V, D, t, seed=0, lean=6.0):
    g = torch.Generator("cuda").manual_seed(seed * 7919 + N + V + D)
    w = torch.randn(V, D, generator=g, device="cuda") / math.sqrt(D)
    target = torch.randint(0, V, (N,), generator=g, device="cuda")
    h = torch.randn(N, D, generator=g, device="cuda") + lean * torch.rand(N, 1, generator=g, device="cuda") * w[target]
    return h.to(t), w.to(t), target


def definition(h, w, target, reduction, dloss=None, ignore=IGN):
    """(loss, dh, dw, the norms of the absolute sums with U and with p for dh and for dw, scores) in 64 bits."""
    hd, wd = h.double(), w.double()
    use = target != ignore
    at = torch.where(use, target, 0).long()
    s = hd @ wd.t()
    logp = s - torch.logsumexp(s, 1, keepdim=True)
    each = torch.where(use, -logp.gather(1, at[:, None])[:, 0], 0.0)
    n = use.sum()
    loss = each if reduction == "none" else each.sum() / (n if reduction == "mean" else 1)
    up = torch.ones((), device="cuda") if dloss is None else dloss
    g = torch.where(use, up.double() / (n if reduction == "mean" else 1), 0.0)[:, None]
    u = (logp.exp() - F.one_hot(at, w.shape[0])) * g
    u = torch.where(use[:, None], u, 0.0)
    p = torch.where(use[:, None], logp.exp() * g.abs(), 0.0)
    sizes = [(x.abs() @ wd.abs()).norm().item() for x in (u, p)] + [(x.abs().t() @ hd.abs()).norm().item() for x in (u, p)]
    return loss, u @ wd, u.t() @ hd, sizes[:2], sizes[2:], s


def score_error(h, w):
    size = float((h.double().abs() @ w.double().abs().t()).max())
    extra = 2.0**-22 if h.dtype == torch.float32 else 0.0
    return ((h.shape[1] + 4) * 2.0**-24 + extra + 2 * 2.0**-24) * size


def check(got, want, h, w, what=""):
    loss, dh, dw = got
    loss_, dh_, dw_, ah, aw, s = want
    e = score_error(h, w)
    room = 2 * e + 8 * 2.0**-24 * (float(s.abs().max()) + math.log(w.shape[0]) + 1)
    many = h.shape[0] if loss.dim() == 0 else 1
    assert loss.dtype == torch.float32 and loss.shape == loss_.shape
    assert ((loss.double() - loss_).abs() <= room * (many if loss_.abs().max() > 100 else 1) + 2.0**-24 * loss_.abs()).all(), what
    out = 2.0**-8 if h.dtype == torch.bfloat16 else 2.0**-24
    plane = 2.0**-12 if h.dtype == torch.bfloat16 else 2.0**-22
    for x, y, a, k, like in ((dh, dh_, ah, w.shape[0], h), (dw, dw_, aw, h.shape[0], w)):
        if x is None:
            continue
        assert x.dtype == like.dtype and x.shape == like.shape and x.is_contiguous()
        room = (plane + math.sqrt(k) * 2.0**-24) * a[0] + (2 * e + 2.0**-22 * 32) * a[1]
        assert float((x.double() - y).norm()) <= out * float(y.norm()) + room + 1e-30, what


def call(h, w, target, reduction="mean", dloss=None, ignore=IGN):
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(h, w, target, ignore, reduction)
    dh, dw = torch.autograd.grad(loss, [h, w], dloss if dloss is not None else torch.ones_like(loss))
    return loss.detach(), dh, dw


SIZES = [(1, 1, 1), (1, 2, 3), (5, 7, 8), (16, 1000, 32), (33, 257, 64), (130, 300, 101), (129, 256, 96), (257, 515, 130),
         (64, 5000, 512), (300, 4097, 96), (1, 30000, 64), (7, 20011, 256), (9000, 100, 64), (2049, 31, 33), (128, 127, 2048)]


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,D", SIZES)
def test_loss_and_gradients(N, V, D, t):
    h, w, target = make(N, V, D, t)
    g = torch.Generator("cuda").manual_seed(1)
    for reduction in ("mean", "sum", "none"):
        dloss = 0.1 + torch.rand((N,) if reduction == "none" else (), generator=g, device="cuda")
        check(call(h, w, target, reduction, dloss), definition(h, w, target, reduction, dloss), h, w, reduction)
    left = target.clone()
    left[torch.rand(N, generator=g, device="cuda") < 0.4] = IGN
    left[0] = target[0]
    got = call(h, w, left.int(), "mean")
    check(got, definition(h, w, left, "mean"), h, w, "ignored rows")
    assert not got[1][left == IGN].any()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_several_pieces_of_the_vocabulary(t):
    h, w, target = make(6000, 60001 if t == torch.bfloat16 else 30001, 64, t)
    check(call(h, w, target), definition(h, w, target, "mean"), h, w)


def test_offsets_beyond_32_bits():
    """Rows so far apart that the last begins beyond 2^31 elements."""
    t = torch.bfloat16
    base = torch.empty(1100, 1 << 21, device="cuda", dtype=t)
    h, w, target = make(1100, 300, 64, t)
    far = base[:, 64:128]
    far.copy_(h)
    a, b = call(far, w, target), call(h, w, target)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_small_and_large_gradients_and_values():
    """Planes are scaled by their largest value: inputs and gradients of other sizes lose nothing."""
    for t in (torch.float32, torch.bfloat16):
        h, w, target = make(70, 200, 64, t)
        for a, b, up in ((2.0**-30, 2.0**30, 1.0), (2.0**20, 2.0**-20, 2.0**-40), (1.0, 1.0, 2.0**60)):
            dloss = torch.tensor(up, device="cuda")
            check(call(h * a, w * b, target, "mean", dloss), definition(h * a, w * b, target, "mean", dloss), h * a, w * b, (t, a, b))


def test_confident_rows():
    """Scores up to 100 and losses near zero: the loss keeps its digits where the target leads."""
    h, w, target = make(64, 300, 64, torch.float32, lean=0.0)
    w = F.normalize(w)
    h = 30.0 * w[target]
    check(call(h, w, target, "none"), definition(h, w, target, "none"), h, w)


def test_rows_that_do_not_count():
    h, w, target = make(40, 90, 32, torch.float32)
    none = torch.full_like(target, IGN)
    loss, dh, dw = call(h, w, none, "mean")
    assert loss.isnan() and not dh.any() and not dw.any()
    loss, dh, dw = call(h, w, none, "sum")
    assert loss == 0 and not dh.any() and not dw.any()
    for ignore in (0, -1, 89, 10**12):        # any value may be the ignored one, a word of the vocabulary too
        left = torch.where(torch.arange(40, device="cuda") % 3 == 0, ignore, target)
        check(call(h, w, left, "sum", ignore=ignore), definition(h, w, left, "sum", ignore=ignore), h, w)
    # what ignored rows hold does not matter
    h2 = h.clone()
    left = target.clone()
    left[3:9] = IGN
    h2[3:9] = math.nan
    h2[5] = math.inf
    a, b = call(h2, w, left), call(h, w, left)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_many_rows_of_which_few_or_none_count(t):
    """From 1024 rows on those that count are put next to each other."""
    h, w, target = make(1500, 700, 64, t)
    at = torch.arange(1500, device="cuda")
    for keep in (at < 0, at == 1499, at == 0, at % 500 == 3, at < 1024, at >= 1200, at % 2 == 1, at >= 0):
        left = torch.where(keep, target, IGN)
        h2 = torch.where(keep[:, None], h, math.nan)
        for reduction in ("sum", "none", "mean"):
            dloss = 0.5 + torch.rand((1500,) if reduction == "none" else (), device="cuda")
            got, want = call(h2, w, left, reduction, dloss), definition(h, w, left, reduction, dloss)
            if reduction == "mean" and not keep.any():
                assert got[0].isnan() and not got[1].any() and not got[2].any()
                continue
            check(got, want, h, w, (reduction, int(keep.sum())))
            assert not got[1][~keep].any()
    wrong = target.clone()
    wrong[::3], wrong[1000] = IGN, 700
    loss, dh, dw = call(h, w, wrong, "none")
    row = at == 1000
    assert torch.equal(loss.isnan(), row) and torch.equal(dh.isnan().all(1), row) and not dh[~row].isnan().any() and dw.isnan().all()


def test_targets_outside_the_vocabulary_and_special_values():
    h, w, target = make(40, 90, 32, torch.float32)
    for bad in (90, -1, 2**40):
        wrong = target.clone()
        wrong[7] = bad
        loss, dh, dw = call(h, w, wrong, "none")
        row = torch.arange(40, device="cuda") == 7
        assert torch.equal(loss.isnan(), row) and torch.equal(dh.isnan().all(1), row) and not dh[~row].isnan().any()
        assert dw.isnan().all()
    h2 = h.clone()
    h2[4, 3] = math.nan
    loss, dh, _ = call(h2, w, target, "none")
    assert torch.equal(loss.isnan(), torch.arange(40, device="cuda") == 4) and dh[4].isnan().all() and not dh[5].isnan().any()
    w2 = w.clone()
    w2[11] = -math.inf                         # inf - inf within a score: NaN, as the scores of F.linear
    assert call(h, w2, target, "none")[0].isnan().all()
    h3, w3 = h.abs(), w.clone()
    w3[11] = -math.inf                         # a word that is never said
    left = torch.where(target == 11, 12, target)
    loss = call(h3.bfloat16(), w3.bfloat16(), left, "none")[0]
    want = definition(h3.bfloat16(), w3.bfloat16(), left, "none")[0]
    assert ((loss - want).abs() < 1e-4).all()


def test_strides_shapes_and_types():
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    h, w, target = make(60, 200, 64, torch.bfloat16)
    want = call(h, w, target)
    wide = torch.randn(60, 200, device="cuda").bfloat16()
    for at in (0, 8, 3):
        wide[:, at:at + 64] = h
        got = call(wide[:, at:at + 64], w, target)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(call(h.t().contiguous().t(), w.t().contiguous().t(), target), want))
    h3 = h.view(5, 12, 64).requires_grad_()
    loss = linear_cross_entropy(h3, w, target.view(5, 12), reduction="none")
    assert loss.shape == (5, 12)
    loss.mean().backward()
    assert torch.equal(h3.grad.view(60, 64), want[1])
    one = linear_cross_entropy(h[0], w, target[0], reduction="none")     # a single row without a batch
    assert one.shape == () and abs(float(one) - float(loss.flatten()[0])) < 1e-6
    same = h[:1].expand(60, 64)
    assert torch.equal(call(same, w, target)[0], call(same.contiguous(), w, target)[0])


def test_no_rows():
    h, w, _ = make(1, 50, 32, torch.float32)
    target = torch.zeros(0, dtype=torch.long, device="cuda")
    for reduction, want in (("none", None), ("sum", 0.0), ("mean", math.nan)):
        loss, dh, dw = call(h[:0], w, target, reduction)
        assert loss.numel() == 0 if want is None else (loss.isnan() if math.isnan(want) else loss == want)
        assert dh.shape == (0, 32) and not dw.any()


def test_one_gradient_alone_and_none():
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    for t in (torch.float32, torch.bfloat16):
        h, w, target = make(200, 700, 64, t)
        loss, dh, dw = call(h, w, target)
        h1 = h.clone().requires_grad_()
        linear_cross_entropy(h1, w, target).backward()
        w1 = w.clone().requires_grad_()
        linear_cross_entropy(h, w1, target).backward()
        assert torch.equal(h1.grad, dh) and torch.equal(w1.grad, dw)
        assert torch.equal(linear_cross_entropy(h, w, target), loss)
        with torch.no_grad():
            assert torch.equal(linear_cross_entropy(h1, w1, target), loss)


def test_gradient_against_differences():
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    h, w, target = make(6, 40, 16, torch.float32)
    loss, dh, dw = call(h, w, target, "sum")
    for x, d in ((h, dh), (w, dw)):
        for i in (0, 17, 55, 95):
            step = torch.zeros_like(x)
            step.view(-1)[i] = 2.0**-6
            f = lambda y: float(linear_cross_entropy(*((y, w) if x is h else (h, y)), target, reduction="sum"))
            slope = (f(x + step) - f(x - step)) / 2.0**-5
            # third derivatives below 8: the difference is off by 2^-12 * 8 / 6; roundings of losses up to 40 by 2^-24 * 80 * 32
            assert abs(slope - float(d.view(-1)[i])) < 2.0**-11 + 2.0**-24 * 80 * 32


def test_the_same_twice():
    for t in (torch.float32, torch.bfloat16):
        h, w, target = make(3000, 5000, 128, t)
        a, b = call(h, w, target), call(h, w, target)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_under_autocast():
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    h, w, target = make(100, 300, 64, torch.float32)
    h.requires_grad_(), w.requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = linear_cross_entropy(h, w, target)
    loss.backward()
    assert h.grad.dtype == w.grad.dtype == torch.float32
    want = call(h.bfloat16(), w.bfloat16(), target)
    assert torch.equal(loss, want[0]) and torch.equal(h.grad, want[1].float()) and torch.equal(w.grad, want[2].float())
    with torch.autocast("cuda", dtype=torch.float16), pytest.raises(ValueError, match="float16"):
        linear_cross_entropy(h, w, target)


@pytest.mark.parametrize("N", [200, 1300])
def test_captured_replayed_and_on_another_stream(N):
    h, w, target = make(N, 3000, 64, torch.bfloat16)
    target[::7] = IGN
    h.requires_grad_(), w.requires_grad_()
    from mathbrain.linear_cross_entropy import linear_cross_entropy

    def step():
        loss = linear_cross_entropy(h, w, target, reduction="mean")
        return (loss, *torch.autograd.grad(loss, [h, w]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [x.detach().clone() for x in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(there, step()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            h.mul_(1.1)
            target.copy_(torch.where(target == IGN, (i * 100 + 5) % 3000, torch.where(target % 5 == i, IGN, target)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_traced():
    from mathbrain.linear_cross_entropy import linear_ce_bwd, linear_ce_fwd
    h, w, target = make(30, 70, 32, torch.float32)
    torch.library.opcheck(linear_ce_fwd.op, (h, w, target, IGN, 1), test_utils=("test_schema", "test_faketensor"))
    loss, stats = linear_ce_fwd(h, w, target, IGN, 1)
    torch.library.opcheck(linear_ce_bwd.op, (h, w, target, stats, torch.ones_like(loss), IGN, 1, True, False),
                          test_utils=("test_schema", "test_faketensor"))


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    h, w, target = make(30, 70, 32, torch.float32)
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        linear_cross_entropy(fwad.make_dual(h, h), w, target)


def test_refusals():
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    h, w, target = make(30, 70, 32, torch.float32)
    for bad in (dict(hidden=h.bfloat16()), dict(hidden=h.half(), weight=w.half()), dict(hidden=h[:, :16]), dict(weight=w[0]),
                dict(target=target[:5]), dict(target=target.float()), dict(reduction="max"), dict(weight=w[:0]),
                dict(hidden=h[:, :0], weight=w[:, :0])):
        with pytest.raises(ValueError):
            linear_cross_entropy(**(dict(hidden=h, weight=w, target=target) | bad))
    with pytest.raises(NotImplementedError):
        linear_cross_entropy(h.cpu(), w, target)
    with pytest.raises(NotImplementedError):
        linear_cross_entropy(h, w, target.cpu())


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 8, 9, 13, 16, 17])
def test_few_rows(N, t):
    """Few rows have kernels of their own, by rows and by channels, in fp32 twice a call for up to 16 rows: each, and sizes on both sides of
    what they take."""
    for V, D in ((3, 1), (33, 7), (64, 64), (1001, 101), (517, 256), (300, 257), (2050, 512), (129, 513), (1030, 1000), (515, 1024), (130, 1025),
                 (259, 2047), (131, 2048), (70, 2049), (40003, 64)):
        h, w, target = make(N, V, D, t, seed=N)
        g = torch.Generator("cuda").manual_seed(N)
        for reduction in ("mean", "none"):
            dloss = 0.1 + torch.rand((N,) if reduction == "none" else (), generator=g, device="cuda")
            check(call(h, w, target, reduction, dloss), definition(h, w, target, reduction, dloss), h, w, (V, D, reduction))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,D", [(3, 700, 96), (8, 1003, 200), (4, 300, 1500), (8, 257, 1024), (13, 301, 101), (16, 1003, 1024), (7, 200, 2048)])
def test_few_rows_at_the_edges(N, V, D, t):
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    h, w, target = make(N, V, D, t, seed=9)
    # ignored rows, with NaN in them; one gradient alone; the same twice
    left = target.clone()
    left[1] = IGN
    hn = h.clone()
    hn[1] = float("nan")
    got, want = call(hn, w, left), definition(h, w, left, "mean")
    check(got, want, h, w)
    assert not got[1][1].any()
    assert all(torch.equal(a, b) for a, b in zip(got, call(hn, w, left)))
    for side in (0, 1):
        x = [hn.clone(), w.clone()]
        x[side].requires_grad_()
        assert torch.equal(torch.autograd.grad(linear_cross_entropy(*x, left), x[side])[0], got[1 + side])
    # all ignored; gradients of zero
    loss, dh, dw = call(h, w, torch.full_like(target, IGN), "sum")
    assert float(loss) == 0 and not dh.any() and not dw.any()
    loss, dh, dw = call(h, w, target, "sum", torch.zeros((), device="cuda"))
    assert not dh.any() and not dw.any()
    # a target outside the vocabulary reaches its own row of dh and all of dw
    out = target.clone()
    out[0] = V
    loss, dh, dw = call(h, w, out, "none")
    assert torch.isnan(loss[0]) and not torch.isnan(loss[1:]).any()
    assert torch.isnan(dh[0]).all() and not torch.isnan(dh[1:]).any() and torch.isnan(dw).all()
    # rows that are further apart, and rows that begin anywhere
    wide = torch.randn(V + 1, D + 9, device="cuda").to(t)
    for at in (0, 1, 8):
        wide[1:, at:at + D] = w
        check(call(h, wide[1:, at:at + D], target), definition(h, w, target, "mean"), h, w, at)
    # captured and replayed with other values
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()

    def step():
        loss = linear_cross_entropy(a, b, left)
        return [loss.detach(), *torch.autograd.grad(loss, [a, b])]

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        with torch.no_grad():
            a.mul_(0.9)
            left.copy_(torch.where(torch.arange(N, device="cuda") == i, IGN, target))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, step()))
