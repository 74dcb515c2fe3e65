"""clip_grad_norm_ / clip_gradients / grad_norm (mathbrain/grad_clip.py) against the definition in
float64: many tensors of mixed types, odd sizes and alignments, more tensors than one launch
takes, values whose squares leave fp32, NaN and infinities, shared memory, and the refusals.

Tolerances: the norm's squares and sums are in 64 bits, so it is off by its one rounding to fp32
(2^-24).  The factor's rounding, the product's and that of an fp32 result are 3 * 2^-24 < 2e-7;
a bf16 result adds half a step of its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(shapes, dtypes, seed, mul=0.1):
    g = torch.Generator().manual_seed(seed)
    return [(mul * torch.randn(s, generator=g)).to(dtypes[i % len(dtypes)]).cuda() for i, s in enumerate(shapes)]


def norm64(grads):
    return float(torch.cat([x.detach().cpu().double().reshape(-1) for x in grads]).norm())


def same_scaled(got, src, factor):
    for a, b in zip(got, src):
        want = b.cpu().double() * factor
        half = torch.finfo(a.dtype).eps / 2 if a.dtype == torch.bfloat16 else 0.0
        assert ((a.cpu().double() - want).abs() <= (half + 2e-7) * want.abs() + 1e-44).all()


SHAPES = [(3,), (64, 64), (1,), (4097,), (128, 130), (0,), (5, 7, 9), (8192,), (333, 77)]
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F32, BF16, BF16]])
@pytest.mark.parametrize("max_norm", [0.0, 1.0, 1e6])
def test_in_place(dtypes, max_norm):
    from mathbrain.grad_clip import clip_grad_norm_
    grads = make(SHAPES, dtypes, 1)
    before = [x.clone() for x in grads]
    params = [torch.nn.Parameter(torch.empty_like(x)) for x in grads] + [torch.nn.Parameter(torch.zeros(2, device="cuda"))]
    for p, x in zip(params, grads):
        p.grad = x
    norm = clip_grad_norm_(params, max_norm)
    want = norm64(before)
    assert norm.shape == () and norm.dtype == F32 and abs(float(norm) - want) <= 1e-7 * want
    assert params[-1].grad is None
    same_scaled(grads, before, min(1.0, max_norm / (want + 1e-6)))
    if max_norm > want:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("src", [[F32], [BF16], [BF16, F32]])
@pytest.mark.parametrize("dst", [F32, BF16])
def test_into_other_buffers(src, dst):
    from mathbrain.grad_clip import clip_gradients
    grads = make(SHAPES, src, 2)
    before = [x.clone() for x in grads]
    flat = torch.full((sum(x.numel() for x in grads) + 16,), 7.0, dtype=dst, device="cuda")
    out, at = [], 8
    for x in grads:   # odd offsets: the buffers' tensors are not aligned
        out.append(flat[at:at + x.numel()].view(x.shape))
        at += x.numel()
    for max_norm in (0.5, 1e9):
        norm = clip_gradients(grads, max_norm, out=out)
        want = norm64(before)
        assert abs(float(norm) - want) <= 1e-7 * want
        same_scaled(out, before, min(1.0, max_norm / (want + 1e-6)))
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    assert (flat[:8] == 7).all() and (flat[-8:] == 7).all()


@pytest.mark.parametrize("offset", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_misaligned_tensors(offset, dtype):
    from mathbrain.grad_clip import clip_gradients
    flat = torch.randn(30000, device="cuda").to(dtype)
    before = flat.clone()
    x = flat[offset:offset + 20001]
    norm = clip_gradients([x], 3.0)
    want = norm64([before[offset:offset + 20001]])
    assert abs(float(norm) - want) <= 1e-7 * want
    same_scaled([x], [before[offset:offset + 20001]], 3.0 / (want + 1e-6))
    assert torch.equal(flat[:offset], before[:offset]) and torch.equal(flat[offset + 20001:], before[offset + 20001:])


def test_more_tensors_than_a_launch_takes():
    from mathbrain.grad_clip import clip_gradients, grad_norm
    grads = make([(i % 37 + 1, 11) for i in range(500)], [F32, BF16], 3)
    before = [x.clone() for x in grads]
    want = norm64(before)
    assert abs(float(grad_norm(grads)) - want) <= 1e-7 * want
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    norm = clip_gradients(grads, 0.25)
    assert abs(float(norm) - want) <= 1e-7 * want
    same_scaled(grads, before, 0.25 / (want + 1e-6))


def test_one_large_tensor():
    from mathbrain.grad_clip import clip_gradients
    x = torch.randn(12_345_679, device="cuda") * 1e-3
    before = x.clone()
    norm = clip_gradients([x], 1.0)
    want = norm64([before])
    assert abs(float(norm) - want) <= 1e-7 * want
    same_scaled([x], [before], 1.0 / (want + 1e-6))


def test_squares_that_leave_fp32():
    from mathbrain.grad_clip import clip_gradients
    for value in (1e30, 1e-30):
        x = torch.full((1000,), value, device="cuda")
        want = norm64([x])
        norm = clip_gradients([x], 1.0)
        assert abs(float(norm) - want) <= 1e-7 * want
        assert abs(float(x[3]) - value * min(1.0, 1 / (want + 1e-6))) <= 2e-7 * value


def test_not_finite_norms_scale_as_their_factor_does():
    from mathbrain.grad_clip import clip_grad_norm_, clip_gradients
    x, y = torch.ones(5, device="cuda"), torch.ones(3, device="cuda")
    y[1] = float("nan")
    assert torch.isnan(clip_gradients([x, y], 1.0)) and torch.isnan(x).all() and torch.isnan(y).all()
    x, y = torch.ones(5, device="cuda"), torch.ones(3, device="cuda")
    y[1] = float("-inf")
    assert torch.isinf(clip_gradients([x, y], 1.0)) and not x.any() and torch.isnan(y[1]) and not y[0]
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    p.grad = torch.tensor([1.0, float("inf"), 2.0], device="cuda")
    with pytest.raises(RuntimeError, match="clip_grad_norm_"):
        clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert p.grad.tolist() == [1.0, float("inf"), 2.0]
    p.grad[1] = 2.0
    assert float(clip_grad_norm_(p, 1.5, error_if_nonfinite=True)) == 3.0


def test_matches_torch_on_a_model():
    from mathbrain.baseline import RoPETransformerLM
    from mathbrain.grad_clip import clip_grad_norm_
    torch.manual_seed(0)
    m = RoPETransformerLM(200, 64, 2, 2, dropout=0.0).cuda()
    m(torch.randint(0, 200, (2, 33), device="cuda")).square().mean().backward()
    before = [p.grad.clone() for p in m.parameters()]
    mine = clip_grad_norm_(m.parameters(), 1e-3)
    scaled = [p.grad.clone() for p in m.parameters()]
    for p, x in zip(m.parameters(), before):
        p.grad = x
    theirs = torch.nn.utils.clip_grad_norm_(m.parameters(), 1e-3)
    assert torch.allclose(mine, theirs, rtol=1e-5)
    assert all(torch.allclose(a, p.grad, rtol=1e-5, atol=0) for a, p in zip(scaled, m.parameters()))


def test_other_orders_of_dimensions():
    from mathbrain.grad_clip import clip_gradients, grad_norm
    base = torch.randn(6, 40, 50, device="cuda")
    before = base.clone()
    norm = clip_gradients([base.permute(2, 0, 1)], 1.0)      # in place: every element once, in any order
    want = norm64([before])
    assert abs(float(norm) - want) <= 1e-7 * want
    same_scaled([base], [before], 1.0 / (want + 1e-6))
    out = torch.empty(50, 6, 40, device="cuda")
    clip_gradients([before.permute(2, 0, 1)], 1e9, out=[out])
    assert torch.equal(out, before.permute(2, 0, 1))
    gaps = before[:, ::2]
    assert abs(float(grad_norm([gaps])) - norm64([gaps])) <= 1e-6 * want
    with pytest.raises(ValueError, match="gaps"):
        clip_gradients([gaps], 1.0)
    with pytest.raises(ValueError, match="gaps"):
        clip_gradients([torch.ones(1, device="cuda").expand(4)], 1.0)


def test_shared_memory_is_refused():
    from mathbrain import _lib
    from mathbrain.grad_clip import clip_gradients
    x = torch.randn(100, device="cuda")
    before = x.clone()
    spare = torch.empty(100, device="cuda")
    for grads, out in (([x, x], None), ([x[:60], x[50:]], None), ([x, x], [spare, spare]), ([x[:50]], [x[1:51]]),
                       ([x[:50], x[50:]], [x[50:], x[:50]])):
        with pytest.raises(_lib.HipKernelError, match="share memory"):
            clip_gradients(grads, 0.1, out=out)
    assert torch.equal(x, before)
    other = torch.empty(100, device="cuda")
    norm = clip_gradients([x, x], 0.1, out=[spare, other])   # read twice: it counts twice
    assert abs(float(norm) - norm64([x, x])) <= 1e-7 * norm64([x, x]) and torch.equal(spare, other)
    clip_gradients([x[:50], x[50:]], 1e9)                    # neighbours


def test_same_norm_each_time_streams_and_graphs():
    from mathbrain.grad_clip import clip_gradients
    grads = make([(1000, 511), (77,), (3, 4096)], [F32, BF16], 5)
    out = [torch.empty_like(x) for x in grads]
    first = clip_gradients(grads, 0.5, out=out)
    keep = [x.clone() for x in out]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = clip_gradients(grads, 0.5, out=out)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first, second) and all(torch.equal(a, b) for a, b in zip(out, keep))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients(grads, 0.5, out=out)
    for i in range(4):
        for x in grads:
            x.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        want = clip_gradients(grads, 0.5, out=out)
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(got, out)), i


@pytest.mark.parametrize("out", [False, True])
def test_a_graph_notices_that_what_it_saved_was_scaled(out):
    from mathbrain.grad_clip import clip_gradients
    x = torch.randn(50, device="cuda", requires_grad=True)
    saved = torch.randn(50, device="cuda")
    y = (x * saved).sum()
    clip_gradients([torch.ones_like(saved)] if out else [saved], 0.1, out=[saved] if out else None)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    from mathbrain.grad_clip import clip_grad_norm_, clip_gradients, grad_norm
    x = torch.randn(4, 4, device="cuda")
    with pytest.raises(NotImplementedError):
        clip_gradients([x.cpu()], 1.0)
    with pytest.raises(NotImplementedError):
        clip_gradients([x], 1.0, out=[x.cpu()])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_gradients([x], bad)
    with pytest.raises(ValueError, match="float16"):
        clip_gradients([x.half()], 1.0)
    for layout in (torch.sparse_coo, torch.sparse_csr):
        with pytest.raises(ValueError, match="dense float32"):
            clip_gradients([x, x.to_sparse(layout=layout)], 1.0)
    with pytest.raises(ValueError, match="1 outputs for 2"):
        clip_gradients([x, x], 1.0, out=[x])
    with pytest.raises(ValueError, match="contiguous"):
        clip_gradients([x], 1.0, out=[torch.empty(4, 4, device="cuda").t()])
    with pytest.raises(ValueError, match="contiguous"):
        clip_gradients([x], 1.0, out=[torch.empty(16, device="cuda")])
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm_([torch.nn.Parameter(x)], 1.0, norm_type=1.0)
    with pytest.raises(ValueError, match="sparse"):
        clip_gradients([torch.sparse_coo_tensor([[0], [1]], [1.0], (4, 4), device="cuda")], 1.0)
    assert float(clip_grad_norm_([], 1.0)) == 0.0 and float(grad_norm([])) == 0.0
    assert float(clip_gradients([torch.empty(0, device="cuda")], 1.0)) == 0.0


def test_tangents_are_refused():
    """A dual tensor's tangent would have to be scaled with it."""
    import torch.autograd.forward_ad as fw
    from mathbrain.grad_clip import clip_gradients, grad_norm
    x = torch.randn(6, device="cuda")
    before = x.clone()
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: clip_gradients([d], 0.1), lambda: clip_gradients([x[:3]], 0.1, out=[d[3:]]), lambda: grad_norm([d])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert float(grad_norm([x])) > 0
    assert torch.equal(x, before)


def test_memory_shared_with_a_copied_gradient_is_refused():
    """A gradient that is not contiguous is copied before the library sees it; the output that would
    overwrite it is refused all the same."""
    from mathbrain import _lib
    from mathbrain.grad_clip import clip_gradients
    x = torch.randn(40, 50, device="cuda")
    before, spare = x.clone(), torch.empty(50, 40, device="cuda")
    for grads, out in (([x.t()], [x.view(50, 40)]), ([x[:, ::2]], [x.view(-1)[:1000].view(40, 25)]),
                       ([spare[:, :1].t(), x.t()], [torch.empty(1, 50, device="cuda"), x.view(50, 40)])):
        with pytest.raises(_lib.HipKernelError, match="share memory"):
            clip_gradients(grads, 0.1, out=out)
    assert torch.equal(x, before)
    clip_gradients([x.t()], 1e9, out=[spare])
    assert torch.equal(spare, x.t())
    both = torch.randn(80, 50, device="cuda")                                   # neighbours
    want = both[:40].t().clone()
    clip_gradients([both[:40].t()], 1e9, out=[both[40:].view(50, 40)])
    assert torch.equal(both[40:].view(50, 40), want) and torch.equal(both[:40].t(), want)
