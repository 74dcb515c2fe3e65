"""relative_bias_attention (mathbrain/bias_attention.py) against its definition in float64: outputs
and the gradients of q, k, v and the bias table.

Tolerances are bounds, element by element, worked out from the same inputs (`bounds` below).  With
e = 2^-24 and u = finfo(t).eps / 2 for bf16 (0 for fp32):
 * a score is a sum of hd products and a bias, off by at most cs = (hd + 8) e (scale |q|.|k| + |bias|);
   a probability is then off by dp = 2 cs + (n + 16) e of itself, n the keys summed over;
 * o: each term p v is off by dp + u (p's rounding before the product), the result by u of itself;
 * delta = dO . o takes o's error times |dO|; ds = p (dO . v - delta) adds to that dp of its size and
   hd e |dO|.|v|; in the products with k and q it is rounded (u), in dbias it is not;
 * sums over m terms add m e of the terms' sizes; results are rounded (u) at the end."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def bucket(n, starts):
    return sum(int(s <= n) for s in starts) - 1


def plan(B, Lq, Lk, buckets, reach, causal, lengths, q_start):
    """(bucket of each pair [B, Lq, Lk], whether it counts)."""
    from mathbrain.bias_attention import bucket_starts
    side = buckets if causal else buckets // 2
    starts = bucket_starts(side, reach)
    table = torch.tensor([bucket(n, starts) for n in range(reach + 1)])
    start = q_start if torch.is_tensor(q_start) else torch.full((B,), Lk - Lq if q_start is None else q_start)
    d = start.cpu().long()[:, None, None] + torch.arange(Lq)[None, :, None] - torch.arange(Lk)
    n = table[d.abs().clamp(max=reach)] + (0 if causal else side) * (d < 0)
    seen = d >= 0 if causal else torch.ones_like(d, dtype=torch.bool)
    if lengths is not None:
        seen = seen & (torch.arange(Lk) < lengths.cpu().long()[:, None, None])
    return n.expand(B, Lq, Lk), seen.expand(B, Lq, Lk)


def definition(q, k, v, bias, do, n, seen, scale, t):
    """o, dq, dk, dv, dbias in float64 with their bounds."""
    u = torch.finfo(t).eps / 2 if t == BF16 else 0.0
    q, k, v, bias, do = (x.detach().cpu().double() for x in (q, k, v, bias, do))
    B, H, Lq, hd = q.shape
    G = H // k.shape[1]
    Lk = k.shape[2]
    live = seen.any(1)[:, None, :, None]        # keys that nobody sees may hold anything
    k = torch.where(live, k, 0.0).repeat_interleave(G, 1)
    v = torch.where(live, v, 0.0).repeat_interleave(G, 1)
    seen = seen[:, None]
    b = bias.t()[:, n].transpose(0, 1)          # [B, H, Lq, Lk]
    s = (q @ k.mT * scale + b).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top.isfinite(), top, 0.0))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    cs = (hd + 8) * E * (q.abs() @ k.abs().mT * scale + b.abs()) * seen
    dp = 2 * cs.amax(-1, keepdim=True) + (Lk + 16) * E
    o = p @ v
    o_off = (dp + u + Lk * E) * (p @ v.abs()) * (1 + u) + u * o.abs()
    back = do @ v.mT
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (back - delta)
    ds_off = p * (dp * (back.abs() + delta.abs()) + hd * E * (do.abs() @ v.abs().mT)
                  + (do.abs() * (o_off + hd * E * o.abs())).sum(-1, keepdim=True)) * (1 + dp)
    f_off = ds_off + u * (ds.abs() + ds_off)

    def shared(x):
        return x.view(B, H // G, G, Lk, hd).sum(2)
    dq, dk, dv = ds @ k * scale, shared(ds.mT @ q * scale), shared(p.mT @ do)
    dq_off = (f_off + Lk * E * ds.abs()) @ k.abs() * scale
    dk_off = shared((f_off + G * Lq * E * ds.abs()).mT @ q.abs() * scale)
    dv_off = shared(((dp + u + G * Lq * E) * p).mT @ do.abs())
    nb = bias.shape[0]
    one = torch.nn.functional.one_hot(n, nb).double().view(B, 1, Lq * Lk, nb)
    db = (ds.reshape(B, H, 1, -1) @ one).sum((0, 2)).t()
    db_off = ((ds_off + (B * Lq * Lk) * E * ds.abs()).reshape(B, H, 1, -1) @ one).sum((0, 2)).t()
    res = []
    for x, off in ((o, o_off), (dq, dq_off), (dk, dk_off), (dv, dv_off), (db, db_off)):
        res.append((x, off * (1 + u) + (u + 2 * E) * x.abs() + 1e-30))
    return res


NAMES = ("o", "dq", "dk", "dv", "dbias")


def near(got, want, name):
    x, off = want
    got = got.detach().cpu().double()
    assert got.shape == x.shape and torch.isfinite(got).all(), name
    worst = float(((got - x).abs() / off).max()) if x.numel() else 0.0
    print(f"{name}: {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, (name, worst)


def inputs(B, H, Hk, Lq, Lk, hd, t, buckets, seed, mul=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = ((mul * torch.randn(s, generator=g)).to(t).cuda() for s in
                   ((B, Lq, H, hd), (B, Lk, Hk, hd), (B, Lk, Hk, hd), (B, Lq, H, hd)))
    bias = torch.randn(buckets, H, generator=g).to(t).cuda()
    return [x.transpose(1, 2) for x in (q, k, v)] + [bias, do.transpose(1, 2)]


def check(q, k, v, bias, do, reach=128, causal=True, scale=None, lengths=None, q_start=None, grads=True):
    from mathbrain.bias_attention import relative_bias_attention
    B, H, Lq, hd = q.shape
    leaves = [x.detach().requires_grad_() for x in (q, k, v, bias)]
    o = relative_bias_attention(*leaves, max_distance=reach, causal=causal, scale=scale, lengths=lengths,
                                q_start=q_start)
    got = [o, *torch.autograd.grad(o, leaves, do)] if grads else [o]
    n, seen = plan(B, Lq, k.shape[2], bias.shape[0], reach, causal, lengths, q_start)
    want = definition(q, k, v, bias, do, n, seen, 1 / math.sqrt(hd) if scale is None else scale, q.dtype)
    assert o.dtype == q.dtype
    for x, leaf in zip(got[1:], leaves):
        assert x.dtype == leaf.dtype
    for x, w, name in zip(got, want, NAMES):
        near(x, w, name)
    with torch.no_grad():
        again = relative_bias_attention(q, k, v, bias, max_distance=reach, causal=causal, scale=scale, lengths=lengths,
                                        q_start=q_start)
    near(again, want[0], "o without gradients")
    return got


SIZES = [(2, 3, 3, 1, 1), (1, 2, 1, 2, 3), (2, 4, 2, 33, 33), (1, 2, 1, 130, 130), (3, 8, 2, 5, 300), (2, 2, 2, 64, 257),
         (1, 1, 1, 257, 129)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("size", SIZES)
def test_matches_the_definition(size, hd, t, causal):
    check(*inputs(*size, hd, t, 32, sum(size) + hd), causal=causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("size", [(1, 4, 2, 700, 700), (2, 2, 1, 300, 1100), (1, 2, 2, 1500, 90), (2, 3, 1, 1, 1000), (2, 12, 4, 500, 800)])
def test_walks_that_are_split(size, hd, t, causal):
    from mathbrain.bias_attention import relative_bias_attention
    q, k, v, bias, do = inputs(*size, hd, t, 32, sum(size) + hd)
    lengths = None if size[0] == 1 else torch.tensor([size[4], size[4] // 3], device="cuda")
    got = check(q, k, v, bias, do, causal=causal, lengths=lengths)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, bias.detach())]
    o = relative_bias_attention(*leaves[:3], bias, causal=causal, lengths=lengths)      # no gradient of the bias
    for x, y in zip(torch.autograd.grad(o, leaves[:3], do), got[1:]):
        assert torch.equal(x, y)
    o = relative_bias_attention(*leaves, causal=causal, lengths=lengths)
    for x, y in zip(torch.autograd.grad(o, leaves, do), got[1:]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("buckets,reach,causal", [(1, 1, True), (2, 9, True), (3, 100, True), (31, 200, True),
                                                  (128, 1024, True), (16, 9, True), (2, 1, False), (6, 2, False),
                                                  (64, 500, False), (256, 1024, False)])
def test_bucket_tables(buckets, reach, causal, t):
    check(*inputs(1, 2, 2, 300, 300, 32, t, buckets, buckets), reach=reach, causal=causal)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_distances_beyond_the_reach(causal, t):
    check(*inputs(1, 1, 1, 700, 700, 64, t, 8, 3), reach=20, causal=causal)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_lengths_and_rows_without_keys(causal, kind, t):
    lengths = torch.tensor([0, 1, 31, 32, 33, 64, 100, 129, 500, -3], dtype=kind).cuda()
    q, k, v, bias, do = inputs(10, 2, 1, 129, 129, 64, t, 32, 5)
    ends = lengths.clamp(0, 129)
    gone = torch.arange(129, device="cuda") >= ends[:, None]
    for bad in (float("nan"), float("inf"), -float("inf")):   # what lies behind a row's end does not matter
        k = torch.where(gone[:, None, :, None], torch.tensor(bad, dtype=t, device="cuda"), k)
        v = torch.where(gone[:, None, :, None], torch.tensor(bad, dtype=t, device="cuda"), v)
        got = check(q, k, v, bias, do, causal=causal, lengths=lengths)
        for x in (got[0], got[1]):
            assert not x[0].any() and not x[9].any()
        for x in (got[2], got[3]):
            assert not x[gone[:, None, :].expand(10, 1, 129)].any()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("Lq,H,Hk", [(1, 4, 4), (3, 8, 2), (70, 4, 4), (200, 2, 1)])
def test_rows_behind_the_last_query_may_hold_anything(Lq, H, Hk, t):
    """A cache that is longer than what it holds, without lengths."""
    q, k, v, bias, do = inputs(4, H, Hk, Lq, 900, 64, t, 32, 37)
    rows = torch.tensor([0, 5, 600, 899 - Lq], device="cuda")
    behind = torch.arange(900, device="cuda") >= (rows + Lq)[:, None]
    for bad in (float("nan"), float("inf")):
        k = torch.where(behind[:, None, :, None], torch.tensor(bad, dtype=t, device="cuda"), k)
        v = torch.where(behind[:, None, :, None], torch.tensor(bad, dtype=t, device="cuda"), v)
        check(q, k, v, bias, do, q_start=rows, grads=Lq > 1)


def test_farthest_positions():
    q, k, v, bias, do = inputs(4, 2, 2, 5, 40, 32, F32, 32, 41)
    for q_start in (1 << 29, -(1 << 29), torch.tensor([1 << 29, -(1 << 29), 1 << 29, 0], device="cuda")):
        check(q, k, v, bias, do, q_start=q_start)
        check(q, k, v, bias, do, q_start=q_start, causal=False)


def test_no_second_derivatives():
    from mathbrain.bias_attention import relative_bias_attention
    q, k, v, bias, do = inputs(1, 1, 1, 4, 4, 32, F32, 4, 43)
    q, do = q.detach().requires_grad_(), do.detach().requires_grad_()
    dq, = torch.autograd.grad(relative_bias_attention(q, k, v, bias), q, do, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dq.sum().backward()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_positions(causal, t):
    args = inputs(6, 4, 2, 40, 210, 64, t, 32, 7)
    for q_start in (0, 170, -20, -40, 100, 209, 100000, -100000):
        check(*args, causal=causal, q_start=q_start)
    rows = torch.tensor([0, 170, -39, 5, 1 << 20, -(1 << 20)], device="cuda")
    check(*args, causal=causal, q_start=rows)
    lengths = torch.tensor([210, 205, 0, 17, 1, 77], dtype=torch.int32, device="cuda")
    check(*args, causal=causal, q_start=rows.int(), lengths=lengths)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("Lq", [1, 2, 3, 5, 8, 16])
@pytest.mark.parametrize("hd,H,Hk", [(64, 8, 8), (128, 8, 2), (32, 5, 1), (64, 16, 1)])
def test_few_queries_against_a_cache(hd, H, Hk, Lq, t):
    for Lk, B in ((1, 2), (63, 3), (777, 3), (4099, 2)):
        lengths = torch.randint(0, Lk + 1, (B,), generator=torch.Generator().manual_seed(Lk)).cuda()
        args = inputs(B, H, Hk, Lq, Lk, hd, t, 32, Lk + Lq)
        check(*args, lengths=lengths, q_start=lengths - Lq, grads=False)
        check(*args, grads=False)


@pytest.mark.parametrize("t", [F32, BF16])
def test_large_scores(t):
    """Scores of hundreds: one key takes all, and nothing leaves the range."""
    q, k, v, bias, do = inputs(1, 2, 2, 70, 150, 64, t, 32, 11)
    check((q * 30).to(t), (k * 10).to(t), v, bias, do)
    check(q, k, v, (bias * 100).to(t), do)
    check(q, k, v, torch.full_like(bias, -3e4), do)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("low", ["-inf", "lowest", -1e9, -70000.0])
@pytest.mark.parametrize("Lq,Lk,hd", [(200, 200, 64), (1, 700, 64), (150, 150, 128)])
def test_biases_that_hide_their_buckets(Lq, Lk, hd, low, t):
    """The buckets of far keys are hidden; the first sequence is short, and its last queries see none."""
    from mathbrain.bias_attention import relative_bias_attention
    q, k, v, bias, do = inputs(2, 4, 2, Lq, Lk, hd, t, 8, 5)
    lengths = torch.tensor([20, Lk], device="cuda")
    hidden = torch.tensor([0, 0, 0, 1, 0, 0, 0, 1], dtype=torch.bool)
    bias[hidden.cuda()] = {"-inf": -math.inf, "lowest": torch.finfo(t).min}.get(low, low)
    n, seen = plan(2, Lq, Lk, 8, 16, False, lengths, None)
    seen = seen & ~hidden[n]
    assert not seen[0, -1].any() and seen[1].any(-1).all()
    want = definition(q, k, v, bias.masked_fill(hidden.cuda()[:, None], 0.0), do, n, seen, 1 / math.sqrt(hd), t)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, bias)]
    o = relative_bias_attention(*leaves, max_distance=16, causal=False, lengths=lengths)
    for x, w, name in zip([o, *torch.autograd.grad(o, leaves, do)], want, NAMES):
        near(x, w, name)


@pytest.mark.parametrize("t", [F32, BF16])
def test_scale_and_bias_types(t):
    q, k, v, bias, do = inputs(2, 2, 2, 50, 50, 32, t, 32, 13)
    check(q, k, v, bias, do, scale=1.0)
    check(q, k, v, bias, do, scale=0.01)
    check(q, k, v, bias.float(), do)


@pytest.mark.parametrize("t", [F32, BF16])
def test_strided_and_broadcast_inputs(t):
    g = torch.Generator().manual_seed(17)
    x = torch.randn(2, 90, 3, 4, 64, generator=g).to(t).cuda()   # a fused projection's parts
    bias, do = torch.randn(32, 4, generator=g).to(t).cuda(), torch.randn(2, 4, 90, 64, generator=g).to(t).cuda()
    check(*(x[:, :, i].transpose(1, 2) for i in range(3)), bias, do)
    heads = torch.randn(3, 2, 4, 90, 64, generator=g).to(t).cuda()
    check(*heads, bias, do)
    odd = torch.randn(2 * 4 * 90 * 64 + 1, generator=g).to(t).cuda()[1:].view(2, 4, 90, 64)
    check(odd, odd, odd, bias, do)                                # rows off the 16 bytes
    channels = torch.randn(2, 4, 90, 128, generator=g).to(t).cuda()[..., ::2]
    check(channels, channels, channels, bias.t().contiguous().t(), do)
    one = torch.randn(1, 4, 1, 64, generator=g).to(t).cuda().expand(2, 4, 90, 64)
    check(one, one, heads[0], bias, do[:, :1, :1].expand(2, 4, 90, 64))


def test_one_tensor_as_all_inputs():
    from mathbrain.bias_attention import relative_bias_attention
    x, _, _, bias, do = inputs(2, 2, 2, 75, 75, 32, F32, 32, 19)
    leaf = x.detach().requires_grad_()
    dx, = torch.autograd.grad(relative_bias_attention(leaf, leaf, leaf, bias), leaf, do)
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    grads = torch.autograd.grad(relative_bias_attention(*parts, bias), parts, do)
    assert torch.allclose(dx, sum(grads), rtol=1e-5, atol=1e-6)


def test_empty_sizes():
    from mathbrain.bias_attention import relative_bias_attention
    for B, Lq, Lk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, bias, do = inputs(B, 2, 1, Lq, Lk, 32, BF16, 32, 1)
        leaves = [x.detach().requires_grad_() for x in (q, k, v, bias)]
        o = relative_bias_attention(*leaves)
        grads = torch.autograd.grad(o, leaves, do)
        assert o.shape == q.shape and not o.any()
        for x, leaf in zip(grads, leaves):
            assert x.shape == leaf.shape and not x.any()


@pytest.mark.parametrize("t", [F32, BF16])
def test_same_bits_each_time_and_on_another_stream(t):
    from mathbrain.bias_attention import relative_bias_attention
    q, k, v, bias, do = inputs(3, 4, 2, 300, 300, 64, t, 32, 23)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, bias)]
    lengths = torch.tensor([300, 77, 222], device="cuda")

    def once():
        o = relative_bias_attention(*leaves, lengths=lengths)
        return [o, *torch.autograd.grad(o, leaves, do)]
    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = once()
    torch.cuda.current_stream().wait_stream(s)
    for a, b, name in zip(first, second, NAMES):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("Lq,Lk", [(1, 3000), (70, 70)])
def test_captured_and_replayed(Lq, Lk):
    from mathbrain.bias_attention import relative_bias_attention
    q, k, v, bias, _ = inputs(2, 4, 2, Lq, Lk, 64, BF16, 32, 29)
    lengths = torch.tensor([Lk, Lk // 2], dtype=torch.int32, device="cuda")

    def once():
        return relative_bias_attention(q, k, v, bias, lengths=lengths, q_start=lengths - Lq)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = once()
    for i in range(4):
        q.copy_(torch.randn_like(q))
        lengths.sub_(1)
        graph.replay()
        want = once()
        torch.cuda.synchronize()
        assert torch.equal(o, want), i


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("L", [100, 1200])
def test_both_directions_captured_and_replayed(L, t):
    from mathbrain.bias_attention import bias_attn_bwd, bias_attn_fwd
    q, k, v, bias, do = inputs(1, 4, 2, L, L, 64, t, 32, 31)
    rest = (128, True, 0.125, None, None, 0)

    def once():
        o, lse = bias_attn_fwd(q, k, v, bias, *rest, True)
        return o, *bias_attn_bwd(q, k, v, bias, o, do, lse, *rest, True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for i in range(4):
        for x in (q, v, do, bias):
            x.copy_(torch.randn_like(x))
        graph.replay()
        want = once()
        torch.cuda.synchronize()
        for x, y, name in zip(got, want, NAMES):
            assert torch.equal(x, y), (i, name)


def test_differences_agree_with_the_gradient():
    """Central differences along a random direction, summed in float64.  At h = 1e-2 the third
    derivative's share (h^2 / 6 of it) and fp32's 2^-24 of the sum over h both stay under 1 % of the
    derivative's scale, which is the norm of the gradient."""
    from mathbrain.bias_attention import relative_bias_attention
    g = torch.Generator().manual_seed(31)
    shapes = ((1, 2, 20, 32), (1, 1, 20, 32), (1, 1, 20, 32), (8, 2))
    leaves = [torch.randn(s, generator=g).cuda().requires_grad_() for s in shapes]
    ways = [torch.randn(s, generator=g).cuda() for s in shapes]
    do = torch.randn(shapes[0], generator=g).cuda()

    def value(*x):
        return (relative_bias_attention(*x, max_distance=12).double() * do.double()).sum()
    grads = torch.autograd.grad(value(*leaves), leaves)
    h = 1e-2
    for i, (grad, way) in enumerate(zip(grads, ways)):
        with torch.no_grad():
            up, down = ([x + (d * h * way if n == i else 0) for n, x in enumerate(leaves)] for d in (1, -1))
            diff = float((value(*up) - value(*down)) / (2 * h))
        along = float((grad.double() * way.double()).sum())
        assert abs(diff - along) <= 1e-2 * float(grad.double().norm() * 6), (i, diff, along)


def test_refusals():
    from mathbrain import _lib
    from mathbrain.bias_attention import relative_bias_attention
    q, k, v, bias, _ = inputs(2, 4, 2, 8, 8, 64, F32, 32, 1)
    base = dict(q=q, k=k, v=v, bias=bias)
    with pytest.raises(NotImplementedError):
        relative_bias_attention(*(x.cpu() for x in base.values()))
    for bad in (dict(q=q[0]), dict(k=k[:, :, :4]), dict(q=q[:1]), dict(q=q.bfloat16()), dict(v=v.bfloat16()),
                dict(q=q.half(), k=k.half(), v=v.half()), dict(bias=bias[:, :2]), dict(bias=bias.half()), dict(bias=bias[:0]),
                dict(bias=bias[:31], causal=False), dict(max_distance=16), dict(max_distance=1025),
                dict(bias=bias.repeat(5, 1), max_distance=500), dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")),
                dict(lengths=torch.zeros(2, device="cuda")), dict(q_start=torch.zeros(2, 1, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError, match="relative_bias_attention"):
            relative_bias_attention(**(base | bad))
    for bad, said in ((dict(k=k[:, :1].expand(2, 3, 8, 64), v=v[:, :1].expand(2, 3, 8, 64)), "multiple of Hk=3"),
                      (dict(q=q[..., :48], k=k[..., :48], v=v[..., :48]), "head_dim=48"), (dict(scale=0.0), "scale"),
                      (dict(scale=float("nan")), "scale"), (dict(q_start=(1 << 29) + 1), "q_start")):
        with pytest.raises(_lib.HipKernelError, match=said):
            relative_bias_attention(**(base | bad))


def with_nan(kind, q, k, v, bias):
    """The inputs with one NaN, and the rows of o [B, H, Lq] that it reaches without a mask."""
    B, H, Lq, _ = q.shape
    q, k, v, bias = (x.clone() for x in (q, k, v, bias))
    rows = torch.zeros(B, H, Lq, dtype=torch.bool)
    G = H // k.shape[1]
    if kind == "q":
        q[0, H - 1, Lq // 2, 3] = math.nan
        rows[0, H - 1, Lq // 2] = True
    elif kind == "bias":       # the bucket of distance 0, which every query here meets
        bias[0, 0] = math.nan
        rows[:, 0] = True
    else:                      # the first key: all queries of its heads see it
        (k if kind == "k" else v)[B - 1, 0, 0] = math.nan
        rows[B - 1, :G] = True
    return q, k, v, bias, rows


# one token and few keys: one part a row; a long cache: several; 128 queries a workgroup: one set of waves, two, and
# (in fp32) runs
@pytest.mark.parametrize("kind", ["q", "k", "v", "bias"])
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("B,H,Hk,Lq,Lk,hd", [(2, 4, 2, 1, 100, 64), (400, 1, 1, 1, 700, 32), (2, 4, 2, 1, 3000, 64), (2, 4, 2, 130, 130, 64),
                                             (2, 8, 4, 300, 300, 128), (2, 20, 4, 512, 600, 64)])
def test_not_a_number_comes_out(B, H, Hk, Lq, Lk, hd, t, kind):
    from mathbrain.bias_attention import bias_attn_fwd, relative_bias_attention
    q, k, v, bias, _ = inputs(B, H, Hk, Lq, Lk, hd, t, 32, 3)
    q, k, v, bias, rows = with_nan(kind, q, k, v, bias)
    o = relative_bias_attention(q, k, v, bias)
    assert torch.equal(torch.isnan(o).any(-1).cpu(), rows)
    if kind != "v":
        assert torch.isnan(o[rows.cuda()]).all()
    _, lse = bias_attn_fwd(q, k, v, bias, 128, True, 0.125, None, None, Lk - Lq, True)
    assert torch.equal(torch.isnan(lse).cpu(), rows if kind != "v" else torch.zeros_like(rows))


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("L,hd", [(40, 64), (300, 128)])
def test_not_a_number_comes_out_of_the_gradients(L, hd, t):
    """A NaN in head 0's bias: that head's rows have no probabilities, and so have no gradients."""
    from mathbrain.bias_attention import relative_bias_attention
    q, k, v, bias, do = inputs(1, 4, 2, L, L, hd, t, 32, 3)
    q, k, v, bias, _ = with_nan("bias", q, k, v, bias)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, bias)]
    dq, dk, dv, dbias = torch.autograd.grad(relative_bias_attention(*leaves), leaves, do)
    for x in (dq[:, :1], dk[:, :1], dv[:, :1], dbias[0, :1]):
        assert torch.isnan(x).all()
    for x in (dq[:, 1:], dk[:, 1:], dv[:, 1:], dbias[:, 1:]):
        assert torch.isfinite(x).all()


@pytest.mark.parametrize("t", [F32, BF16])
def test_a_position_outside_the_rotation_shows_in_a_decoded_token(t):
    from mathbrain.baseline import rotary_tables
    from mathbrain.qk_norm import qk_norm_rotary
    from mathbrain.bias_attention import relative_bias_attention
    _, k, v, bias, _ = inputs(3, 4, 4, 1, 50, 64, t, 32, 5)
    cos, sin = (x.cuda() for x in rotary_tables(64, 50))
    w = torch.ones(64, device="cuda")
    x = torch.randn(3, 1, 4, 64, device="cuda").to(t)
    q, _ = qk_norm_rotary(x, x, w, w, cos, sin, start=torch.tensor([49, 50, 3], device="cuda"))
    o = relative_bias_attention(q.transpose(1, 2), k, v, bias, lengths=torch.tensor([50, 50, 4], device="cuda"), q_start=torch.tensor([49, 49, 3], device="cuda"))
    assert torch.isnan(o[1]).all() and torch.isfinite(o[0]).all() and torch.isfinite(o[2]).all()


def test_forward_mode_derivatives_are_refused():
    """A dual tensor asks for a tangent without requiring a gradient; an output without one would be
    a derivative of zero."""
    import torch.autograd.forward_ad as fw
    from mathbrain.bias_attention import relative_bias_attention
    q, k, v, bias, _ = inputs(1, 2, 1, 5, 5, 32, F32, 8, 1)
    want = relative_bias_attention(q, k, v, bias)
    with fw.dual_level():
        for i in range(4):
            args = [q, k, v, bias]
            args[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(NotImplementedError, match="jvp"):
                    relative_bias_attention(*args)
        assert torch.equal(relative_bias_attention(q, k, v, bias), want)     # no tangents: as ever


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("low", [-1e5, -3e30])
@pytest.mark.parametrize("Lq,Lk,hd,causal", [(200, 200, 64, True), (150, 300, 128, False), (1, 700, 64, True), (2, 90, 32, False)])
def test_a_whole_table_far_below_zero(Lq, Lk, hd, causal, low, t):
    """What a softmax leaves out, one number added to all scores, does not change the answer: head 0's
    biases are all low, head 1's and head 2's hide one bucket (head 1's others are low too), head 3's are the
    lowest of their type.  Differences within a low head are exact in fp32 (neighbours of one size), so
    the bounds are those of the biases less their head's largest."""
    from mathbrain.bias_attention import relative_bias_attention
    q, k, v, bias, do = inputs(2, 4, 2, Lq, Lk, hd, t, 8, 7)
    bias = bias.float()
    bias[:, 0] = low
    if low == -1e5:    # in steps of fp32's there; at -3e30 a step is more than scores can make up for
        bias[:, 0] += 2.0 ** -7 * torch.arange(8, device="cuda")
    bias[:, 1] = low
    bias[6, 1] = 2 * low
    bias[6, 2] = low
    bias[:, 3] = torch.finfo(F32).min
    rest = bias.double().cpu()
    rest = rest - rest.amax(0)
    hidden = rest < -65536
    assert hidden.sum() == 2
    n, seen = plan(2, Lq, Lk, 8, 16, causal, None, None)
    seen = seen[:, None].expand(2, 4, Lq, Lk) & ~hidden.t()[:, n].transpose(0, 1)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, bias)]
    o = relative_bias_attention(*leaves, max_distance=16, causal=causal)
    got = [o, *torch.autograd.grad(o, leaves, do)]
    for h in range(4):    # a head at a time: their pairs differ
        kv = h // 2
        alone = [x.detach().requires_grad_() for x in (q[:, h:h + 1], k[:, kv:kv + 1], v[:, kv:kv + 1], bias[:, h:h + 1])]
        o1 = relative_bias_attention(*alone, max_distance=16, causal=causal)
        g1 = torch.autograd.grad(o1, alone, do[:, h:h + 1])
        want = definition(*(x.detach() for x in alone[:3]), rest[:, h:h + 1].masked_fill(hidden[:, h:h + 1], 0.0), do[:, h:h + 1], n,
                          seen[:, h], 1 / math.sqrt(hd), t)
        for x, w, name in zip([o1, *g1], want, NAMES):
            near(x, w, name)
        near(got[0][:, h:h + 1], want[0], "o of all heads")
        near(got[1][:, h:h + 1], want[1], "dq of all heads")
        near(got[4][:, h:h + 1], want[4], "dbias of all heads")
