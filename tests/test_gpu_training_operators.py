"""The rotation, the cross entropy without logits, the clipping and Muon together, as a training program runs them:
the comparison model and the slot model against float64, and several steps against the same steps in float64.

Tolerance of the fp32 models as in the tests of their other options: norm-wise, 1e-4 for gradients (a layer's products sum
at most 384 terms in fp32, 384 * 2^-24 = 2.3e-5 of the terms' sizes in the worst order, a tenth of that in a blocked one, and
two layers pass about ten of them on)."""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

V, D, HEADS, LAYERS = 97, 128, 4, 2


def model(**options):
    from mathbrain.baseline import RoPETransformerLM
    torch.manual_seed(0)
    return RoPETransformerLM(V, D, LAYERS, HEADS, max_seq_len=256, dropout=0.0, **options).cuda()


def norm(x, w):
    return w * x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()


def definition(p, x, cos, sin, layout):
    """The model's logits in float64 from the parameters p and the tables [L, d / 2]."""
    B, L = x.shape
    hd, d = D // HEADS, 2 * cos.shape[1]
    i = torch.arange(d // 2)
    a, b = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + d // 2)
    hidden = torch.tril(torch.ones(L, L)) == 0

    def turn(t):
        y = t.clone()
        y[..., a] = t[..., a] * cos - t[..., b] * sin
        y[..., b] = t[..., a] * sin + t[..., b] * cos
        return y

    h = p["embed.weight"][x]
    for n in range(LAYERS):
        w = {k[len(f"layers.{n}."):]: v for k, v in p.items() if k.startswith(f"layers.{n}.")}
        y = norm(h, w["attn_norm.weight"])
        q, k, v = ((y @ w[f"attn.w{c}.weight"].T).view(B, L, HEADS, hd).transpose(1, 2) for c in "qkv")
        s = turn(q) @ turn(k).transpose(-1, -2) / math.sqrt(hd)
        o = s.masked_fill(hidden, -math.inf).softmax(-1) @ v
        h = h + o.transpose(1, 2).reshape(B, L, D) @ w["attn.wo.weight"].T
        y = norm(h, w["ffn_norm.weight"])
        h = h + (F.silu(y @ w["ffn.w1.weight"].T) * (y @ w["ffn.w3.weight"].T)) @ w["ffn.w2.weight"].T
    return norm(h, p["final_norm.weight"]) @ p["embed.weight"].T


def orthogonal(g):
    x = g / (g.norm() + 1e-7)
    x = x.t() if x.shape[0] > x.shape[1] else x
    for _ in range(5):
        y = x @ x.t()
        x = 3.4445 * x + (-4.7750 * y + 2.0315 * y @ y) @ x
    return x.t() if g.shape[0] > g.shape[1] else x


def batch(seed, B=3, L=70):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(0, V, (B, L + 1), generator=g)
    x, t = x[:, :-1], x[:, 1:].clone()
    t[torch.rand(B, L, generator=g) < 0.2] = -1
    return x, t


OPTIONS = [dict(), dict(rope_layout="half"), dict(rope_dims=8, rope_scaling=dict(scaling="linear", factor=2.0)),
           dict(rope_layout="half", rope_dims=16, rope_scaling=dict(scaling="yarn", factor=4.0, trained=64))]


@pytest.mark.parametrize("options", OPTIONS)
def test_steps_against_float64(options):
    """Three steps: the losses, the clipped norms and the parameters follow the definition's.  Muon's update has entries up to
    1, so what gradients are off by (1e-4 of the largest, above) moves a matrix by at most lr * 1e-4 * its update's slope in
    them, of the order of the slope of X / |X| (1 / the smallest kept singular value): held to 2e-3 of the movement."""
    from mathbrain.grad_clip import clip_grad_norm_
    from mathbrain.muon import Muon
    m = model(**options)
    p = {k: v.detach().cpu().double() for k, v in m.named_parameters()}
    matrices = [v for k, v in m.named_parameters() if v.dim() == 2 and "embed" not in k]
    rest = [v for k, v in m.named_parameters() if v.dim() != 2 or "embed" in k]
    muon, sgd = Muon(matrices, lr=0.02, weight_decay=0.1), torch.optim.SGD(rest, lr=0.1)
    momenta = {k: torch.zeros_like(v) for k, v in p.items()}
    begin = copy.deepcopy(p)
    for step in range(3):
        x, t = batch(step)
        loss = m(x.cuda(), targets=t.cuda())
        muon.zero_grad(), sgd.zero_grad()
        loss.backward()
        q = {k: v.clone().requires_grad_() for k, v in p.items()}
        cos, sin = (y[:x.shape[1]].cpu().double() for y in (m.rope_cos, m.rope_sin))
        want = F.cross_entropy(definition(q, x, cos, sin, options.get("rope_layout", "interleaved")).view(-1, V), t.flatten(),
                               ignore_index=-1)
        want.backward()
        assert abs(float(loss) - float(want)) < 2e-5 * float(want) * (1 if step == 0 else 20)
        total = math.sqrt(sum(float(v.grad.square().sum()) for v in q.values()))
        got = clip_grad_norm_(m.parameters(), 0.5 * total)
        assert abs(float(got) - total) < 1e-4 * total * (1 if step == 0 else 20)
        for k, v in m.named_parameters():
            g = q[k].grad * (0.5 * total / (total + 1e-6) if total > 0.5 * total else 1.0)
            assert float((v.grad.cpu().double() - g).norm()) < 1e-4 * total * (1 if step == 0 else 20), k
            if v.dim() == 2 and "embed" not in k:
                momenta[k] = 0.95 * momenta[k] + g
                p[k] = p[k] * (1 - 0.02 * 0.1) - 0.02 * math.sqrt(max(1.0, g.shape[0] / g.shape[1])) * orthogonal(g + 0.95 * momenta[k])
            else:
                p[k] = p[k] - 0.1 * g
        muon.step(), sgd.step()
        if step == 0:
            for k, v in m.named_parameters():
                assert float((v.detach().cpu().double() - p[k]).norm()) < 2e-3 * float((p[k] - begin[k]).norm()), k


@pytest.mark.parametrize("kind", ["rope", "slot"])
def test_targets_give_the_loss_of_the_logits(kind):
    """forward(targets=...) against the cross entropy of the same model's logits, and its gradients."""
    if kind == "rope":
        m, x, more = model(), batch(5)[0], {}
    else:
        from mathbrain.model import SlotTransformerLM
        from mathbrain.synthetic import make_batch
        torch.manual_seed(0)
        m = SlotTransformerLM(V, 64, 2, 2, N=16, dropout=0.0, max_hl=512.0, attn_precision="fp32").cuda()
        d = make_batch(3, 70, V, 16, 60, seed=2, max_hl=512.0)
        x, more = d["x"], dict(unique_slots=d["unique"].cuda(), c_base=d["c_base"].cuda(), pad_mask=(d["unique"] >= 0).cuda())
    t = batch(6, *x.shape)[1].cuda()
    names, params = zip(*m.named_parameters())
    logits = m(x.cuda(), **more)
    plain = F.cross_entropy(logits.double().view(-1, V), t.flatten(), ignore_index=-1)
    want = torch.autograd.grad(plain, params)
    loss = m(x.cuda(), **more, targets=t)
    got = torch.autograd.grad(loss, params)
    assert abs(float(loss) - float(plain)) < 1e-6 * float(plain)
    total = math.sqrt(sum(float(g.double().square().sum()) for g in want))
    for k, a, b in zip(names, got, want):      # atomics in the slot model's sums: not the same twice
        assert float((a - b).norm()) < 1e-5 * total, k
    with torch.autocast("cuda", dtype=torch.bfloat16):
        low = m(x.cuda(), **more, targets=t)
        assert low.dtype == torch.float32 and abs(float(low) - float(plain)) < 3e-2 * float(plain)
    low.backward()
    assert all(p.grad is not None and p.grad.dtype == torch.float32 and p.grad.isfinite().all() for p in params)
    ignored = m(x.cuda(), **more, targets=torch.where(t == -1, 7, t), ignore_index=7)
    assert ignored.isfinite()


def test_a_step_in_bf16_throughout():
    from mathbrain.grad_clip import clip_grad_norm_
    from mathbrain.muon import Muon
    m = model().bfloat16()
    matrices = [v for k, v in m.named_parameters() if v.dim() == 2 and "embed" not in k]
    opt = Muon(matrices, lr=0.01)
    for step in range(2):
        x, t = batch(step)
        before = [v.detach().clone() for v in matrices]
        loss = m(x.cuda(), targets=t.cuda())
        loss.backward()
        clip_grad_norm_(m.parameters(), 1.0)
        opt.step()
        assert loss.isfinite() and all(v.isfinite().all() and not torch.equal(v, b) for v, b in zip(matrices, before))


def test_a_whole_step_captured():
    """Forward, backward, clipping and Muon in one graph, replayed with new tokens and checked against eager steps."""
    from mathbrain.grad_clip import clip_gradients
    from mathbrain.muon import muon_step

    def build():
        m = model()
        names = [k for k, v in m.named_parameters() if v.dim() == 2 and "embed" not in k]
        params = dict(m.named_parameters())
        return m, params, [params[k] for k in names], [torch.zeros_like(params[k]) for k in names]

    def step(m, params, matrices, momenta, x, t):
        loss = m(x, targets=t)
        grads = torch.autograd.grad(loss, list(params.values()))
        clip_gradients(grads, 0.5)
        at = {id(p): g for p, g in zip(params.values(), grads)}
        muon_step([p.data for p in matrices], [at[id(p)] for p in matrices], momenta, 0.02)
        return loss

    x, t = (y.cuda() for y in batch(0))
    captured, eager = build(), build()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*build(), x, t)                    # everything is loaded and allocated once
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(*captured, x, t)
    for i in range(3):
        a, b = batch(10 + i)
        x.copy_(a), t.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*eager, x, t)
        torch.cuda.synchronize()
        assert torch.allclose(loss, want, rtol=1e-5 * 4**i)
        # the library's products may sum in another order within the graph: the matrices agree to that
        for p, q in zip(captured[2], eager[2]):
            assert float((p - q).norm()) < 1e-3 * 4**i * float(q.norm())


def test_calls_on_two_streams_at_once():
    """Each operator on two streams, in turn and without a wait between them, gives what it gives alone (all sums have a
    fixed order: bit for bit)."""
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    from mathbrain.muon import orthogonalize
    from mathbrain.rotary import apply_rotary, rotary_tables
    cos, sin = rotary_tables(32, 300, device="cuda")
    made = []
    for seed in range(2):
        g = torch.Generator("cuda").manual_seed(seed)
        made.append([torch.randn(1500, 128, device="cuda", generator=g) * 0.3, torch.randn(901, 128, device="cuda", generator=g) * 0.3,
                     torch.randint(0, 901, (1500,), device="cuda", generator=g), torch.randn(260, 190, device="cuda", generator=g),
                     torch.randn(2, 300, 3, 32, device="cuda", generator=g)])

    def work(h, w, t, m, q):
        h, w, q = (x.detach().requires_grad_() for x in (h, w, q))
        loss = linear_cross_entropy(h, w, t)
        a, b = apply_rotary(q, q, cos, sin)
        return [loss, *torch.autograd.grad(loss, [h, w]), a, b, *torch.autograd.grad((a * b.detach()).sum(), [q]), orthogonalize(m)]

    alone = [work(*x) for x in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = [[], []]
    for _ in range(4):
        for s, x, out in zip(streams, made, got):
            with torch.cuda.stream(s):
                out.append(work(*x))
    torch.cuda.synchronize()
    for want, runs in zip(alone, got):
        assert all(torch.equal(x, y) for run in runs for x, y in zip(want, run))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_hidden_and_weight_are_one_tensor(t):
    """F.cross_entropy(x x^T): x's gradient is the sum of both.  Scores of 48 products of values below 4 * 0.25: off by
    48 * 2^-24 * |h| |w| at most, far below the outputs' own step: 2^-8 of the largest for bf16 (two roundings of half a step and
    their sum's), 1e-5 of it for fp32."""
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    torch.manual_seed(5)
    x = (torch.randn(70, 48, device="cuda") * 0.25).to(t).requires_grad_()
    target = torch.randint(0, 70, (70,), device="cuda")
    y = x.detach().double().requires_grad_()
    want = F.cross_entropy(y @ y.T, target)
    loss = linear_cross_entropy(x, x, target)
    assert abs(float(loss) - float(want)) < 1e-5 * float(want)
    got, = torch.autograd.grad(loss, [x])
    exact, = torch.autograd.grad(want, [y])
    tol = 1e-5 if t == torch.float32 else 3 * 2.0**-8
    assert float((got.double() - exact).abs().max()) < tol * float(exact.abs().max())
