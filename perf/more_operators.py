"""Cases of what a training step does around its layers: the rotation of queries and keys
(``rotary``), the softmax cross entropy of the tied output matrix without its logits (``loss``),
the orthogonalised updates of the weight matrices (``ortho``) and the optimiser's step that
applies them (``muon``).

Each has a plain form in elementary torch operations (``own`` false), the framework's call
(``own`` true) and its definition in 64 bits (``exact``).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
IGNORED = -1


# ---- cases -------------------------------------------------------------------------------

def _named(c, name):
    return c if name is None else dict(c, name=name)


def _rotary(batch, length, heads, kv_heads, head_dim, turned, layout, at, dtype, train, scaled=False, name=None):
    return _named(dict(op="rotary", batch=batch, length=length, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                       turned=turned, layout=layout, at=at, dtype=dtype, train=train, scaled=scaled), name)


def _loss(rows, vocab, dim, dtype, train, reduction="mean", ignored=0.0, name=None):
    return _named(dict(op="loss", rows=rows, vocab=vocab, dim=dim, dtype=dtype, train=train, reduction=reduction,
                       ignored=ignored), name)


def _ortho(count, rows, cols, dtype, name=None):
    return _named(dict(op="ortho", count=count, rows=rows, cols=cols, dtype=dtype), name)


def _muon(layers, dim, scales, dtype, name=None):
    return _named(dict(op="muon", layers=layers, dim=dim, scales=scales, dtype=dtype), name)


def listed():
    return [
        # one new token for each of 16 sequences: latency
        _rotary(16, 1, 8, 8, 64, 64, "interleaved", "rows", "bf16", False, name="rotary one token"),
        # the training batch of the comparison model's attention, 56 chunks of 512
        _rotary(56, 512, 8, 8, 64, 64, "interleaved", "zero", "bf16", True, name="rotary train 56x512"),
        # full precision, documents packed into odd rows, half of each head turned, shared keys
        _rotary(6, 1021, 10, 5, 64, 32, "half", "tokens", "f32", True, name="rotary packed f32"),
        # reading long prompts with rescaled angles, wide heads
        _rotary(2, 16384, 8, 2, 128, 128, "half", "rows", "bf16", False, scaled=True, name="rotary prompt 16384"),
        # a small model's step: latency
        _loss(128, 1000, 128, "bf16", True, name="loss small"),
        # scoring the next token of 16 sequences
        _loss(16, 50257, 512, "bf16", False, reduction="none", name="loss score 16"),
        # the training batch of 56 chunks of 512 on the whole vocabulary
        _loss(28672, 50257, 512, "bf16", True, name="loss train 56x512"),
        # full precision, odd sizes, padded targets
        _loss(4093, 20011, 384, "f32", True, reduction="sum", ignored=0.3, name="loss train f32 odd"),
        # the attention matrices of a small model
        _ortho(8, 128, 128, "bf16", name="ortho 8 of 128"),
        # a wide feed-forward's matrices
        _ortho(4, 2816, 1024, "bf16", name="ortho 4 of 2816x1024"),
        # full precision, odd sizes
        _ortho(3, 777, 1234, "f32", name="ortho f32 odd"),
        # all matrices of the six-layer model, with momentum and weight decay
        _muon(6, 512, 64, "f32", name="muon model"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "loss", "loss", "loss", "ortho", "ortho", "muon"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "rotary":
        kv = rng.choice([1, 2, 3, 4, 5, 8])
        heads = kv * rng.choice([1, 1, 2, 4]) if kv < 5 else kv
        hd = rng.choice([32, 64, 80, 96, 128])
        turned = rng.choice([hd, hd, hd // 2, hd // 4])
        layout, scaled = rng.choice(["interleaved", "half"]), rng.random() < 0.3
        if rng.random() < 0.25:
            return _rotary(_log_int(rng, 1, 300), rng.choice([1, 1, 2, 5]), heads, kv, hd, turned, layout, "rows", dtype,
                           False, scaled)
        length = _log_int(rng, 2, 16384)
        batch = _log_int(rng, 1, max(1, min(64, 30_000_000 // (length * (heads + kv) * hd))))
        return _rotary(batch, length, heads, kv, hd, turned, layout, rng.choice(["zero", "rows", "tokens"]), dtype,
                       rng.random() < 0.7, scaled)
    if op == "loss":
        dim = rng.choice([64, 96, 101, 130, 256, 384, 512, 768, 1024, 2048])
        vocab = _log_int(rng, 30, 131072)
        most = min(28672 * 50257 * 512 // (vocab * dim), 1_400_000_000 // vocab)
        rows = _log_int(rng, 1, max(1, min(32768, most)))
        return _loss(rows, vocab, dim, dtype, rng.random() < 0.75, rng.choice(["mean", "mean", "sum", "none"]),
                     rng.choice([0.0, 0.0, 0.1, 0.5]))
    if op == "ortho":
        rows, cols = _log_int(rng, 8, 2816), _log_int(rng, 8, 2816)
        small, large = min(rows, cols), max(rows, cols)
        cost = small * small * (4 * large + 2 * small) * STEPS
        return _ortho(_log_int(rng, 1, max(1, min(40, 4 * 10**11 // cost))), rows, cols, dtype)
    return _muon(rng.randrange(1, 7), rng.choice([64, 128, 130, 256, 384, 512]), rng.choice([16, 32, 64]), dtype)


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, mul=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * mul).to(dtype)


def _angles(case, rows):
    """The table of cosines and sines that the model keeps, from angles in 64 bits; rescaled ones have
    their slow frequencies divided by 8 and the fast ones left, with a ramp between."""
    d = case["turned"]
    rate = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    if case["scaled"]:
        turns = 2048 * rate / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        rate = rate * keep + rate / 8 * (1 - keep)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def _shapes(case):
    """The matrices of the slot model's layers: attention, counters' projection and feed-forward."""
    d = case["dim"]
    ff = 256 * ((int(8 * d / 3) + 255) // 256)
    return ([(d, d)] * 4 + [(d, case["scales"])] + [(ff, d), (d, ff), (ff, d)]) * case["layers"]


def _views(flat, shapes):
    sizes = [math.prod(x) for x in shapes]
    return [p.view(x) for p, x in zip(flat.split(sizes), shapes)]


def _low_rank(g, count, rows, cols):
    """Matrices with the spectra of momenta: a few strong directions over weak noise."""
    k = max(1, min(rows, cols) // 8)
    fall = 2.0 ** -torch.linspace(0, 5, k, device="cuda")
    strong = torch.bmm(_randn(g, count, rows, k) * fall, _randn(g, count, k, cols)) / math.sqrt(k)
    return (strong + 0.05 * _randn(g, count, rows, cols)) * 1e-3


def prepare(case, seed):
    g = _gen(seed)
    t = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "rotary":
        b, n, h, hk, hd = (case[x] for x in ("batch", "length", "heads", "kv_heads", "head_dim"))
        train = case["train"]
        s["q"] = _randn(g, b, n, h, hd, dtype=t).requires_grad_(train)
        s["k"] = _randn(g, b, n, hk, hd, dtype=t).requires_grad_(train)
        table = 2 * 16384
        s["cos"], s["sin"] = _angles(case, table)
        s["start"] = 0
        if case["at"] == "rows":      # each row goes on from its own position
            s["start"] = torch.randint(0, table - n + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        elif case["at"] == "tokens":  # documents packed into rows: positions begin again within them
            first = torch.rand(b, n, generator=g, device="cuda") < 4 / n
            first[:, 0] = True
            at = torch.arange(n, device="cuda")
            s["start"] = (at - torch.where(first, at, 0).cummax(1).values).int()
        if train:
            s["dq"] = _randn(g, b, n, h, hd, dtype=t)
            s["dk"] = _randn(g, b, n, hk, hd, dtype=t)
    elif case["op"] == "loss":
        n, v, d = case["rows"], case["vocab"], case["dim"]
        train = case["train"]
        weight = _randn(g, v, d, mul=1 / math.sqrt(d))
        target = torch.randint(0, v, (n,), generator=g, device="cuda")
        # the rows lean towards their targets, some hardly and some strongly
        lean = 12 * torch.rand(n, 1, generator=g, device="cuda")
        s["hidden"] = (_randn(g, n, d) + lean * weight[target]).to(t).requires_grad_(train)
        s["weight"] = weight.to(t).requires_grad_(train)
        left = torch.rand(n, generator=g, device="cuda") < case["ignored"]
        left[0] = False  # a batch has a target at least
        s["target"] = target.masked_fill(left, IGNORED)
        if train:
            shape = (n,) if case["reduction"] == "none" else ()
            s["dloss"] = 0.5 + torch.rand(shape, generator=g, device="cuda")
    elif case["op"] == "ortho":
        s["matrices"] = list(_low_rank(g, case["count"], case["rows"], case["cols"]).to(t).unbind())
    else:
        shapes = _shapes(case)
        n = sum(math.prod(x) for x in shapes)
        s["flat"] = _randn(g, n, dtype=t, mul=0.03)
        s["flat_momentum"] = _randn(g, n, dtype=t, mul=2e-3)
        grads = torch.cat([_low_rank(g, 1, *x).flatten() for x in shapes]).to(t)
        s["params"], s["momenta"], s["grads"] = (_views(x, shapes) for x in (s["flat"], s["flat_momentum"], grads))
    return s


# ---- the framework's calls ----------------------------------------------------------------

def _own(s):
    case = s["case"]
    op = case["op"]
    if op == "rotary":
        from mathbrain.rotary import apply_rotary
        q, k = apply_rotary(s["q"], s["k"], s["cos"], s["sin"], start=s["start"], layout=case["layout"])
        if not case["train"]:
            return [q, k]
        return [q, k, *torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])]
    if op == "loss":
        from mathbrain.linear_cross_entropy import linear_cross_entropy
        loss = linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORED,
                                    reduction=case["reduction"])
        if not case["train"]:
            return [loss]
        return [loss, *torch.autograd.grad(loss, [s["hidden"], s["weight"]], s["dloss"])]
    if op == "ortho":
        from mathbrain.muon import orthogonalize
        return orthogonalize(s["matrices"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    from mathbrain.muon import muon_step
    muon_step(s["params"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY,
              steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    return [s["flat"], s["flat_momentum"]]


# ---- plain forms --------------------------------------------------------------------------

def _turn(x, c, s, layout):
    """The pairs of the first 2 * c.shape[-1] channels turned by the angles whose cosines and sines are c
    and s; the other channels as they are."""
    d = 2 * c.shape[-1]
    xf, rest = x[..., :d].float(), x[..., d:]
    if layout == "interleaved":
        a, b = xf[..., 0::2], xf[..., 1::2]
        y = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = xf[..., :d // 2], xf[..., d // 2:]
        y = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((y.to(x.dtype), rest), dim=-1) if rest.shape[-1] else y.to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    at = torch.arange(case["length"], device="cuda")[None]
    if case["at"] == "rows":
        at = at + s["start"][:, None]
    elif case["at"] == "tokens":
        at = s["start"]
    c, sn = s["cos"][at][:, :, None, :], s["sin"][at][:, :, None, :]
    got = [_turn(s[x].detach(), c, sn, case["layout"]) for x in ("q", "k")]
    if case["train"]:
        got += [_turn(s[x], c, -sn, case["layout"]) for x in ("dq", "dk")]
    return got


def _plain_loss(s):
    case = s["case"]
    h, w, target = s["hidden"].detach().float(), s["weight"].detach().float(), s["target"]
    rows = torch.arange(case["rows"], device="cuda")
    counts = target != IGNORED
    at = torch.where(counts, target, 0)
    logits = torch.matmul(h, w.t())
    top = logits.amax(1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(1, keepdim=True)
    each = torch.where(counts, (torch.log(total) + top)[:, 0] - logits[rows, at], 0.0)
    n = counts.sum()
    if case["reduction"] == "none":
        loss = each
    else:
        loss = each.double().sum()
        loss = (loss / n if case["reduction"] == "mean" else loss).float()
    if not case["train"]:
        return [loss]
    per_row = s["dloss"] / n if case["reduction"] == "mean" else s["dloss"]
    p = p / total
    p[rows, at] -= 1
    p = p * torch.where(counts, per_row, 0.0)[:, None]
    return [loss, torch.matmul(p, w).to(s["hidden"].dtype), torch.matmul(p.t(), h).to(s["weight"].dtype)]


def _orthogonal(g):
    """Matrices [count, rows, cols] in 32 bits."""
    tall = g.shape[1] > g.shape[2]
    x = g.transpose(1, 2).contiguous() if tall else g
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = torch.bmm(x, x.transpose(1, 2))
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.transpose(1, 2) if tall else x


def _by_shape(matrices):
    """Indices of the matrices of each shape: those of one shape go through the products together."""
    found = {}
    for i, x in enumerate(matrices):
        found.setdefault(tuple(x.shape), []).append(i)
    return found.values()


def _orthogonal_all(matrices):
    got = [None] * len(matrices)
    for at in _by_shape(matrices):
        for i, y in zip(at, _orthogonal(torch.stack([matrices[i] for i in at]).float())):
            got[i] = y
    return got


def _plain_ortho(s):
    return [x.to(y.dtype, memory_format=torch.contiguous_format) for x, y in zip(_orthogonal_all(s["matrices"]), s["matrices"])]


def _plain_muon(s):
    grads = [x.float() for x in s["grads"]]
    new = [x.float() * MOMENTUM + y for x, y in zip(s["momenta"], grads)]
    turned = _orthogonal_all([y + MOMENTUM * x for x, y in zip(new, grads)])
    for p, m, x, o in zip(s["params"], s["momenta"], new, turned):
        m.copy_(x)
        p.copy_(p.float() * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * o)
    return [s["flat"], s["flat_momentum"]]


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "loss": _plain_loss, "ortho": _plain_ortho, "muon": _plain_muon}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------

def _products(rows, cols):
    """Operations of the iterations' products; of the two symmetric ones half the entries suffice."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        n = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"])
        ways = 2 if case["train"] else 1
        return {"bytes": 2 * ways * n * case["head_dim"] * size + 4 * case["length"] * case["turned"],
                "flops": 3 * ways * n * case["turned"]}
    if case["op"] == "loss":
        n, v, d = case["rows"], case["vocab"], case["dim"]
        ways = 2 if case["train"] else 1
        return {"bytes": ways * (n + v) * d * size + 8 * n, "flops": (6 if case["train"] else 2) * n * v * d}
    if case["op"] == "ortho":
        n = case["count"] * case["rows"] * case["cols"]
        return {"bytes": 2 * n * size, "flops": case["count"] * _products(case["rows"], case["cols"])}
    shapes = _shapes(case)
    return {"bytes": 5 * sum(math.prod(x) for x in shapes) * size, "flops": sum(_products(*x) for x in shapes)}


# ---- the definitions in 64 bits ------------------------------------------------------------

def _exact_rotary(s):
    case = s["case"]
    b, n, d, hd = (case[x] for x in ("batch", "length", "turned", "head_dim"))
    start = s["start"] if torch.is_tensor(s["start"]) else torch.zeros(b, dtype=torch.int64, device="cuda")
    at = start.long().view(b, -1)
    if case["at"] != "tokens":
        at = at + torch.arange(n, device="cuda").view(1, n)
    spin = torch.complex(s["cos"].double(), s["sin"].double())[at.reshape(-1)].view(b, n, 1, d // 2)
    # channel 2i or i holds the real part of pair i, 2i + 1 or i + d / 2 its imaginary part
    i = torch.arange(d // 2, device="cuda")
    real, imaginary = (2 * i, 2 * i + 1) if case["layout"] == "interleaved" else (i, i + d // 2)

    def turned(x, z):
        y = x.detach().double().clone()
        w = torch.complex(y[..., real], y[..., imaginary]) * z
        y[..., real], y[..., imaginary] = w.real, w.imag
        return y

    got = [turned(s["q"], spin), turned(s["k"], spin)]
    if case["train"]:
        got += [turned(s["dq"], spin.conj()), turned(s["dk"], spin.conj())]
    return got


def _exact_loss(s):
    case = s["case"]
    n, train = case["rows"], case["train"]
    w = s["weight"].detach().double()
    used = s["target"].ne(IGNORED)
    share = torch.ones((), dtype=torch.float64, device="cuda")
    if case["reduction"] == "mean":
        share = share / used.sum()
    each, dh, dw = [], [], torch.zeros_like(w)
    step = max(1, 400_000_000 // case["vocab"])
    for lo in range(0, n, step):
        rows = slice(lo, lo + step)
        h, t, use = s["hidden"].detach()[rows].double(), s["target"][rows].clamp(min=0), used[rows]
        score = torch.log_softmax(h @ w.t(), -1)
        each.append(-score.gather(1, t[:, None])[:, 0] * use)
        if train:
            up = s["dloss"][rows] if case["reduction"] == "none" else s["dloss"]
            weight = torch.where(use, up.double() * share, 0.0)[:, None]
            ds = score.exp_().mul_(weight).scatter_add_(1, t[:, None], -weight)
            dh.append(ds @ w)
            dw += ds.t() @ h
    each = torch.cat(each)
    loss = each if case["reduction"] == "none" else each.sum() * share
    return [loss, torch.cat(dh), dw] if train else [loss]


def _exact_orthogonal(g):
    """One matrix, from the side with fewer rows; a polynomial of x x^T a step."""
    x = g.double()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (torch.linalg.norm(x) + EPS)
    a, b, c = COEFFICIENTS
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        y = x @ x.t()
        x = (a * eye + (b * eye + c * y) @ y) @ x
    return (x.t() if flip else x).contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s)
    if case["op"] == "loss":
        return _exact_loss(s)
    if case["op"] == "ortho":
        return [_exact_orthogonal(x) for x in s["matrices"]]
    params, momenta = [], []
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        m = MOMENTUM * m.double() + g.double()
        o = _exact_orthogonal(g.double() + MOMENTUM * m)
        scale = LR * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        params.append((p.double() * (1 - LR * DECAY) - scale * o).flatten())
        momenta.append(m.flatten())
    return [torch.cat(params), torch.cat(momenta)]
