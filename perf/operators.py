"""Cases of the comparison transformer's and the trainer's operators: the query/key norm with the
rotation (``qk``), attention with a learned bias by distance buckets (``attn``) and the global
gradient norm with clipping (``clip``).

Each has a plain form in elementary torch operations (``own`` false), the framework's call
(``own`` true) and its definition in 64 bits (``exact``).
"""
import math

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases -------------------------------------------------------------------------------

def _qk(batch, length, heads, kv_heads, head_dim, dtype, train, name=None):
    c = dict(op="qk", batch=batch, length=length, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             dtype=dtype, train=train)
    return c if name is None else dict(c, name=name)


def _attn(batch, queries, keys, heads, kv_heads, head_dim, dtype, train, causal=True, ragged=False,
          buckets=32, reach=128, name=None):
    c = dict(op="attn", batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads,
             head_dim=head_dim, dtype=dtype, train=train, causal=causal, ragged=ragged,
             buckets=buckets, reach=reach)
    return c if name is None else dict(c, name=name)


def _clip(vocab, dim, layers, dtype, in_place, name=None):
    c = dict(op="clip", vocab=vocab, dim=dim, layers=layers, dtype=dtype, in_place=in_place)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one new token for each of 16 sequences: latency
        _qk(16, 1, 8, 8, 64, "bf16", False, name="qk one token"),
        # the training batch of the model's attention, 56 chunks of 512
        _qk(56, 512, 8, 8, 64, "bf16", True, name="qk train 56x512"),
        # full precision, an odd length, keys shared by two query heads
        _qk(6, 1021, 10, 5, 32, "f32", True, name="qk train f32 odd"),
        # the long chunks, wide heads
        _qk(16, 4096, 8, 8, 128, "bf16", True, name="qk train 16x4096"),
        # one new token against caches of different lengths
        _attn(16, 1, 4096, 8, 8, 64, "bf16", False, ragged=True, name="attn one token"),
        # reading a prompt: forward alone, an odd length, wide shared heads
        _attn(3, 2047, 2047, 8, 2, 128, "bf16", False, name="attn prompt"),
        # the training batch of 56 chunks of 512
        _attn(56, 512, 512, 8, 8, 64, "bf16", True, name="attn train 56x512"),
        # full precision, both directions, padded rows, odd sizes
        _attn(5, 333, 333, 6, 6, 32, "f32", True, causal=False, ragged=True, name="attn train f32 odd"),
        # the comparison model's longest chunks
        _attn(4, 4096, 4096, 8, 8, 64, "bf16", True, name="attn train 4x4096"),
        # a small model below its norm's bound: the norm is taken, nothing is scaled
        _clip(1000, 128, 2, "f32", True, name="clip small in place"),
        # the six-layer model's gradients, clipped into the buffer that its optimiser reads
        _clip(50257, 512, 6, "f32", False, name="clip model"),
        # bf16 gradients clipped into fp32 master gradients
        _clip(20011, 512, 6, "bf16", False, name="clip bf16 to master"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 5, 8])
    return kv * rng.choice([1, 1, 2, 4]) if kv < 5 else kv, kv


def draw(rng):
    op = rng.choice(["qk", "qk", "attn", "attn", "attn", "clip", "clip"])
    if op == "qk":
        heads, kv = _heads(rng)
        hd = rng.choice([32, 64, 128])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        if rng.random() < 0.25:
            return _qk(_log_int(rng, 1, 300), 1, heads, kv, hd, dtype, False)
        length = _log_int(rng, 2, 4096)
        batch = _log_int(rng, 1, max(1, min(64, 50_000_000 // (length * (heads + kv) * hd))))
        return _qk(batch, length, heads, kv, hd, dtype, True)
    if op == "attn":
        heads, kv = _heads(rng)
        hd = rng.choice([32, 64, 128])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        buckets, reach = rng.choice([(32, 128), (32, 128), (16, 64), (64, 500), (31, 200)])
        kind = rng.choice(["token", "prompt", "train", "train"])
        if kind == "token":
            keys = _log_int(rng, 1, 16384)
            batch = _log_int(rng, 1, max(1, min(64, 400_000 // keys)))
            return _attn(batch, rng.choice([1, 1, 1, 2, 5]), keys, heads, kv, hd, dtype, False, ragged=True,
                         buckets=buckets, reach=reach)
        causal = rng.random() < 0.75
        if not causal:
            buckets += buckets % 2
        length = _log_int(rng, 3, 4096)
        most = 250_000_000 if dtype == "bf16" else 60_000_000
        batch = _log_int(rng, 1, max(1, min(64, most // (length * length * heads) * 64 // hd)))
        if length * length * heads * hd > 64 * most:
            length = int(math.sqrt(64 * most / (heads * hd)))
        keys = length
        if kind == "prompt" and causal:
            length = max(1, length - rng.randrange(0, length // 2 + 1))  # earlier tokens are in the cache
        return _attn(batch, length, keys, heads, kv, hd, dtype, kind == "train", causal=causal,
                     ragged=kind == "train" and rng.random() < 0.4, buckets=buckets, reach=reach)
    return _clip(_log_int(rng, 100, 50257), rng.choice([64, 96, 130, 256, 384, 512]), rng.randrange(1, 7),
                 rng.choice(["f32", "bf16"]), rng.random() < 0.4)


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, mul=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * mul).to(dtype)


def _shapes(case):
    """The parameter shapes of the slot model: embedding, its layers' attention and feed-forward, norms."""
    d, v = case["dim"], case["vocab"]
    ff = 256 * ((int(8 * d / 3) + 255) // 256)
    layer = [(d,), (d, d), (d, d), (d, d), (d, d), (d, 64), (d,), (d,), (d,), (d,), (d,), (ff, d), (d, ff), (ff, d)]
    return [(v, d)] + layer * case["layers"] + [(d,)]


def prepare(case, seed):
    g = _gen(seed)
    t = DTYPES[case.get("dtype")]
    s = dict(case=case)
    if case["op"] == "qk":
        b, n, h, hk, hd = (case[x] for x in ("batch", "length", "heads", "kv_heads", "head_dim"))
        train = case["train"]
        s["q"] = _randn(g, b, n, h, hd, dtype=t, mul=1.3).requires_grad_(train)
        s["k"] = _randn(g, b, n, hk, hd, dtype=t, mul=0.8).requires_grad_(train)
        s["q_weight"] = (1 + 0.2 * _randn(g, hd)).requires_grad_(train)
        s["k_weight"] = (1 + 0.2 * _randn(g, hd)).requires_grad_(train)
        # one table of cosines and sines, which the model keeps
        rate = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        angle = torch.arange(4096, dtype=torch.float64, device="cuda")[:, None] * rate
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        # a step's rows stand at the ends of their sequences, a chunk's at the start
        s["start"] = (torch.zeros(b, dtype=torch.int32, device="cuda") if train else
                      torch.randint(0, 4096 - n + 1, (b,), generator=g, device="cuda", dtype=torch.int32))
        if train:
            s["dq"] = _randn(g, b, n, h, hd, dtype=t)
            s["dk"] = _randn(g, b, n, hk, hd, dtype=t)
    elif case["op"] == "attn":
        b, nq, nk, h, hk, hd = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
        train = case["train"]
        # projections as the model has them, [batch, length, heads, head_dim], seen per head
        s["q"] = _randn(g, b, nq, h, hd, dtype=t).transpose(1, 2).requires_grad_(train)
        s["k"] = _randn(g, b, nk, hk, hd, dtype=t).transpose(1, 2).requires_grad_(train)
        s["v"] = _randn(g, b, nk, hk, hd, dtype=t).transpose(1, 2).requires_grad_(train)
        # near keys weigh more than far ones
        fall = torch.linspace(1.0, -1.0, case["buckets"], device="cuda")[:, None]
        s["bias"] = (fall + 0.5 * _randn(g, case["buckets"], h)).to(t).requires_grad_(train)
        s["lengths"] = None
        s["start"] = nk - nq
        if case["ragged"]:
            low = max(nq, nk // 2)
            s["lengths"] = torch.randint(min(low, nk), nk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            if not train:
                s["start"] = s["lengths"] - nq  # the newest tokens of each cache
        if train:
            s["do"] = _randn(g, b, nq, h, hd, dtype=t).transpose(1, 2)
    else:
        shapes = _shapes(case)
        flat = _randn(g, sum(math.prod(x) for x in shapes), dtype=t, mul=0.01)
        at = [0] + torch.tensor([math.prod(x) for x in shapes]).cumsum(0).tolist()
        s["flat"] = flat
        s["grads"] = [flat[p:p + math.prod(x)].view(x) for p, x in zip(at, shapes)]
        if case["in_place"]:
            s["max_norm"] = 1000.0  # above the norm: a step that needs no clipping
            s["params"] = [torch.nn.Parameter(torch.empty_like(x)) for x in s["grads"]]
            for p, x in zip(s["params"], s["grads"]):
                p.grad = x
        else:
            s["max_norm"] = 1.0
            s["master"] = torch.empty(flat.numel(), dtype=torch.float32, device="cuda")
            s["out"] = [s["master"][p:p + math.prod(x)].view(x) for p, x in zip(at, shapes)]
    return s


# ---- the framework's calls ----------------------------------------------------------------

def _own(s):
    op = s["case"]["op"]
    if op == "qk":
        from mathbrain.qk_norm import qk_norm_rotary
        q, k = qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], EPS, s["start"])
        if not s["case"]["train"]:
            return [q, k]
        leaves = [s[x] for x in ("q", "k", "q_weight", "k_weight")]
        return [q, k, *torch.autograd.grad([q, k], leaves, [s["dq"], s["dk"]])]
    if op == "attn":
        from mathbrain.bias_attention import relative_bias_attention
        o = relative_bias_attention(s["q"], s["k"], s["v"], s["bias"], max_distance=s["case"]["reach"],
                                    causal=s["case"]["causal"], lengths=s["lengths"], q_start=s["start"])
        if not s["case"]["train"]:
            return [o]
        return [o, *torch.autograd.grad(o, [s[x] for x in ("q", "k", "v", "bias")], s["do"])]
    if s["case"]["in_place"]:
        from mathbrain.grad_clip import clip_grad_norm_
        return [clip_grad_norm_(s["params"], s["max_norm"]), s["flat"]]
    from mathbrain.grad_clip import clip_gradients
    return [clip_gradients(s["grads"], s["max_norm"], out=s["out"]), s["master"]]


# ---- plain forms --------------------------------------------------------------------------

def _turn(x, c, s):
    """The pairs (x[..., 2i], x[..., 2i+1]) turned by the angles whose cosines and sines are c and s."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)


def _plain_norm(x, w, c, s, dy):
    xf = x.detach().float()
    r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
    n = xf * r
    y = _turn(n * w.detach(), c, s).to(x.dtype)
    if dy is None:
        return y, None, None
    g = _turn(dy.float(), c, -s)
    gw = g * w.detach()
    dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), (g * n).sum((0, 1, 2))


def _plain_qk(s):
    n = s["case"]["length"]
    at = s["start"][:, None] + torch.arange(n, device="cuda")
    c, sn = s["cos"][at][:, :, None, :], s["sin"][at][:, :, None, :]
    q, dq, dwq = _plain_norm(s["q"], s["q_weight"], c, sn, s.get("dq"))
    k, dk, dwk = _plain_norm(s["k"], s["k_weight"], c, sn, s.get("dk"))
    return [q, k, dq, dk, dwq, dwk] if s["case"]["train"] else [q, k]


def _bucket(n, count, reach):
    """The bucket of each distance n >= 0: exact below count // 2, by logarithms up to reach. In 64
    bits, with a nudge that no distance comes near, so that a border's own distance is above it."""
    near = count // 2
    far = torch.log(n.clamp(min=near).double() / near) / math.log(reach / near) * (count - near)
    return torch.where(n < near, n, (near + torch.floor(far + 1e-9).long()).clamp(max=count - 1))


def _plain_attn(s):
    case = s["case"]
    b, nq, nk, h, hk, hd = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    count, reach, causal, t = case["buckets"], case["reach"], case["causal"], s["q"].dtype
    scale = 1 / math.sqrt(hd)
    q = s["q"].detach().float()
    k, v = (s[x].detach().float().repeat_interleave(h // hk, dim=1) for x in ("k", "v"))
    start = s["start"].long()[:, None, None] if torch.is_tensor(s["start"]) else s["start"]
    j = torch.arange(nk, device="cuda")
    dist = start + torch.arange(nq, device="cuda")[None, :, None] - j  # [1 or b, nq, nk]
    # the bias of each distance, clamped to where it no longer changes: [h, 2 * reach + 1]
    each = torch.arange(-reach, reach + 1, device="cuda")
    if causal:
        bucket = _bucket(each.clamp(min=0), count, reach)
    else:
        bucket = _bucket(each.abs(), count // 2, reach) + (each < 0) * (count // 2)
    by_distance = s["bias"].detach().float()[bucket].t()
    bias = by_distance[:, dist.clamp(-reach, reach) + reach].transpose(0, 1)  # [1 or b, h, nq, nk]
    left = torch.ones(1, nq, nk, dtype=torch.bool, device="cuda")
    if causal:
        left = dist >= 0
    if s["lengths"] is not None:
        left = left & (j < s["lengths"][:, None, None])
    left = left[:, None]
    x = (torch.matmul(q, k.transpose(2, 3)) * scale + bias).masked_fill(~left, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p, v)
    if not case["train"]:
        return [o.to(t)]
    do = s["do"].float()
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(-1, keepdim=True))
    shared = (b, hk, h // hk, nk, hd)
    dv = torch.matmul(p.transpose(2, 3), do).view(shared).sum(2)
    dk = (torch.matmul(ds.transpose(2, 3), q) * scale).view(shared).sum(2)
    dq = torch.matmul(ds, k) * scale
    # the sums along the diagonals: rows padded to nq + nk and read one longer, so that each begins a
    # column earlier than the one before it
    wide = nq + nk + 1
    rows = torch.nn.functional.pad(ds.sum(0), (0, nq)).view(h, -1)
    along = torch.nn.functional.pad(rows, (0, nq)).view(h, nq, wide).sum(1)
    # column c of them holds j - i = c, or j - i = c - wide where that came around
    c = torch.arange(wide, device="cuda")
    away = start - torch.where(c < nk, c, c - wide)
    at = bucket[away.clamp(-reach, reach) + reach]
    dbias = torch.matmul((torch.arange(count, device="cuda")[:, None] == at).float(), along.t())
    return [o.to(t), dq.to(t), dk.to(t), dv.to(t), dbias.to(t)]


def _plain_clip(s):
    squares = torch.stack([x.float().square().sum() for x in s["grads"]])
    norm = squares.sum().sqrt()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    if s["case"]["in_place"]:
        [x.mul_(factor) for x in s["grads"]]
        return [norm, s["flat"]]
    [y.copy_(x.float() * factor) for x, y in zip(s["grads"], s["out"])]
    return [norm, s["master"]]


def run(state):
    if own:
        return _own(state)
    return {"qk": _plain_qk, "attn": _plain_attn, "clip": _plain_clip}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "qk":
        n = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        table = 4 * case["length"] * case["head_dim"]
        return {"bytes": (4 if case["train"] else 2) * n * size + table, "flops": (22 if case["train"] else 8) * n}
    if case["op"] == "attn":
        b, nq, nk, h, hk, hd = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
        keys = (max(nq, nk // 2) + nk) / 2 if case["ragged"] else nk  # the mean length
        if not case["causal"]:
            pairs = nq * keys
        elif case["train"]:
            pairs = nq * (nq + 1) / 2 - (nq - keys) * (nq - keys + 1) / 2
        else:
            pairs = sum(max(0.0, keys - i) for i in range(nq))
        q, kv = b * h * nq * hd * size, b * hk * keys * hd * size
        moved = 4 * q + 4 * kv if case["train"] else 2 * q + 2 * kv
        return {"bytes": moved, "flops": (14 if case["train"] else 4) * hd * pairs * b * h}
    n = sum(math.prod(x) for x in _shapes(case))
    return {"bytes": n * size if case["in_place"] else n * (size + 4), "flops": 3 * n}


# ---- the definitions in 64 bits ------------------------------------------------------------

def _exact_qk(s):
    case = s["case"]
    b, n, hd = case["batch"], case["length"], case["head_dim"]
    at = (s["start"].long().view(b, 1) + torch.arange(n, device="cuda").view(1, n)).view(-1)
    spin = torch.complex(s["cos"].double(), s["sin"].double())[at].view(b, n, 1, hd // 2)
    got, grads = [], []
    for x, w, dy in (("q", "q_weight", "dq"), ("k", "k_weight", "dk")):
        xd, wd = (s[y].detach().double().clone().requires_grad_(case["train"]) for y in (x, w))
        unit = xd / (xd.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * wd
        y = torch.view_as_real(torch.view_as_complex(unit.unflatten(-1, (-1, 2))) * spin).flatten(-2)
        got.append(y.detach())
        if case["train"]:
            grads.append(torch.autograd.grad(y, [xd, wd], s[dy].double()))
    return got + [x[i] for i in (0, 1) for x in grads]


def _exact_bucket(n, count, reach):
    """By whole numbers: the bucket is near + k, with k the largest whose border reach^k near^(m - k)
    is at most n^m, m = count - near."""
    near = count // 2
    if n < near:
        return n
    m = count - near
    return near + max(k for k in range(m) if n ** m >= reach ** k * near ** (m - k))


def _exact_attn(s):
    case = s["case"]
    b, nq, nk, h, hk, hd = (case[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    if b * h * nq * nk > 1_500_000_000:
        return None
    count, reach = case["buckets"], case["reach"]
    half = count if case["causal"] else count // 2
    table = torch.tensor([_exact_bucket(n, half, reach) for n in range(reach + 1)], device="cuda")
    i = (s["start"].long() if torch.is_tensor(s["start"]) else torch.full((b,), s["start"], device="cuda"))
    i = (i.view(b, 1) + torch.arange(nq, device="cuda")).view(b, nq, 1)
    j = torch.arange(nk, device="cuda").view(1, 1, nk)
    if s["lengths"] is None and not torch.is_tensor(s["start"]):
        i = i[:1]
    bucket = table[(i - j).abs().clamp(max=reach)]
    if case["causal"]:
        seen = (j <= i).expand(i.shape[0], nq, nk)
    else:
        bucket = bucket + torch.where(j > i, half, 0)
        seen = torch.ones_like(bucket, dtype=torch.bool)
    if s["lengths"] is not None:
        seen = seen & (j < s["lengths"].view(b, 1, 1))
    wants = case["train"]
    q, k, v = (s[x].detach().double().clone().requires_grad_(wants) for x in ("q", "k", "v"))
    bias = s["bias"].detach().double().t().contiguous()[:, bucket].transpose(0, 1)
    grouped = q.reshape(b, hk, (h // hk) * nq, hd)
    score = (grouped @ k.transpose(-1, -2).contiguous()).reshape(b, h, nq, nk) / hd ** 0.5 + bias
    weight = torch.softmax(score.masked_fill(~seen[:, None], -1e300), -1) * seen[:, None].any(-1, keepdim=True)
    o = (weight.reshape(b, hk, (h // hk) * nq, nk) @ v).reshape(b, h, nq, hd)
    if not wants:
        return [o.detach()]
    dq, dk, dv, ds = torch.autograd.grad(o, [q, k, v, score], s["do"].double())
    dbias = torch.stack([(ds * (bucket == c)[:, None]).sum((0, 2, 3)) for c in range(count)])
    return [o.detach(), dq, dk, dv, dbias]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "qk":
        return _exact_qk(s)
    if case["op"] == "attn":
        return _exact_attn(s)
    flat = s["flat"].double()
    norm = torch.linalg.vector_norm(flat)
    return [norm, flat * min(1.0, s["max_norm"] / (float(norm) + 1e-6))]
