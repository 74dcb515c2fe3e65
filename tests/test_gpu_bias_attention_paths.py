"""relative_bias_attention (mathbrain/bias_attention.py) on the launches that full grids and long walks take, and
its bias gradient to the roundings that the kernels make, against float64 on the GPU, head by head.

Bounds of o, dq, dk and dv are worst cases, element by element.  With e = 2^-24, u half a step of bf16,
2^-8 (0 for fp32), n keys in a row:
 * a score is off by cs = (hd + 8) e (scale |q|.|k| + |bias| + |lse|); its row's denominator by the largest of
   them and n + 16 additions; a probability by dp, the sum of both, of itself;
 * the terms of o are off by dp + u, o by u at its end; delta = dO . o takes o's error; ds = p (dO . v - delta)
   adds dp of itself and hd e |dO|.|v|, and is rounded (u) for the products with k and q.

The bias gradient is a sum of many ds that cancel, and such worst cases would let zeros pass.  What enters it is
known better:
 * delta's error e_i is read off the output itself: dO_i . (o_i - exact o_i).  Every pair of the row takes it with its
   probability, so dbias[n] is off by -sum_i e_i P_i[n], with P_i[n] the row's probability in bucket n, from
   which this test's expectation starts.  In bf16 the kernels put the blocks of 32 x 32 pairs of one bucket right
   (by the row's sum of ds), and take delta from the pairs themselves where a workgroup's 128 queries see at most 128
   keys: those pairs are left out of it.
 * all other errors are roundings to fp32, independent of each other.  A sum of independent errors, each bounded by
   a_k, passes 6 sqrt(sum a_k^2) once in 3e7 times (Hoeffding's bound: 2 exp(-18)); `rest` below adds their squares:
   a pair's score and dO . v, sums of hd terms; a row's denominator and delta; the additions.  Depth d over terms
   of absolute sum A has at most d roundings of e A each, so sqrt(d) e A.  Of blocks of one bucket a lane adds its row's 16 values
   and then the walk's blocks (d = 64 + n / 32); of the others the diagonals are added, 32 rows together (rows that share
   roundings, hence the factor of 32 under the root); a workgroup adds its table's entries, rows' sums and diagonals
   (d = entries / 16 + 40), one launch the workgroups (d = workgroups).
Zeros, and in bf16 a correction left out, have to lie outside these bounds, or the test would say nothing."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
REACH = 128


def inputs(B, H, Hk, Lq, Lk, hd, t, buckets, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, do = (torch.randn(s, generator=g, device="cuda").to(t).transpose(1, 2) for s in
                   ((B, Lq, H, hd), (B, Lk, Hk, hd), (B, Lk, Hk, hd), (B, Lq, H, hd)))
    return q, k, v, torch.randn(buckets, H, generator=g, device="cuda"), do


def plan(B, Lq, Lk, buckets, causal, lengths):
    """starts, the pairs' distances and buckets [1, Lq, Lk], and whether they count [B, Lq, Lk]."""
    from mathbrain.bias_attention import bucket_starts
    side = buckets if causal else buckets // 2
    starts = bucket_starts(side, REACH)
    d = torch.arange(Lk - Lq, Lk, device="cuda")[:, None] - torch.arange(Lk, device="cuda")
    n = sum((d.abs() >= s).long() for s in starts) - 1 + side * (d < 0) * (not causal)
    seen = (d >= 0 if causal else torch.ones_like(d, dtype=torch.bool)).expand(B, Lq, Lk)
    if lengths is not None:
        seen = seen & (torch.arange(Lk, device="cuda") < lengths[:, None, None])
    return starts, d[None], n.clamp(min=0)[None], seen


def by_bucket(x, n, nb):
    """Sums of x [B, Lq, Lk] by its pairs' buckets: [B, Lq, nb]."""
    return torch.zeros(*x.shape[:2], nb, dtype=x.dtype, device=x.device).scatter_add_(2, n.expand(x.shape), x)


def parts(x, size, dim):
    """Sums over runs of `size` along dim."""
    pad = -x.shape[dim] % size
    x = torch.cat([x, x.new_zeros(*x.shape[:dim], pad, *x.shape[dim + 1:])], dim) if pad else x
    return x.unflatten(dim, (-1, size)).sum(dim + 1)


def head(q, k, v, b, do, o_got, lengths, causal, t):
    """One query head in float64, [B, L, hd] each: (value, bound) of o, dq, and this head's share of dk and dv, then
    dbias as (exact, expected, bound, what a correction left out would add)."""
    u = torch.finfo(t).eps / 2 if t == BF16 else 0.0
    B, Lq, hd = q.shape
    Lk, nb, scale = k.shape[1], b.shape[0], hd ** -0.5
    starts, d, n, seen = plan(B, Lq, Lk, nb, causal, lengths)
    q, k, v, b, do, o_got = (x.detach().double() for x in (q, k, v, b, do, o_got))
    live = seen.any(1)[:, :, None]
    k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)
    s = (q @ k.mT * scale + b[n[0]]).masked_fill(~seen, -math.inf)
    lse = s.logsumexp(-1, keepdim=True)
    lse = torch.where(lse.isfinite(), lse, 0.0)
    p = torch.exp(s - lse)
    cs = (hd + 8) * E * (q.abs() @ k.abs().mT * scale + b[n[0]].abs() + lse.abs()) * seen
    rows_off = cs.amax(-1, keepdim=True) + (Lk + 16) * E
    dp = cs + rows_off
    o = p @ v
    o_off = ((dp + u + Lk * E) * p @ v.abs()) * (1 + u) + u * o.abs()
    back, sizes = do @ v.mT, do.abs() @ v.abs().mT
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (back - delta)
    ds_off = (p * (dp * (back.abs() + delta.abs()) + hd * E * (sizes + delta.abs())
                   + (do.abs() * (o_off + hd * E * o.abs())).sum(-1, keepdim=True))) * (1 + dp)
    f_off = ds_off + u * (ds.abs() + ds_off)
    res = [(o, o_off), (ds @ k * scale, (f_off + Lk * E * ds.abs()) @ k.abs() * scale),
           (ds.mT @ q * scale, (f_off + 16 * Lq * E * ds.abs()).mT @ q.abs() * scale),
           (p.mT @ do, ((dp + u + 16 * Lq * E) * p).mT @ do.abs())]

    # the bias gradient
    lo, hi = (0 if causal else -max(starts[-1], 1)), starts[-1]
    w0 = Lk - Lq + torch.arange(Lq, device="cuda")[:, None] // 32 * 32
    jb = torch.arange(Lk, device="cuda") // 32 * 32
    one = ((w0 - jb - 31 >= hi) | (w0 + 31 - jb <= lo))[None]
    ends = (torch.arange(Lq, device="cuda") // 128 * 128 + 128).clamp(max=Lq) + Lk - Lq if causal else torch.full((Lq,), Lk, device="cuda")
    ends = ends.expand(B, Lq) if lengths is None else torch.minimum(ends.expand(B, Lq), lengths[:, None])
    from_pairs = (ends <= 128) & (u > 0)
    err = torch.where(from_pairs, 0.0, (do * (o_got - o)).sum(-1))
    exact = by_bucket(ds, n, nb).sum((0, 1))
    put_right = one & (u > 0)
    left = (err[..., None] * by_bucket(p * ~put_right, n, nb)).sum((0, 1))
    dropped = (err[..., None] * by_bucket(p * put_right, n, nb)).sum((0, 1))
    few = (hd + 8) ** 0.5 / (hd + 8)     # a score's or product's roundings are independent as well
    rows_ind = few * cs.amax(-1, keepdim=True) + (Lk + 16) ** 0.5 * E
    pair = p * ((few * cs + 4 * E) * (back - delta).abs() + hd ** 0.5 * E * (sizes + delta.abs()))
    A1, A2, P, S, S1 = (by_bucket(x, n, nb) for x in (ds.abs() * one, ds.abs() * ~one, p, ds, ds * one))
    a_row = (64 + Lk / 32) ** 0.5 * E * ds.abs().sum(-1, keepdim=True)
    delta_off = hd ** 0.5 * E * (do.abs() * o.abs()).sum(-1, keepdim=True) + (Lk ** 0.5 * E + rows_ind) * (p * back.abs()).sum(-1, keepdim=True) * from_pairs[..., None]
    row = rows_ind * S.abs() + (delta_off + a_row + pair.square().sum(-1, keepdim=True).sqrt()) * P
    entries = hi - lo + 193
    rest = (by_bucket(pair.square(), n, nb) + row.square() + (64 + Lk / 32) * E ** 2 * (A1.square() + 32 * A2.square())).sum((0, 1))
    rest += (entries / 16 + 40) * (E * parts(S1.abs() + A2, 128, 1)).square().sum((0, 1))
    groups = parts(S, 128, 1)
    rest += groups[..., 0].numel() * (E * groups.abs().sum((0, 1))).square()
    bound = 6 * rest.sqrt() + 2 * E * exact.abs() + 1e-30     # a bucket without pairs: 0
    return res, (exact, exact - left, bound, dropped)


def within(got, want, bound, what):
    got = got.detach().double()
    worst = float(((got - want).abs() / bound).max())
    print(f"{what}: {worst:.3f} of its bound", flush=True)
    assert torch.isfinite(got).all() and worst <= 1.0, (what, worst)


def check(size, hd, t, causal, lengths, key_heads=(0,), buckets=32):
    from mathbrain.bias_attention import relative_bias_attention
    B, H, Hk, Lq, Lk = size
    G = H // Hk
    u = torch.finfo(t).eps / 2 if t == BF16 else 0.0
    q, k, v, bias, do = inputs(B, H, Hk, Lq, Lk, hd, t, buckets, sum(size) + hd)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, bias)]
    o = relative_bias_attention(*leaves, max_distance=REACH, causal=causal, lengths=lengths)
    dq, dk, dv, dbias = torch.autograd.grad(o, leaves, do)
    without, = torch.autograd.grad(relative_bias_attention(leaves[0], k, v, bias, max_distance=REACH, causal=causal, lengths=lengths),
                                   leaves[:1], do)
    assert torch.equal(without, dq)
    lost, bounds = [], []
    for hk in key_heads:
        shared = [[0, 0], [0, 0]]
        for h in range(hk * G, (hk + 1) * G):
            res, (exact, expected, bound, dropped) = head(q[:, h], k[:, hk], v[:, hk], bias[:, h], do[:, h], o[:, h], lengths, causal, t)
            for got, (x, off), what in zip((o[:, h], dq[:, h]), res, ("o", "dq")):
                within(got, x, off * (1 + u) + (u + 2 * E) * x.abs() + 1e-30, f"{what} of head {h}")
            for n in range(2):
                for i in range(2):
                    shared[n][i] = shared[n][i] + res[2 + n][i]
            within(dbias[:, h], expected, bound, f"dbias of head {h}")
            assert exact.norm() > 10 * bound.norm()        # zeros would not pass
            lost.append(dropped)
            bounds.append(bound)
        for got, (x, off), what in zip((dk[:, hk], dv[:, hk]), shared, ("dk", "dv")):
            within(got, x, off * (1 + u) + (u + 2 * E) * x.abs() + 1e-30, f"{what} of key head {hk}")
    if t == BF16:   # nor dbias without the correction of the blocks of one bucket
        ratio = float((torch.stack(lost).abs() / torch.stack(bounds)).max())
        print(f"the correction left out: {ratio:.2f} bounds", flush=True)
        assert ratio > 1.5


def some_lengths(B, Lk):
    return torch.tensor([Lk, Lk // 2 + 3, 140, Lk - 1, 1, 64][:B] + [Lk - 7 * i for i in range(max(0, B - 6))], device="cuda")


def sizes_of(size, hd, causal, t, buckets=32):
    """The workspaces, in floats, that tell which launches a size takes: (forward, backward, backward without runs)."""
    from mathbrain import _lib
    B, H, Hk, Lq, Lk = size
    code = _lib.MB_DTYPE_BF16 if t == BF16 else _lib.MB_DTYPE_F32
    fwd = _lib.lib().mb_bias_attn_fwd_workspace(B, H, Hk, Lq, Lk, hd, causal, code) // 4
    bwd = _lib.lib().mb_bias_attn_bwd_workspace(B, H, Hk, Lq, Lk, hd, causal, code, buckets) // 4
    up = lambda x: -(-x // 4) * 4  # noqa: E731
    return fwd, bwd, up(2 * B * H * Lq) + up(H * B * -(-Lq // 128) * buckets)


# more than 512 workgroups in every pass: one set of waves in the forward, no runs, the grid's reversed halves
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd,t", [(64, BF16), (32, BF16), (128, BF16), (64, F32), (32, F32), (128, F32)])
def test_full_grids(hd, t, causal, ragged):
    size = (20, 8, 8, 520, 520) if t == BF16 else (18, 8, 8, 500, 530)
    fwd, bwd, least = sizes_of(size, hd, causal, t)
    assert fwd == 0 and bwd == least
    check(size, hd, t, causal, some_lengths(size[0], size[4]) if ragged else None, key_heads=(0, 7))


# heads that share keys, and walks of more than a thousand keys
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_long_walks_of_full_grids(hd, causal):
    size = (2, 66, 33, 1090, 1090)
    fwd, bwd, least = sizes_of(size, hd, causal, BF16)
    assert fwd == 0 and (causal or bwd == least)
    check(size, hd, BF16, causal, None, key_heads=(0, 16, 32))


# fp32 with two sets of waves in the forward: few workgroups, walks too short for runs (heads of 128: too many workgroups for runs)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd,size", [(32, (3, 8, 4, 400, 400)), (64, (3, 8, 4, 390, 400)), (128, (4, 8, 8, 1100, 1100))])
def test_two_sets_of_waves_in_fp32(hd, size, causal, ragged):
    assert sizes_of(size, hd, causal, F32)[0] == 0
    check(size, hd, F32, causal, some_lengths(size[0], size[4]) if ragged else None)


# walks split into runs, in the queries' pass (whose correction is a launch of its own then) and the keys'
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd,size", [(64, (1, 4, 2, 700, 700)), (64, (2, 12, 4, 500, 800)), (128, (1, 4, 2, 900, 900)), (32, (3, 5, 5, 1300, 1300))])
def test_bias_gradients_of_split_walks(hd, size, causal, t):
    fwd, bwd, least = sizes_of(size, hd, causal, t)
    assert bwd > least
    check(size, hd, t, causal, None, key_heads=range(size[2]))
