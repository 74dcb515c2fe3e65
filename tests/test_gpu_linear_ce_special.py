"""Infinities and NaN in the weights: rows that do not count, or whose loss has no gradient, get none of them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [3, 8, 13, 40, 200, 1300])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_without_a_gradient(N, t, bad):
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    g = torch.Generator("cuda").manual_seed(N)
    w = (torch.randn(300, 64, generator=g, device="cuda") / 8).to(t)
    w[17] = bad
    h = torch.randn(N, 64, generator=g, device="cuda").to(t)
    target = torch.randint(0, 17, (N,), generator=g, device="cuda")
    target[1] = -100
    dloss = torch.ones(N, device="cuda")
    dloss[2] = 0.0
    h.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(h, w, target, reduction="none")
    dh, dw = torch.autograd.grad(loss, [h, w], dloss)
    assert loss[1] == 0 and not dh[1].any() and not dh[2].any()
    # and the others are as the scores of F.linear make them
    s = h.detach().double() @ w.detach().double().t()
    want = torch.logsumexp(s, 1) - s.gather(1, target.clamp(min=0)[:, None])[:, 0]
    assert torch.equal(loss.isfinite()[2:], want.isfinite()[2:])


def test_autocast_leaves_64_bits():
    """As nn.Linear: tensors in 64 bits are not cast, and refused as they are outside of autocast."""
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    h, w, target = torch.randn(4, 8, device="cuda"), torch.randn(9, 8, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.long)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for a, b in ((h.double(), w.double()), (h.double(), w), (h, w.double())):
            with pytest.raises(ValueError, match="float64"):
                linear_cross_entropy(a, b, target)
