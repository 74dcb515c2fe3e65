"""linear_cross_entropy of inputs times powers of two: hidden times a and weight times 1 / a have the same scores, so the loss is
the same, dhidden is divided by a and dweight multiplied, and both follow the losses' gradients, bit for bit as long as nothing
leaves the type's range (nothing rounds otherwise than at the other size)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [3, 16, 40, 200, 1300])
def test_powers_of_two(N, t):
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    g = torch.Generator("cuda").manual_seed(N)
    w = (torch.randn(700, 96, generator=g, device="cuda") / math.sqrt(96)).to(t)
    target = torch.randint(0, 700, (N,), generator=g, device="cuda")
    h = (torch.randn(N, 96, generator=g, device="cuda") + 4 * w[target].float()).to(t)
    dloss = 0.5 + torch.rand(N, generator=g, device="cuda")

    def call(a, c):
        x, y = (h * a).requires_grad_(), (w / a).requires_grad_()
        loss = linear_cross_entropy(x, y, target, reduction="none")
        return loss.detach(), *torch.autograd.grad(loss, [x, y], dloss * c)

    loss, dh, dw = call(1.0, 1.0)
    assert loss.isfinite().all() and dh.abs().max() > 0 and dw.abs().max() > 0
    # small enough that the largest of the products stay in range and the smallest of the results that count are normal numbers
    for a, c in ((2.0**50, 1.0), (2.0**-50, 1.0), (2.0**70, 1.0), (2.0**-70, 1.0), (1.0, 2.0**80), (1.0, 2.0**-60), (2.0**66, 2.0**30), (2.0**-66, 2.0**30)):
        loss_, dh_, dw_ = call(a, c)
        assert torch.equal(loss_, loss), (a, c)
        for x, y, f in ((dh_, dh, c / a), (dw_, dw, c * a)):
            want = y.double() * f
            far = want.abs() < 2.0**-110
            assert torch.equal(x.double()[~far], want[~far]), (a, c, f)
            assert x.isfinite().all()
