"""linear_cross_entropy where scores are large and the target leads by far: the loss and the rows' gradients are zero.

A score and the maximum that is subtracted from it are the same rounded number, so the target's probability is
exp2(0) / sum, off by no more than the sum's and the logarithm's rounding, a few 2^-24, whatever the scores' size."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 5, 8, 16, 40, 64, 200, 1300])
@pytest.mark.parametrize("size", [2.0**6, 2.0**12, 2.0**20])
def test_confident_rows(N, size, t):
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    g = torch.Generator("cuda").manual_seed(N)
    # unit vectors in 96 dimensions: products of different ones stay below 0.6, so the others' probabilities below exp(-0.4 size)
    w = F.normalize(torch.randn(900, 96, generator=g, device="cuda")).to(t)
    target = torch.randint(0, 900, (N,), generator=g, device="cuda")
    h = (w[target].float() * size).to(t)
    s = h.double() @ w.double().t()
    lead = s.gather(1, target[:, None])[:, 0] - s.scatter(1, target[:, None], -1e30).amax(1)
    assert lead.min() > 0.35 * size            # 900 exp(-22) is 2e-7
    h.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(h, w, target, reduction="none")
    dh, dw = torch.autograd.grad(loss, [h, w], torch.ones_like(loss))
    assert loss.abs().max() < 2.0**-20
    # U is at most 2^-22 and 2e-7 there; dh and dw (up to N rows of one word, in truth few) are its products
    assert dh.float().norm(dim=1).max() < 2.0**-20
    assert dw.float().norm(dim=1).max() < 2.0**-20 * size * torch.bincount(target).max()
