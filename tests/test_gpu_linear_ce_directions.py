"""linear_cross_entropy's backward takes the scores of the forward: where the target leads by far, its probability is 1 for scores
of any size, for each way through the kernels that either direction has."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 3, 4, 8, 9, 16, 17, 70])
@pytest.mark.parametrize("D", [64, 128, 1024, 2048])
def test_confident_rows(N, D, t):
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    g = torch.Generator("cuda").manual_seed(N)
    w = F.normalize(torch.randn(600, D, generator=g, device="cuda")).to(t)
    target = torch.randint(0, 600, (N,), generator=g, device="cuda")
    for size in (2.0**12, 2.0**20):
        h = (w[target].float() * size).to(t).requires_grad_()
        loss = linear_cross_entropy(h, w, target, reduction="none")
        dh, = torch.autograd.grad(loss, [h], torch.ones_like(loss))
        # products of different unit vectors stay below 0.7: the others' probabilities are below exp(-0.2 * 4096)
        assert loss.abs().max() < 2.0**-20 and dh.float().norm(dim=1).max() < 2.0**-20, (size, float(loss.abs().max()), float(dh.float().abs().max()))


def test_without_gradients():
    """Calls that no backward follows may take other kernels: the same loss to its roundings (48 of 2^-24 of scores up to 12)."""
    from mathbrain.linear_cross_entropy import linear_cross_entropy
    for N in (1, 5, 8, 40):
        h, w = torch.randn(N, 128, device="cuda").bfloat16().requires_grad_(), (torch.randn(900, 128, device="cuda") / 8).bfloat16()
        target = torch.randint(0, 900, (N,), device="cuda")
        a = linear_cross_entropy(h, w, target, reduction="none")
        with torch.no_grad():
            b = linear_cross_entropy(h, w, target, reduction="none")
        assert (a - b).abs().max() < 48 * 2.0**-24 * 12
