"""forward(targets=...) of models whose lm_head is not the plain linear layer that they begin with: the loss of their own logits."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


class Doubled(nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


@pytest.mark.parametrize("kind", ["plain", "bias", "subclass", "hook", "pre_hook", "module"])
def test_loss_of_the_logits(kind):
    from mathbrain.baseline import RoPETransformerLM
    torch.manual_seed(0)
    m = RoPETransformerLM(60, 64, 1, 2, max_seq_len=16, dropout=0.0)
    if kind == "bias":
        m.lm_head = nn.Linear(64, 60)
    elif kind == "subclass":
        m.lm_head = Doubled(64, 60, bias=False)
    elif kind == "module":
        m.lm_head = nn.Sequential(nn.Linear(64, 32), nn.Linear(32, 60))
    elif kind == "hook":
        m.lm_head.register_forward_hook(lambda mod, x, y: 3 * y)
    elif kind == "pre_hook":
        m.lm_head.register_forward_pre_hook(lambda mod, x: (3 * x[0],))
    m = m.cuda()
    x = torch.randint(0, 60, (3, 10), device="cuda")
    t = torch.randint(-1, 60, (3, 10), device="cuda", dtype=torch.int32)
    want = F.cross_entropy(m(x).double().view(-1, 60), t.long().flatten(), ignore_index=-1)
    loss = m(x, targets=t)
    assert abs(float(loss) - float(want)) < 1e-5 * float(want)
    loss.backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())
