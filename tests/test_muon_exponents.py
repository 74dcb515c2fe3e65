"""muon._exponents is host arithmetic, whatever device tensors are made on by default."""
import torch


def test_default_device():
    from mathbrain.muon import _exponents
    want = _exponents(4, (2.0, -1.5, 0.5))
    _exponents.cache_clear()
    with torch.device("meta"):
        assert _exponents(4, (2.0, -1.5, 0.5)) == want
