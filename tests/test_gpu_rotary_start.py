"""The forms that apply_rotary's start takes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_whole_numbers():
    from mathbrain.rotary import apply_rotary, rotary_tables
    cos, sin = rotary_tables(32, 20, device="cuda")
    q = torch.randn(2, 4, 2, 32, device="cuda")
    want = apply_rotary(q, q, cos, sin, 3)[0]
    for start in (np.int32(3), np.int64(3), torch.full((2,), 3, device="cuda")):
        assert torch.equal(apply_rotary(q, q, cos, sin, start)[0], want)
    for start in (3.0, 2.7, "3", None, 2**63, -2**63 - 1, 2**100):
        with pytest.raises(ValueError, match="start"):
            apply_rotary(q, q, cos, sin, start)
