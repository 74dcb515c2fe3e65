"""The workspace of mb_muon_run: bounded for lists of any length, and what it takes for a step in groups."""
import ctypes

import pytest
import torch


def workspace(shapes, is_step=1):
    from mathbrain import _lib
    from mathbrain.muon import _ARGS, _MATRIX
    table = b"".join(_MATRIX.pack((3 * i + 1) << 36, (3 * i + 2) << 36, (3 * i + 3) << 36, r, c, 0, 0, 0, 1.0) for i, (r, c) in enumerate(shapes))
    held = ctypes.create_string_buffer(table, len(table))
    return _lib.lib().mb_muon_workspace(_ARGS.pack(ctypes.addressof(held), len(shapes), 5, is_step, 1, 3.4, -4.7, 2.0, 1e-7, 14, 14, 13, 0.1, 0.9,
                                                   0.0, 0, 0))


def test_bounded():
    one = workspace([(8192, 4096)])
    assert 8 * 4096 * (8192 + 4096) + 4 * 8192 * 4096 <= one < 600 << 20
    assert workspace([(8192, 4096)] * 5) > 4 * one           # together
    for shapes in ([(8192, 4096)] * 100, [(8192, 4096), (512, 512)] * 50, [(300, 200)] * 30000, [(1, 1)] * 100000):
        assert workspace(shapes) < (5 << 30), len(shapes)
    assert workspace([(32768, 60000)]) > 20 << 30             # a single matrix takes what it takes


@pytest.mark.gpu
def test_a_list_that_goes_in_groups():
    """Twelve matrices of 8192 x 4096 with small ones: more than one group, each checked; memory that two groups share is not mixed up.
    The tolerance is that of the other tests of orthogonalize: 2 * 4^5 * 4 * 2^-23 of the result's norm."""
    from mathbrain.muon import muon_step, orthogonalize
    g = torch.Generator("cuda").manual_seed(1)
    shapes = [(8192, 4096), (4096, 8192)] * 6 + [(300, 200), (20, 5000), (64, 64)]
    mats = [torch.randn(s, generator=g, device="cuda") for s in shapes]
    assert workspace(shapes) < workspace(shapes[:6]) * 2      # no room for all at once

    def definition(x):
        x = x.double()
        flip = x.shape[0] > x.shape[1]
        x = x.t() if flip else x
        x = x / (x.norm() + 1e-7)
        for _ in range(5):
            y = x @ x.t()
            x = 3.4445 * x + (-4.7750 * y + 2.0315 * y @ y) @ x
        return x.t() if flip else x

    out = orthogonalize(mats)
    params, momenta = [torch.zeros_like(x) for x in mats], [torch.zeros_like(x) for x in mats]
    muon_step(params, mats, momenta, 1.0, momentum=0.9, nesterov=False)
    for x, y, p, m in zip(mats, out, params, momenta):
        want = definition(x)
        room = 2 * 4.0**5 * 4 * 2.0**-23 * float(want.norm())
        assert float((y.double() - want).norm()) <= room, tuple(x.shape)
        scale = max(1.0, x.shape[0] / x.shape[1]) ** 0.5
        assert float((p.double() / -scale - want).norm()) <= room and torch.equal(m, x), tuple(x.shape)
