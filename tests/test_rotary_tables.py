"""rotary.rotary_tables against the formulas, on the CPU."""
import math

import pytest
import torch


def test_plain_tables():
    from mathbrain.rotary import rotary_tables
    cos, sin = rotary_tables(8, 100001, theta=500.0)
    assert cos.shape == (100001, 4) and cos.dtype == torch.float32
    for t in (0, 1, 77, 100000):
        for i in range(4):
            a = t * 500.0 ** (-2 * i / 8)
            assert abs(float(cos[t, i]) - math.cos(a)) < 2.0**-24 and abs(float(sin[t, i]) - math.sin(a)) < 2.0**-24


def test_scaled_tables():
    from mathbrain.rotary import rotary_tables
    angle = lambda t: torch.atan2(t[1], t[0])[1].double()       # of position 1
    plain = angle(rotary_tables(64, 2))
    assert (angle(rotary_tables(64, 2, scaling="linear", factor=4.0)) - plain / 4).abs().max() < 1e-7
    ntk = angle(rotary_tables(64, 2, scaling="ntk", factor=4.0))
    assert abs(ntk[0] - plain[0]) < 1e-7 and abs(ntk[-1] * 4 / plain[-1] - 1) < 1e-5
    c, s = rotary_tables(64, 2, scaling="yarn", factor=4.0, trained=2048)
    assert ((c[1] ** 2 + s[1] ** 2).sqrt() - (0.1 * math.log(4.0) + 1)).abs().max() < 1e-6
    turns = 2048 * plain / (2 * math.pi)
    ratio = angle((c, s)) / plain
    assert ((ratio - 1).abs()[turns > 40] < 1e-5).all() and ((ratio * 4 - 1).abs()[turns < 0.8] < 1e-5).all()
    assert (ratio[1:] <= ratio[:-1] + 1e-6).all()


@pytest.mark.parametrize("bad", [dict(dim=7), dict(dim=0), dict(scaling="other"), dict(factor=0.5), dict(factor=math.inf),
                                 dict(scaling="yarn"), dict(scaling="ntk", dim=2)])
def test_refusals(bad):
    from mathbrain.rotary import rotary_tables
    with pytest.raises(ValueError):
        rotary_tables(**(dict(dim=64, positions=8) | bad))


def test_refusals_of_the_library():
    """On the host, before anything is launched."""
    from mathbrain import _lib
    from mathbrain.rotary import _ARGS
    lib = _lib.lib()
    P = 1 << 20
    names = ("q k q0 q1 q2 k0 k1 k2 cos sin table_rows start start_bytes start_per_token start0 B L H Hk hd turned layout "
             "inverse dtype q_out k_out").split()
    good = dict.fromkeys(names, P) | dict(q0=512, q1=128, q2=64, k0=512, k1=128, k2=64, table_rows=64, start=0, start_bytes=4,
                                          start_per_token=0, start0=0, B=2, L=4, H=2, Hk=2, hd=64, turned=64, layout=0,
                                          inverse=0, dtype=0)
    for bad, said in ((dict(hd=0), "head_dim=0"), (dict(hd=8193), "head_dim=8193"), (dict(turned=63), "63 of 64"),
                      (dict(turned=66), "66 of 64"), (dict(layout=2), "layout=2"), (dict(dtype=2), "dtype=2"),
                      (dict(B=-1), "B=-1"), (dict(H=0, Hk=0), "H=0"), (dict(H=1 << 17), "H=131072"),
                      (dict(start=P, start_bytes=2), "start_bytes=2"), (dict(start0=61), "pass the table"),
                      (dict(table_rows=-1), "table_rows"), (dict(q=0), "null"), (dict(sin=0), "null"), (dict(k_out=0), "null")):
        assert lib.mb_apply_rotary(_ARGS.pack(*(good | bad).values()), None) == _lib.MB_ERR_INVALID_ARGUMENT, bad
        assert said in lib.mb_last_error().decode(), (bad, lib.mb_last_error())
    assert lib.mb_apply_rotary(None, None) < 0
    assert lib.mb_apply_rotary(_ARGS.pack(*(good | dict(B=0, q=0)).values()), None) == 0
