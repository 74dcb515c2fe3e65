"""The argument checks of the cross entropy's and the Muon step's entry points: they run on the host before
anything is launched (no GPU needed)."""
import ctypes
import math

import pytest
import torch  # noqa: F401  (the library binds to torch's HIP runtime)

P = 1 << 20     # any aligned non-null address: the refused calls never use it


@pytest.fixture(scope="module")
def lib():
    from mathbrain import _lib
    return _lib.lib()


def message(lib):
    return lib.mb_last_error().decode()


def ce(**fields):
    from mathbrain.linear_cross_entropy import _ARGS
    names = ("hidden weight hidden_ld weight_ld target target_bytes ignore_index N V D dtype reduction loss lse count dloss "
             "dhidden dweight workspace workspace_bytes").split()
    a = dict.fromkeys(names, P) | dict(hidden_ld=64, weight_ld=64, target_bytes=8, ignore_index=-1, N=100, V=1000, D=64, dtype=1,
                                       reduction=1, workspace_bytes=1 << 40)
    assert set(fields) <= set(names)
    return _ARGS.pack(*(a | fields).values())


@pytest.mark.parametrize("bad,said", [
    (dict(N=0), "N=0"), (dict(N=(1 << 28) + 1), "N=268435457"), (dict(V=0), "V=0"), (dict(V=(1 << 24) + 1), "V=16777217"),
    (dict(D=0), "D=0"), (dict(D=65537), "D=65537"), (dict(dtype=2), "dtype=2"), (dict(reduction=3), "reduction=3"),
    (dict(reduction=-1), "reduction=-1"), (dict(target_bytes=2), "target_bytes=2"), (dict(hidden=0), "null"), (dict(weight=0), "null"),
    (dict(target=0), "null"), (dict(lse=0), "null"), (dict(count=0), "null"), (dict(hidden_ld=63), "63 elements apart"),
    (dict(weight_ld=(1 << 22) + 1), "4194305 elements apart")])
def test_cross_entropy_refusals(lib, bad, said):
    for name in ("mb_linear_ce_fwd", "mb_linear_ce_bwd"):
        assert getattr(lib, name)(ce(**bad), None) < 0
        assert said in message(lib) and name in message(lib)
    assert lib.mb_linear_ce_workspace(ce(**bad), 0) == -1


def test_cross_entropy_refusals_of_one_direction(lib):
    from mathbrain import _lib
    assert lib.mb_linear_ce_fwd(None, None) < 0 and "null args" in message(lib)
    for name, bad, rc, said in (("fwd", dict(loss=0), -1, "null"), ("bwd", dict(dloss=0), -1, "null"),
                                ("fwd", dict(workspace=P + 16), -1, "multiple of 256"), ("bwd", dict(workspace=P + 16), -1, "multiple of 256"),
                                ("fwd", dict(workspace=0), _lib.MB_ERR_WORKSPACE, "workspace"),
                                ("bwd", dict(workspace_bytes=64), _lib.MB_ERR_WORKSPACE, "workspace of 64 bytes"),
                                ("fwd", dict(N=1 << 28, V=1 << 24), _lib.MB_ERR_UNSUPPORTED, "too many"),
                                ("bwd", dict(N=1 << 28, V=1 << 24), _lib.MB_ERR_UNSUPPORTED, "too many"),
                                ("bwd", dict(N=1 << 28, D=1 << 16, hidden_ld=1 << 16, weight_ld=1 << 16), _lib.MB_ERR_UNSUPPORTED, "too many")):
        assert getattr(lib, "mb_linear_ce_" + name)(ce(**bad), None) == rc and said in message(lib), (name, bad, message(lib))


def test_cross_entropy_workspaces(lib):
    """No copies of bf16 operands that the products can read as they are; U's pieces have a bound."""
    small = lib.mb_linear_ce_workspace(ce(), 0)
    assert small < 100 * 1000 * 2
    assert lib.mb_linear_ce_workspace(ce(weight_ld=65), 0) > small + 1000 * 64 * 2 - 1
    assert lib.mb_linear_ce_workspace(ce(hidden=P + 2), 0) > small + 100 * 64 * 2 - 1
    large = lib.mb_linear_ce_workspace(ce(N=28672, V=50257, D=512, hidden_ld=512, weight_ld=512), 1)
    assert 512 << 20 < large < 1400 << 20


def muon(each=None, **fields):
    from mathbrain.muon import _ARGS, _MATRIX
    good = dict(src=P, dst=2 * P, momentum=3 * P, rows=8, cols=16, src_dtype=0, dst_dtype=0, momentum_dtype=0, rate=1.0)
    table = b"".join(_MATRIX.pack(*(good | m).values()) for m in (each if each is not None else [{}]))
    muon.keep = ctypes.create_string_buffer(table, len(table) or 1)
    a = dict(matrices=ctypes.addressof(muon.keep), count=len(table) // _MATRIX.size, steps=5, is_step=1, nesterov=1, a=3.0, b=-4.0, c=2.0,
             eps=1e-7, x_exponent=14, a_exponent=14, b_exponent=13, lr=0.1, momentum=0.9, weight_decay=0.0, workspace=P << 4,
             workspace_bytes=1 << 40)
    assert set(fields) <= set(a)
    return _ARGS.pack(*(a | fields).values())


@pytest.mark.parametrize("matrices,fields,said", [
    (None, dict(count=-1), "count=-1"), (None, dict(matrices=0), "count=1"), (None, dict(steps=0), "steps=0"), (None, dict(steps=101), "steps=101"),
    (None, dict(x_exponent=16), "exponent of 16"), (None, dict(b_exponent=-15), "exponent of -15"), (None, dict(eps=-1.0), "eps=-1"),
    (None, dict(eps=math.nan), "eps="), ([dict(rows=-1)], {}, "-1 x 16"), ([dict(rows=1 << 16, cols=1 << 15)], {}, "65536 x 32768"),
    ([dict(rows=40000, cols=40000)], {}, "40000 x 40000"), ([{}, dict(dst=5 * P, momentum=6 * P, src_dtype=2)], {}, "matrix 1: dtype"),
    ([dict(momentum_dtype=-1)], {}, "matrix 0: dtype")])
def test_muon_refusals(lib, matrices, fields, said):
    assert lib.mb_muon_run(muon(matrices, **fields), None) < 0 and said in message(lib) and "mb_muon_run" in message(lib)
    assert lib.mb_muon_workspace(muon(matrices, **fields)) == -1


@pytest.mark.parametrize("matrices,fields,rc,said", [
    ([dict(src=0)], {}, -1, "null"), ([dict(dst=0)], {}, -1, "null"), ([dict(momentum=0)], {}, -1, "null"),
    ([{}, dict(dst=9 * P, momentum=10 * P)], dict(workspace=(P << 4) + 8), -1, "multiple of 256"),
    ([{}], dict(workspace=0), -3, "workspace"), ([{}], dict(workspace_bytes=100), -3, "workspace of 100 bytes"),
    ([{}, {}], {}, -1, "share memory"), ([dict(momentum=2 * P)], {}, -1, "share memory"), ([dict(src=2 * P + 4)], {}, -1, "share memory"),
    ([dict(momentum=2 * P + 8 * 16 * 4 - 1)], {}, -1, "share memory")])
def test_muon_refusals_of_memory(lib, matrices, fields, rc, said):
    assert lib.mb_muon_run(muon(matrices, **fields), None) == rc and said in message(lib), message(lib)


def test_muon_nothing_to_do(lib):
    assert lib.mb_muon_run(None, None) < 0 and "null args" in message(lib)
    assert lib.mb_muon_run(muon([]), None) == 0
    assert lib.mb_muon_run(muon([dict(rows=0, src=0, dst=0, momentum=0)]), None) == 0
    assert lib.mb_muon_workspace(muon([])) >= 0


def test_exponents_of_the_iterates():
    """Bounds on the iterates: the largest values, scaled, stay within fp16, whatever the spectrum."""
    from mathbrain.muon import COEFFICIENTS, _exponents
    for steps, (a, b, c) in ((5, COEFFICIENTS), (1, (1.5, -0.5, 0.0)), (9, (1.875, -1.25, 0.375)), (3, (2.0, 0.0, 0.0))):
        ex, ea, eb = _exponents(steps, (a, b, c))
        s = torch.cat((torch.linspace(0, 1, 100001, dtype=torch.float64), torch.logspace(-9, 0, 1000, dtype=torch.float64)))
        most = 0.0
        for _ in range(steps):
            second = b * s**2 + c * s**4
            assert s.max() * 2.0**ex < 65504 / 1.5 and s.max() ** 2 * 2.0**ea < 65504 / 1.5 and second.abs().max() * 2.0**eb < 65504 / 1.5
            most = max(most, float(s.max()))
            s = (s * (a + second)).abs()
        assert most * 2.0**ex > 2**13 or ex == 15      # and no more bits are given away than that takes
    with pytest.raises(ValueError, match="grow"):
        _exponents(5, (9.0, 0.0, 0.0))
