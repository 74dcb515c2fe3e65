"""Outputs that share memory with something else of the call: refused on the host by the loss's and the rotation's entry points,
before anything is launched (no GPU needed)."""
import pytest
import torch  # noqa: F401  (the library binds to torch's HIP runtime)

M = 1 << 30     # tensors this far apart share nothing


@pytest.fixture(scope="module")
def lib():
    from mathbrain import _lib
    return _lib.lib()


def refused(lib, rc):
    from mathbrain import _lib
    said = lib.mb_last_error().decode()
    return rc == _lib.MB_ERR_INVALID_ARGUMENT and ("shared with an input" in said or "share memory" in said), (rc, said)


def loss(N, dtype, **fields):
    from mathbrain.linear_cross_entropy import _ARGS
    a = dict(hidden=1 * M, weight=2 * M, hidden_ld=70, weight_ld=64, target=3 * M, target_bytes=8, ignore_index=-1, N=N, V=1000, D=64,
             dtype=dtype, reduction=0, loss=4 * M, lse=5 * M, count=6 * M, dloss=7 * M, dhidden=8 * M, dweight=9 * M, workspace=10 * M,
             workspace_bytes=1 << 29)
    assert set(fields) <= set(a)
    return _ARGS.pack(*(a | fields).values())


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("N", [3, 40, 100, 3000])
def test_loss(lib, N, dtype):
    size = 4 if dtype == 0 else 2
    last = ((N - 1) * 70 + 64) * size - 1
    for bad in (dict(loss=M), dict(loss=M + last - last % 4), dict(lse=2 * M + 4), dict(count=3 * M + 8 * N - 4), dict(lse=4 * M),
                dict(count=5 * M + 8 * N - 4), dict(workspace=M), dict(workspace=4 * M), dict(loss=10 * M + 512), dict(hidden=10 * M + 4096)):
        ok, why = refused(lib, lib.mb_linear_ce_fwd(loss(N, dtype, **bad), None))
        assert ok, (bad, why)
    for bad in (dict(dhidden=M), dict(dhidden=2 * M), dict(dweight=2 * M), dict(dweight=2 * M - 64), dict(dweight=M + last - last % 4),
                dict(dhidden=9 * M), dict(dhidden=3 * M), dict(dweight=5 * M), dict(dhidden=6 * M), dict(dweight=7 * M), dict(workspace=8 * M),
                dict(workspace=9 * M), dict(workspace=2 * M), dict(dhidden=10 * M + (1 << 28))):
        ok, why = refused(lib, lib.mb_linear_ce_bwd(loss(N, dtype, **bad), None))
        assert ok, (bad, why)


def test_rotation(lib):
    from mathbrain.rotary import _ARGS
    names = ("q k q0 q1 q2 k0 k1 k2 cos sin table_rows start start_bytes start_per_token start0 B L H Hk hd turned layout "
             "inverse dtype q_out k_out").split()
    good = dict(q=M, k=2 * M, q0=4 * 3 * 128, q1=3 * 128, q2=64, k0=512, k1=128, k2=64, cos=3 * M, sin=4 * M, table_rows=64, start=5 * M,
                start_bytes=4, start_per_token=0, start0=0, B=2, L=4, H=2, Hk=2, hd=64, turned=64, layout=0, inverse=0, dtype=0, q_out=6 * M,
                k_out=7 * M)
    assert list(good) == names
    last = (4 * 3 * 128 + 3 * 3 * 128 + 64 + 64) * 4          # behind q's last element
    for bad in (dict(q_out=M), dict(k_out=M), dict(q_out=2 * M), dict(k_out=2 * M), dict(q_out=M + last - 4), dict(q_out=M - 2 * 4 * 2 * 64 * 4 + 4),
                dict(k_out=6 * M), dict(q_out=3 * M), dict(k_out=4 * M), dict(q_out=5 * M), dict(q_out=5 * M + 4),
                dict(q=M, q0=-512, q1=-128, q_out=M - 4 * 512)):
        ok, why = refused(lib, lib.mb_apply_rotary(_ARGS.pack(*(good | bad).values()), None))
        assert ok, (bad, why)
