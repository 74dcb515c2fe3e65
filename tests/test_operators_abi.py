"""The argument checks of the query/key norm's and the gradient clipping's entry points: they run on
the host before anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch  # noqa: F401  (the library binds to torch's HIP runtime)


@pytest.fixture(scope="module")
def lib():
    from mathbrain import _lib
    return _lib.lib()


def message(lib):
    return lib.mb_last_error().decode()


# any aligned non-null address: the refused calls never use it
P = 1 << 20


def qk_fwd(**bad):
    a = dict(q=P, q_sb=8192, q_sl=512, q_sh=64, k=P, k_sb=8192, k_sl=512, k_sh=64, wq=P, wk=P, cos=P, sin=P,
             table_rows=64, start=None, start_bytes=4, start0=0, B=2, L=16, H=8, Hk=8, hd=64, eps=1e-6, dtype=0,
             q_out=P, k_out=P) | bad
    return tuple(a.values()) + (None,)


@pytest.mark.parametrize("bad,said", [
    (dict(hd=48), "head_dim=48"), (dict(dtype=2), "dtype=2"), (dict(q=None), "null"), (dict(sin=None), "null"),
    (dict(B=-1), "B=-1"), (dict(H=0), "H=0"), (dict(start=P, start_bytes=2), "start_bytes=2"),
    (dict(start0=49), "pass the table"), (dict(start0=-1), "pass the table"), (dict(table_rows=15), "pass the table"),
    (dict(q=P + 4), "16 bytes"), (dict(k_sl=513), "16 bytes"), (dict(k_out=P + 8), "16 bytes")])
def test_qk_norm_forward_refusals(lib, bad, said):
    assert lib.mb_qk_norm_rotary_fwd(*qk_fwd(**bad)) < 0
    assert said in message(lib)


def test_qk_norm_empty_batches_launch_nothing(lib):
    assert lib.mb_qk_norm_rotary_fwd(*qk_fwd(B=0)) == 0
    assert lib.mb_qk_norm_rotary_fwd(*qk_fwd(L=0, q=None)) == 0
    assert lib.mb_qk_norm_rotary_bwd_workspace(0, 5, 64) == 0
    assert lib.mb_qk_norm_rotary_bwd_workspace(1, 1, 64) == 2 * 64 * 4
    assert lib.mb_qk_norm_rotary_bwd_workspace(64, 4096, 128) == 1024 * 2 * 128 * 4


def test_qk_norm_backward_refusals(lib):
    f = qk_fwd()
    strides = (8192, 512, 64)

    def call(dq=P, ws=P, nbytes=1 << 30, dw=P):
        return lib.mb_qk_norm_rotary_bwd(*f[:8], dq, *strides, P, *strides, *f[8:23], P, P, dw, P, ws, nbytes, None)
    from mathbrain import _lib
    for args, rc, said in ((dict(dq=None), -1, "null"), (dict(dq=P + 4), -1, "16 bytes"), (dict(dw=None), -1, "null"),
                           (dict(ws=None), _lib.MB_ERR_WORKSPACE, "workspace"),
                           (dict(nbytes=8), _lib.MB_ERR_WORKSPACE, "workspace of 8 bytes")):
        assert call(**args) == rc and said in message(lib)


def clip(lib, src, dst, n, codes=None, dcodes=None, max_norm=1.0, norm=P, ws=P, nbytes=1 << 30):
    k = len(src)
    arr = lambda t, v: None if v is None else (t * k)(*v)  # noqa: E731
    return lib.mb_grad_clip(arr(ctypes.c_void_p, src), arr(ctypes.c_int32, codes or [0] * k),
                            arr(ctypes.c_void_p, dst), arr(ctypes.c_int32, dcodes or codes or [0] * k),
                            arr(ctypes.c_int64, n), k, max_norm, norm, ws, nbytes, None)


@pytest.mark.parametrize("args,said", [
    (dict(src=[P], dst=[P], n=[-1]), "-1 elements"), (dict(src=[None], dst=[P], n=[4]), "null pointer"),
    (dict(src=[P], dst=[None], n=[4]), "null pointer"), (dict(src=[P], dst=[P], n=[4], codes=[7]), "dtype=7"),
    (dict(src=[P], dst=[P], n=[4], dcodes=[7]), "dtype=7"), (dict(src=[P], dst=[P], n=[4], max_norm=-1.0), "max_norm"),
    (dict(src=[P], dst=[P], n=[4], max_norm=float("nan")), "max_norm"), (dict(src=[P], dst=[P], n=[4], norm=None), "norm_out"),
    (dict(src=[P], dst=[P], n=[4], nbytes=100), "workspace of 100"),
    (dict(src=[P, P], dst=[P, P], n=[4, 4]), "share memory"),
    (dict(src=[P, P + 12], dst=[P, P + 12], n=[4, 4]), "share memory"),
    (dict(src=[P, P + 4096], dst=[P + 8192, P + 4100], n=[4, 4]), "share memory"),
    (dict(src=[P, P + 4096], dst=[P + 4096, P], n=[4, 4]), "share memory"),
    (dict(src=[P], dst=[P], n=[4], codes=[1], dcodes=[0]), "share memory")])
def test_grad_clip_refusals(lib, args, said):
    assert clip(lib, **args) < 0
    assert said in message(lib)


def test_cpu_tensors_are_refused():
    from mathbrain.grad_clip import clip_gradients
    from mathbrain.qk_norm import qk_norm_rotary
    x = torch.zeros(1, 1, 1, 32)
    with pytest.raises(NotImplementedError, match="no CPU path"):
        qk_norm_rotary(x, x, x[0, 0, 0], x[0, 0, 0], x[0, 0, :, :16], x[0, 0, :, :16])
    with pytest.raises(NotImplementedError, match="no CPU path"):
        clip_gradients([x], 1.0)
