"""The argument checks of the query/key norm's, the attention's with a bucket bias and the gradient
clipping's entry points: they run on the host before anything is launched (no GPU needed)."""
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


def qk(**fields):
    """The packed struct with some fields changed: (name, index) as in the header."""
    from mathbrain.qk_norm import _ARGS
    names = ("q k q0 q1 q2 k0 k1 k2 wq wk cos sin table_rows start start_bytes start0 B L H Hk hd dtype eps q_out k_out "
             "dq_out dk_out g0 g1 g2 h0 h1 h2 dq dk dwq dwk workspace workspace_bytes").split()
    a = dict.fromkeys(names, P) | dict(q0=8192, q1=512, q2=64, k0=8192, k1=512, k2=64, g0=8192, g1=512, g2=64, h0=8192,
                                       h1=512, h2=64, table_rows=64, start=0, start_bytes=4, start0=0, B=2, L=16, H=8,
                                       Hk=8, hd=64, dtype=0, eps=1e-6, workspace_bytes=1 << 30)
    assert set(fields) <= set(names)
    return _ARGS.pack(*(a | fields).values())


REFUSED_QK = [
    (dict(hd=48), "head_dim=48"), (dict(dtype=2), "dtype=2"), (dict(q=0), "null"), (dict(sin=0), "null"),
    (dict(B=-1), "B=-1"), (dict(B=1 << 40), "B=1099511627776"), (dict(H=0), "H=0"),
    (dict(start=P, start_bytes=2), "start_bytes=2"), (dict(start0=49), "pass the table"),
    (dict(start0=-1), "pass the table"), (dict(table_rows=15), "pass the table"), (dict(q=P + 4), "16 bytes"),
    (dict(k1=513), "16 bytes")]


@pytest.mark.parametrize("bad,said", REFUSED_QK)
def test_qk_norm_refusals(lib, bad, said):
    for name in ("mb_qk_norm_rotary_fwd", "mb_qk_norm_rotary_bwd"):
        assert getattr(lib, name)(qk(**bad), None) < 0
        assert said in message(lib) and name in message(lib)


def test_qk_norm_refusals_of_one_direction(lib):
    from mathbrain import _lib
    assert lib.mb_qk_norm_rotary_fwd(None, None) < 0 and "null args" in message(lib)
    for bad, said in ((dict(k_out=0), "null"), (dict(k_out=P + 8), "16 bytes")):
        assert lib.mb_qk_norm_rotary_fwd(qk(**bad), None) < 0 and said in message(lib)
    for bad, rc, said in ((dict(dq_out=0), -1, "null"), (dict(dq=0), -1, "null"), (dict(g1=513), -1, "16 bytes"),
                          (dict(dwq=0), -1, "null"), (dict(workspace=0), _lib.MB_ERR_WORKSPACE, "workspace"),
                          (dict(workspace_bytes=8), _lib.MB_ERR_WORKSPACE, "workspace of 8 bytes")):
        assert lib.mb_qk_norm_rotary_bwd(qk(**bad), None) == rc and said in message(lib)


def test_qk_norm_empty_batches_launch_nothing(lib):
    assert lib.mb_qk_norm_rotary_fwd(qk(B=0), None) == 0
    assert lib.mb_qk_norm_rotary_fwd(qk(L=0, q=0), None) == 0
    assert lib.mb_qk_norm_rotary_bwd_workspace(0, 5, 64) == 0
    assert lib.mb_qk_norm_rotary_bwd_workspace(1, 1, 64) == 2 * 64 * 4
    assert lib.mb_qk_norm_rotary_bwd_workspace(64, 4096, 128) == 1024 * 2 * 128 * 4


def attn(first=(0, 1, 5), **fields):
    from mathbrain.bias_attention import _ARGS
    names = ("q k v q0 q1 q2 k0 k1 k2 v0 v1 v2 bias starts buckets n_starts lengths lengths_bytes q_start q_start_bytes "
             "q_start0 B H Hk Lq Lk hd causal dtype bias_dtype scale o o0 o1 o2 lse d_o g0 g1 g2 dq dk dv dq0 dq1 dq2 dk0 "
             "dk1 dk2 dv0 dv1 dv2 dbias workspace workspace_bytes").split()
    attn.keep = (ctypes.c_int32 * len(first))(*first)
    a = dict.fromkeys(names, P)
    for n in names:
        if n[-1] in "012" and n[:-1] in ("q", "k", "v", "o", "g", "dq", "dk", "dv"):
            a[n] = (64 * 8 * 100, 64, 512)[int(n[-1])]
    a |= dict(starts=ctypes.addressof(attn.keep), buckets=len(first), n_starts=len(first), lengths=0, lengths_bytes=4,
              q_start=0, q_start_bytes=4, q_start0=0, B=2, H=8, Hk=8, Lq=100, Lk=100, hd=64, causal=1, dtype=1, bias_dtype=0,
              scale=0.125, workspace_bytes=1 << 40)
    assert set(fields) <= set(names)
    return _ARGS.pack(*(a | fields).values())


@pytest.mark.parametrize("bad,said", [
    (dict(hd=96), "head_dim=96"), (dict(dtype=3), "dtype=3"), (dict(bias_dtype=-1), "bias_dtype=-1"), (dict(q=0), "null"),
    (dict(v=0), "null"), (dict(bias=0), "null"), (dict(Lq=-1), "Lq=-1"), (dict(Lk=(1 << 29) + 1), "Lk=536870913"),
    (dict(Hk=3), "multiple of Hk=3"), (dict(Hk=0), "Hk=0"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=1e-30), "scale=1e-30"), (dict(scale=1e30), "scale=1e+30"),
    (dict(starts=0), "first distances"), (dict(buckets=4), "4 buckets for 3"), (dict(causal=0), "3 buckets for 3"),
    (dict(lengths=P, lengths_bytes=2), "4 or 8 bytes"), (dict(q_start=P, q_start_bytes=1), "4 or 8 bytes"),
    (dict(q_start0=1 << 30), "q_start=1073741824"), (dict(q=P + 2), "16 bytes"), (dict(k2=513), "16 bytes"),
    (dict(v2=-512), "elements apart"), (dict(q2=1 << 24), "elements apart"), (dict(B=1 << 20, H=1 << 12), "too many"),
    (dict(B=1 << 21), "too many")])
def test_bias_attention_refusals(lib, bad, said):
    for name in ("mb_bias_attn_fwd", "mb_bias_attn_bwd"):
        assert getattr(lib, name)(attn(**bad), None) < 0
        assert said in message(lib) and name in message(lib)


@pytest.mark.parametrize("starts,said", [((1, 2), "distance 1, not at 0"), ((0, 5, 4), "must not fall"), ((0, 0, 4), "one alone is 0"),
                                         ((0, 1025), "distance 1025"), (tuple(range(129)), "129 buckets")])
def test_bias_attention_bucket_refusals(lib, starts, said):
    assert lib.mb_bias_attn_fwd(attn(starts), None) < 0 and said in message(lib)


def test_bias_attention_refusals_of_one_direction(lib):
    from mathbrain import _lib
    assert lib.mb_bias_attn_fwd(None, None) < 0 and "null args" in message(lib)
    for bad, rc, said in ((dict(o=0), -1, "null"), (dict(o=P + 8), -1, "16 bytes"),
                          (dict(Lq=1, Lk=4096, workspace=P + 8), -1, "multiple of 16"),
                          (dict(Lq=1, Lk=4096, workspace=0), _lib.MB_ERR_WORKSPACE, "workspace"),
                          (dict(Lq=1, Lk=4096, workspace_bytes=64), _lib.MB_ERR_WORKSPACE, "workspace of 64 bytes")):
        assert lib.mb_bias_attn_fwd(attn(**bad), None) == rc and said in message(lib)
    for bad, rc, said in ((dict(d_o=0), -1, "null"), (dict(lse=0), -1, "null"), (dict(dk=0), -1, "null"),
                          (dict(g2=513), -1, "16 bytes"), (dict(g2=1 << 24), -1, "elements apart"), (dict(dv=P + 4), -1, "16 bytes"),
                          (dict(workspace=P + 4), -1, "multiple of 16"),
                          (dict(workspace=0), _lib.MB_ERR_WORKSPACE, "workspace"),
                          (dict(workspace_bytes=64), _lib.MB_ERR_WORKSPACE, "workspace of 64 bytes")):
        assert lib.mb_bias_attn_bwd(attn(**bad), None) == rc and said in message(lib)


def test_bias_attention_workspaces(lib):
    assert lib.mb_bias_attn_fwd(attn(B=0), None) == 0 and lib.mb_bias_attn_fwd(attn(Lq=0), None) == 0
    size = lib.mb_bias_attn_fwd_workspace
    assert size(56, 8, 8, 512, 512, 64, 1, 1) == 0                    # a grid that fills the device
    assert size(16, 8, 8, 1, 4096, 64, 1, 1) > 0 and size(16, 8, 8, 1, 100, 64, 1, 1) == 0
    assert size(0, 8, 8, 1, 4096, 64, 1, 1) == 0 and size(1, 8, 3, 1, 4096, 64, 1, 1) == 0
    assert size(1 << 30, 1 << 30, 1, 1 << 30, 1 << 30, 64, 1, 1) == 0  # no overflow on the way to "no"
    size = lib.mb_bias_attn_bwd_workspace
    assert size(2, 8, 8, 100, 100, 64, 1, 1, 32) == (2 * 2 * 8 * 100 + 8 * 2 * 32) * 4
    assert size(2, 8, 8, 0, 100, 64, 1, 1, 32) == 0 and size(1, 8, 3, 5, 5, 64, 1, 1, 32) == 0
    # few blocks of long walks: the runs that they are split into
    assert size(1, 8, 2, 1000, 1000, 64, 1, 1, 32) > (2 * 8 * 1000 + 8 * 8 * 32) * 4 + 2 * 8 * 1000 * 64 * 4


def test_bucket_starts():
    from mathbrain.bias_attention import bucket_starts
    assert bucket_starts(1, 5) == (0,) and bucket_starts(2, 100) == (0, 1) and bucket_starts(3, 100) == (0, 1, 10)
    assert bucket_starts(32, 128)[:17] == tuple(range(17)) and bucket_starts(32, 128)[-1] == 113
    # the border of 4 buckets up to 16 lies at sqrt(2 * 16) = 5.66, that of 4 up to 18 at 6 itself
    assert bucket_starts(4, 16) == (0, 1, 2, 6) and bucket_starts(4, 18) == (0, 1, 2, 6) and bucket_starts(4, 19)[-1] == 7
    for n, reach in ((16, 9), (31, 200), (128, 1024)):
        starts = bucket_starts(n, reach)
        assert len(starts) == n and list(starts) == sorted(starts) and starts[-1] <= reach


def test_rows_of_one_token_with_odd_strides_are_copied():
    """A tensor may be contiguous by its sizes and have any strides where a size is 1."""
    from mathbrain import bias_attention, qk_norm
    x = torch.arange(200.0)[2:].as_strided((1, 1, 1, 64), (7, 5, 3, 1))
    for rows16 in (bias_attention._rows16, qk_norm._rows16):
        y = rows16(x)
        assert y.data_ptr() % 16 == 0 and all(s % 4 == 0 for s in y.stride()[:3]) and torch.equal(x, y)


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
    from mathbrain.bias_attention import relative_bias_attention
    from mathbrain.grad_clip import clip_gradients
    from mathbrain.qk_norm import qk_norm_rotary
    x = torch.zeros(1, 1, 1, 32)
    with pytest.raises(NotImplementedError, match="no CPU path"):
        qk_norm_rotary(x, x, x[0, 0, 0], x[0, 0, 0], x[0, 0, :, :16], x[0, 0, :, :16])
    with pytest.raises(NotImplementedError, match="no CPU path"):
        clip_gradients([x], 1.0)
    with pytest.raises(NotImplementedError, match="no CPU path"):
        relative_bias_attention(x, x, x, torch.zeros(4, 1))


def test_inline_assembly_that_writes_m0_says_so():
    """The compiler uses M0 itself; a statement that sets it has to name it as overwritten."""
    import glob
    import os
    import re

    import mathbrain
    found = 0
    for path in glob.glob(os.path.join(os.path.dirname(mathbrain.__file__), "csrc", "*.h*")):
        for statement in re.findall(r"\basm\b[^;]*;", open(path).read()):
            code, *rest = statement.split("\n                 :")   # the operands' lines
            if re.search(r"s_mov_b32 m0\b", code):
                found += 1
                assert '"m0"' in "".join(rest), (path, statement)
    assert found == 2


def test_a_model_that_does_not_drop_out_probabilities_says_so():
    import warnings

    from mathbrain.baseline import RoPETransformerLM
    with pytest.warns(UserWarning, match="not dropped out"):
        RoPETransformerLM(10, 64, 1, 2, max_seq_len=8, rel_buckets=8)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        RoPETransformerLM(10, 64, 1, 2, max_seq_len=8, dropout=0.0, rel_buckets=8)
        RoPETransformerLM(10, 64, 1, 2, max_seq_len=8)


def test_the_first_distances_live_until_the_call_is_made(monkeypatch):
    """The struct holds their address; a cache may drop the array meanwhile (another thread's calls)."""
    import weakref

    from mathbrain import _lib, bias_attention
    alive, calls = [], []

    def starts(num_buckets, max_distance, causal):
        array = (ctypes.c_int32 * 4)(0, 1, 2, 3)
        alive.append(weakref.ref(array))
        return array, ctypes.addressof(array), 4

    def call(dev, name, args):
        calls.append(name)
        assert alive[-1]() is not None, name
    monkeypatch.setattr(bias_attention, "_starts_array", starts)
    monkeypatch.setattr(_lib, "call_on", call)
    monkeypatch.setattr(_lib, "workspace_bytes", lambda *sizes: 16)
    x = torch.zeros(1, 1, 2, 32)
    rest = (8, True, 1.0, None, None, 0, True)
    o, lse = bias_attention.bias_attn_fwd(x, x, x, torch.zeros(4, 1), *rest)
    bias_attention.bias_attn_bwd(x, x, x, torch.zeros(4, 1), o, x, lse, *rest)
    assert calls == ["mb_bias_attn_fwd", "mb_bias_attn_bwd"]
