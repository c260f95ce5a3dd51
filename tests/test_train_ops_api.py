"""What the training operators refuse, checked on the host: no GPU is needed and nothing is launched."""
import ctypes

import pytest
import torch

from opendde_b200 import _abi, kernels


def _shape(**kw):
    s = dict(batch=2, n_q=4, n_k=5, heads=4, kv_heads=2, head_dim=32, scale=1.0, dtype=_abi.PF_F32,
             bias_dtype=_abi.PF_F32)
    s.update(kw)
    return _abi.AttentionShape(*s.values())


HV = _abi.HeadView(256, 4096, 128, 32)
NOB, NOM = _abi.BiasView(None, 0, 0, 0), _abi.MaskView(None, 0, 0)


def _fwd(shape, q=HV, k=HV, v=HV, bias=NOB, mask=NOM, o=HV):
    none = _abi.HeadView(None, 0, 0, 0)
    call = _abi.AttentionCall(shape, q, k, v, bias, mask, o, None, None, none, none, none, none, NOB) if shape else None
    return _abi.load().pf_attention_fwd(ctypes.byref(call) if shape else None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), _abi.PF_EINVAL_SHAPE), (dict(n_q=1 << 31), _abi.PF_EINVAL_SHAPE),
    (dict(heads=0), _abi.PF_EINVAL_SHAPE), (dict(kv_heads=3), _abi.PF_EINVAL_SHAPE),
    (dict(head_dim=0), _abi.PF_EINVAL_SHAPE), (dict(head_dim=129), _abi.PF_EUNSUPPORTED),
    (dict(dtype=5), _abi.PF_EINVAL_DTYPE), (dict(bias_dtype=-1), _abi.PF_EINVAL_DTYPE)])
def test_attention_shapes_refused(kw, status):
    assert _fwd(_shape(**kw)) == status
    out = ctypes.c_size_t(0)
    assert _abi.load().pf_attention_bwd_workspace_size(ctypes.byref(_shape(**kw)), ctypes.byref(out)) == status


def test_attention_views_refused():
    null, neg, odd = _abi.HeadView(None, 0, 0, 0), _abi.HeadView(256, -1, 1, 1), _abi.HeadView(257, 4096, 128, 32)
    lap = _abi.HeadView(256, 4096, 16, 32)
    assert _fwd(None) == _abi.PF_EINVAL_ARG
    for bad in (null, neg, odd):
        for arg in ("q", "k", "v", "o"):
            assert _fwd(_shape(), **{arg: bad}) == _abi.PF_EINVAL_ARG, arg
    assert _fwd(_shape(), o=lap) == _abi.PF_EINVAL_ARG      # outputs that share elements
    assert _fwd(_shape(), bias=_abi.BiasView(256, 0, -5, 5)) == _abi.PF_EINVAL_ARG
    assert _fwd(_shape(), bias=_abi.BiasView(258, 0, 20, 5)) == _abi.PF_EINVAL_ARG
    assert _fwd(_shape(), mask=_abi.MaskView(256, -1, 1)) == _abi.PF_EINVAL_ARG
    assert _fwd(_shape(n_q=0), q=null, o=null) == _abi.PF_OK


def test_attention_backward_refused():
    def bwd(shape=None, stats=256, o_lo=256, dq=HV, dk=HV, dv=HV, bias=NOB, dbias=NOB, ws=None, nbytes=0):
        call = _abi.AttentionCall(shape or _shape(), HV, HV, HV, bias, NOM, HV, stats, o_lo, HV, dq, dk, dv, dbias)
        return _abi.load().pf_attention_bwd(ctypes.byref(call), ws, nbytes, None)
    null = _abi.HeadView(None, 0, 0, 0)
    plane = _abi.BiasView(256, 80, 20, 5)
    assert bwd(dk=null) == _abi.PF_EINVAL_ARG               # dk and dv come together
    assert bwd(stats=None) == _abi.PF_EINVAL_ARG
    assert bwd(shape=_shape(dtype=_abi.PF_BF16), o_lo=None) == _abi.PF_EINVAL_ARG
    assert bwd(dbias=plane) == _abi.PF_EINVAL_ARG           # dbias without a bias
    assert bwd(bias=plane, dbias=_abi.BiasView(256, 0, 20, 5)) == _abi.PF_EINVAL_ARG   # shared only in one
    assert bwd(bias=plane, dbias=_abi.BiasView(256, 80, 20, 4)) == _abi.PF_EINVAL_ARG  # rows overlap
    assert bwd(dq=_abi.HeadView(256, 4096, 16, 32)) == _abi.PF_EINVAL_ARG
    need = _abi.workspace_bytes("pf_attention_bwd_workspace_size", ctypes.byref(_shape()))
    assert need >= 3 * 2 * 4 * 4 * 4
    assert bwd(bias=plane, dbias=plane) == _abi.PF_EWORKSPACE
    assert bwd(ws=256, nbytes=need - 1) == _abi.PF_EWORKSPACE
    assert bwd(ws=264, nbytes=need) == _abi.PF_EWORKSPACE   # alignment
    assert b"aligned" in _abi.load().pf_last_error_string()


def test_layernorm_backward_refused():
    lib = _abi.load()
    for rows, c in ((-1, 8), (4, 0), (4, 1025)):
        assert lib.pf_layernorm_bwd(256, 256, None, 256, None, None, rows, c, 1e-5, 0, 256, 1 << 30, None) == \
            _abi.PF_EINVAL_SHAPE
    assert lib.pf_layernorm_bwd(256, None, None, 256, None, None, 4, 8, 1e-5, 0, 256, 1 << 30, None) == _abi.PF_EINVAL_ARG
    assert lib.pf_layernorm_bwd(256, 256, None, 256, None, None, 4, 8, 1e-5, 3, 256, 1 << 30, None) == \
        _abi.PF_EINVAL_DTYPE
    assert lib.pf_layernorm_bwd(256, 256, None, 256, None, None, 4, 8, 1e-5, 0, None, 0, None) == _abi.PF_EWORKSPACE
    assert lib.pf_layernorm_bwd(256, 256, None, None, None, None, 4, 8, 1e-5, 0, None, 0, None) == _abi.PF_OK


def test_relpos_refused():
    lib = _abi.load()
    ids, none = _abi.TokenIds(*[256] * 5), _abi.TokenIds(*[256] * 4, None)

    def fwd(ids=ids, n=10, row0=0, rows=10, col0=0, cols=10, heads=2, r=32, s=2, hs=100, rs=10, dtype=0):
        return lib.pf_relpos_bias_fwd(256, 0, ids, 256, hs, rs, dtype, n, row0, rows, col0, cols, heads, r, s, None)
    assert fwd(row0=1) == fwd(col0=-1) == fwd(cols=11) == fwd(heads=0) == fwd(r=-1) == _abi.PF_EINVAL_SHAPE
    assert fwd(r=511) == fwd(s=1 << 30) == _abi.PF_EUNSUPPORTED
    assert fwd(ids=none) == fwd(rs=9) == fwd(hs=3) == _abi.PF_EINVAL_ARG
    assert fwd(dtype=9) == _abi.PF_EINVAL_DTYPE
    assert fwd(rows=0) == _abi.PF_OK
    assert lib.pf_relpos_bias_bwd(256, 100, 10, 0, ids, None, 10, 0, 10, 0, 10, 2, 32, 2, None, 0, None) == \
        _abi.PF_EINVAL_ARG
    assert lib.pf_relpos_bias_bwd(256, 100, 10, 0, ids, 256, 10, 0, 10, 5, 10, 2, 32, 2, None, 0, None) == \
        _abi.PF_EINVAL_SHAPE
    assert lib.pf_relpos_bias_bwd(256, 1000000, 1000, 0, ids, 256, 1000, 0, 1000, 0, 1000, 2, 32, 2, None, 0, None) == \
        _abi.PF_EWORKSPACE


def test_cpu_tensors_are_rejected():
    q = torch.zeros(1, 2, 3, 8)
    for call in (lambda: kernels.attention(q, q, q), lambda: kernels.layernorm_bwd(q, q, None),
                 lambda: kernels.relpos_bias_bwd(torch.zeros(1, 2, 2), (torch.zeros(2).int(),) * 5, 0, 0, 32, 2)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("change,error", [
    (dict(k=torch.zeros(1, 5, 4, 16)), ValueError), (dict(v=torch.zeros(1, 6, 2, 8)), ValueError),
    (dict(k=torch.zeros(1, 5, 2, 8).double()), TypeError), (dict(q=torch.zeros(4, 4, 8)), ValueError),
    (dict(q=torch.zeros(1, 4, 8, 4).transpose(2, 3)), ValueError), (dict(bias=torch.zeros(4, 4, 6)), ValueError),
    (dict(bias=torch.zeros(3, 4, 4, 5)), ValueError), (dict(bias=torch.zeros(4, 4)), ValueError),
    (dict(bias=torch.zeros(4, 5, 4).transpose(1, 2)), ValueError), (dict(mask=torch.zeros(2, 5)), ValueError),
    (dict(mask=torch.zeros(5).double()), TypeError), (dict(bias=torch.zeros(4, 4, 5).half()), TypeError)])
def test_attention_arguments_refused(change, error, monkeypatch):
    """The wrapper's own checks (its device check set aside, so that CPU tensors reach them)."""
    monkeypatch.setattr(kernels, "require_cuda", lambda *a: None)
    args = dict(q=torch.zeros(1, 4, 4, 8), k=torch.zeros(1, 5, 2, 8), v=torch.zeros(1, 5, 2, 8), bias=None, mask=None,
                scale=None)
    kernels._attention_args(**args)
    with pytest.raises(error):
        kernels._attention_args(**{**args, **change})
