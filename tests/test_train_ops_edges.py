"""Edges of the training operators' entry points that need no GPU."""
import ctypes

from opendde_b200 import _abi


def test_layernorm_of_no_rows():
    """No rows have no address; without one, rows are still refused."""
    lib = _abi.load()
    assert lib.pf_layernorm_fwd(None, None, None, None, 0, 64, 1e-5, _abi.PF_F32, None) == _abi.PF_OK
    assert lib.pf_layernorm_fwd(None, None, None, None, 1, 64, 1e-5, _abi.PF_F32, None) == _abi.PF_EINVAL_ARG
    assert lib.pf_layernorm_fwd(None, None, None, None, 0, 1025, 1e-5, _abi.PF_F32, None) == _abi.PF_EINVAL_SHAPE


def test_layernorm_backward_workspace_goes_by_the_rows():
    """Few rows need few partial rows: never more than one pair per eight rows."""
    for rows, c in ((1, 8), (64, 384), (1000, 65), (9, 1024)):
        need = _abi.workspace_bytes("pf_layernorm_bwd_workspace_size", rows, c, _abi.PF_F32)
        assert 0 < need <= -(-rows // 8) * 2 * c * 4
    large = [_abi.workspace_bytes("pf_layernorm_bwd_workspace_size", rows, 128, _abi.PF_F32) for rows in (1 << 20, 1 << 40)]
    assert large[0] == large[1]


def test_attention_backward_workspace_goes_by_the_call():
    """Partial planes are room for a gradient that is summed over the batch, and for no other call."""
    shape = _abi.AttentionShape(64, 300, 300, 4, 4, 64, 1.0, _abi.PF_BF16, _abi.PF_BF16)
    view, none = _abi.HeadView(256, 300 * 256, 256, 64), _abi.BiasView(None, 0, 0, 0)
    shared, each = _abi.BiasView(256, 0, 90000, 300), _abi.BiasView(256, 360000, 90000, 300)

    def need(bias, dbias):
        call = _abi.AttentionCall(shape, view, view, view, bias, _abi.MaskView(None, 0, 0), view, 256, 256, view, view,
                                  view, view, dbias)
        return _abi.workspace_bytes("pf_attention_bwd_call_workspace_size", ctypes.byref(call))
    rows = 16 * 64 * 4 * 300
    most = _abi.workspace_bytes("pf_attention_bwd_workspace_size", ctypes.byref(shape))
    assert need(shared, shared) == most > rows
    assert need(none, none) == need(each, each) == need(shared, none) == need(shared, each) == rows
    assert _abi.load().pf_attention_bwd_call_workspace_size(None, ctypes.byref(ctypes.c_size_t())) == _abi.PF_EINVAL_ARG
