"""Edges of the training operators' entry points that need no GPU."""
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
