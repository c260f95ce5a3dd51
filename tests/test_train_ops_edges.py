"""Edges of the training operators' entry points that need no GPU."""
from opendde_b200 import _abi


def test_layernorm_of_no_rows():
    """No rows have no address; without one, rows are still refused."""
    lib = _abi.load()
    assert lib.pf_layernorm_fwd(None, None, None, None, 0, 64, 1e-5, _abi.PF_F32, None) == _abi.PF_OK
    assert lib.pf_layernorm_fwd(None, None, None, None, 1, 64, 1e-5, _abi.PF_F32, None) == _abi.PF_EINVAL_ARG
    assert lib.pf_layernorm_fwd(None, None, None, None, 0, 1025, 1e-5, _abi.PF_F32, None) == _abi.PF_EINVAL_SHAPE
