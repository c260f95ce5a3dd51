"""Edges of the training operators on the GPU."""
import pytest
import torch

from opendde_b200 import autograd, kernels
from test_gpu_train_ops import _att, _rand, _run
from train_ops_support import check, layernorm_ref, token_ids

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("bias", [None, "shared", "batch"])
@pytest.mark.parametrize("n_q,n_k,d", [(70, 80, 32), (33, 200, 64)])
def test_attention_padded_entries_may_hold_anything(n_q, n_k, d, bias, bad, dtype, cuda_device):
    """A batch entry whose keys are all masked has output and gradients 0 whatever its queries and the gradient of its
    output hold; the other entries and a shared bias's gradient keep their bits."""
    q, k, v, do, bt, mask = _att(9, n_q, n_k, 2, 2, d, dtype, cuda_device, bias, F32, "holes")
    want = _run(q, k, v, do, bt, mask)
    gone = (mask == 0).all(1)
    assert gone.sum() == 1
    q2, do2 = q.clone(), do.clone()
    q2[gone], do2[gone] = bad, bad
    got = _run(q2, k, v, do2, bt, mask)
    for name in want:
        assert torch.equal(got[name], want[name]), name
        if not (name == "dbias" and bias == "shared"):
            assert not got[name][gone].any(), name


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,c", [(2600, 513), (2100, 640), (3001, 768), (2000, 769), (1800, 896), (2500, 1000),
                                    (1500, 1001), (3000, 1024), (600, 1023)])
def test_layernorm_bwd_of_many_wide_rows(rows, c, dtype, cuda_device):
    """More than 512 channels, several rows to each warp, partial sums of many blocks."""
    x, dy = _rand((rows, c), dtype, cuda_device, 1, 2.0), _rand((rows, c), dtype, cuda_device, 2)
    w = _rand((c,), F32, cuda_device, 3, 0.3) + 1
    val, bound = layernorm_ref(x, dy, w, 1e-5)
    got = dict(zip(("dx", "dw", "db"), kernels.layernorm_bwd(x, dy, w)))
    for name in got:
        check(got[name], val[name], bound[name], name)
    again = dict(zip(got, kernels.layernorm_bwd(x, dy, w)))
    assert all(torch.equal(got[name], again[name]) for name in got)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c,limits", [(37, (512,)), (65, (256,)), (128, (1024,)), (384, (128, 256)), (512, (256,)),
                                      (768, (128,)), (1001, (128,)), (1024, (128,)), (7, (1024, 2048)), (16, (4096,))])
def test_layernorm_bwd_where_the_launches_change(c, limits, dtype, cuda_device):
    """One cluster up to some number of rows, two launches from there on; a call that wants dx alone has neither sums."""
    w = _rand((c,), F32, cuda_device, 3, 0.3) + 1
    for rows in (r + more for r in limits for more in (0, 1)):
        x, dy = _rand((rows, c), dtype, cuda_device, 1, 2.0), _rand((rows, c), dtype, cuda_device, 2)
        val, bound = layernorm_ref(x, dy, w, 1e-5)
        got = kernels.layernorm_bwd(x, dy, w)
        for name, t in zip(("dx", "dw", "db"), got):
            check(t, val[name], bound[name], f"{name} of {rows}")
        assert torch.equal(kernels.layernorm_bwd(x, dy, w, need=(True, False, False))[0], got[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_gradient_of_an_expanded_plane_needs_no_copies(dtype, cuda_device):
    """One plane expanded over the batch: a gradient for each entry, and no room for a plane of each beside it."""
    B, n = 32, 256
    q, k, v, do, plane, mask = _att(B, n, n, 4, 4, 32, dtype, cuda_device, "shared", dtype, "pad")
    o, saved = kernels.attention(q, k, v, plane, mask, save=True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = kernels.attention_bwd(do, q, k, v, o, saved, plane.expand(B, -1, -1, -1), mask)
    peak = torch.cuda.max_memory_allocated() - before
    # the gradients, the row constants (16 bytes a row) and the allocator's rounding of a dozen blocks
    assert peak <= sum(t.numel() * t.element_size() for t in got) + 16 * B * n * 4 + 12 * (2 << 20)
    want = kernels.attention_bwd(do, q, k, v, o, saved, plane.repeat(B, 1, 1, 1), mask)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_backward_of_an_eager_forward_is_refused_in_a_capture(cuda_device):
    """A forward pass made before the capture: its backward is refused inside, and works afterwards."""
    x = _rand((1, 8, 2, 32), F32, cuda_device, 1).requires_grad_()
    table = _rand((2, 139), F32, cuda_device, 2).requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [autograd.layer_norm(x), autograd.attention(x, x, x),
                autograd.relative_position_bias(table, token_ids(8, 2, cuda_device), 32, 2)]
        grads = [torch.ones_like(y) for y in outs]
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            for y, g in zip(outs, grads):
                with pytest.raises(RuntimeError, match="not captured"):
                    y.backward(g, retain_graph=True)
            z = kernels.layernorm(x, None, None)
        finally:
            graph.capture_end()
        graph.replay()
        side.synchronize()
        assert torch.equal(z, outs[0].detach()) and x.grad is None and table.grad is None
        for y, g in zip(outs, grads):
            y.backward(g)
        side.synchronize()
    assert torch.isfinite(x.grad).all() and table.grad.any()
