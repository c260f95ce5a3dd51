"""The differentiable forms: autograd over the training kernels and the modules built from them, against fp64
autograd of the oracle's restatement of the reference (its functions are plain torch)."""
import math

import pytest
import torch

from oracle import pairformer_oracle as O
from opendde_b200 import autograd, kernels
from opendde_b200.model import (AttentionPairBias, LayerNorm, RelativePositionEncoding, TriangleAttention)
from opendde_b200.utils import make_inputs, ragged_pair_mask, seeded_init_
from train_ops_support import U, relpos_columns, token_ids

pytestmark = pytest.mark.gpu


def _compare(mod, device, dtype, inputs, ref, run, tol):
    """Outputs and gradients of inputs and parameters, relative 2-norms against fp64 autograd."""
    params = seeded_init_(mod, seed=3, perturb_1d=True)
    mod = mod.to(device)
    p64 = {n: t.double().to(device).requires_grad_() for n, t in params.items()}
    x64 = [t.to(device, dtype).double().requires_grad_() for t in inputs]
    # layernorm_z.bias moves all logits of a head alike, so its gradient is a sum over positions that is zero in exact
    # arithmetic; an error relative to it says nothing. Each term is within tol of its own size, the sum within tol of
    # the sum of sizes: its gradient is taken position by position here.
    zero = "layernorm_z.bias"
    if zero in p64:
        p64[zero] = params[zero].double().to(device).expand(*inputs[-1].shape).clone().requires_grad_()
    x = [t.to(device, dtype).requires_grad_() for t in inputs]
    want = ref(p64, *x64)
    got = run(mod, *x)
    assert got.dtype == dtype and got.shape == want.shape
    g = torch.Generator().manual_seed(9)
    dy = torch.randn(want.shape, generator=g).to(device, dtype)
    names = [n for n, _ in mod.named_parameters()]
    gw = torch.autograd.grad(want, x64 + [p64[n] for n in names], dy.double(), allow_unused=True)
    gg = torch.autograd.grad(got, x + [p for _, p in mod.named_parameters()], dy, allow_unused=True)
    for name, a, b in zip(["out"] + [f"x{i}" for i in range(len(x))] + names, (got,) + gg, (want,) + gw):
        assert (a is None) == (b is None), name
        if b is not None:
            size = b
            if name == zero:
                b, size = b.sum((0, 1)), b.abs().sum((0, 1))
            rel = ((a.double() - b).norm() / size.norm().clamp_min(1e-30)).item()
            assert rel <= tol, (name, rel)


# fp32: a chain of some eight products of at most 400 terms, each relative error below 400 U, amplified by the logits'
# size (below 20) at the softmax. bf16: each of the chain's dozen intermediate tensors is rounded once (2^-8), twice
# over for their gradients; the errors are independent, so their squares add: sqrt(24) 2^-8 = 1.9e-2.
TOL = {torch.float32: 8 * 400 * 20 * U / 4, torch.bfloat16: 24 ** 0.5 * 2.0 ** -8}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_pair_bias(dtype, cuda_device):
    s, z, _ = make_inputs(37, c_z=64, c_s=96, seed=5)
    mod = AttentionPairBias(has_s=False, create_offset_ln_z=True, n_heads=4, c_a=96, c_z=64)
    _compare(mod, cuda_device, dtype, [s, z], lambda p, s, z: O.attention_pair_bias(s, z, p, 4),
             lambda m, s, z: m.differentiable(s, z), TOL[dtype])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("starting", [True, False])
def test_triangle_attention(starting, dtype, cuda_device):
    _, z, _ = make_inputs(29, c_z=64, seed=6, with_s=False)
    mask = ragged_pair_mask(29, seed=8, drop=0.2, full_rows=[4]).to(cuda_device)
    if not starting:
        mask = mask.t()  # the ending node's keys run down the columns
    mod = TriangleAttention(c_in=64, c_hidden=32, no_heads=2, starting=starting)

    def ref(p, z):  # autograd through the oracle's rows; it writes them into one tensor
        out = O.triangle_attention(z, mask.double(), p, 2, starting=starting, row_chunk=29)
        return out
    _compare(mod, cuda_device, dtype, [z], ref, lambda m, z: m.differentiable(z, mask), TOL[dtype])


def test_layer_norm_module_and_parameter_types(cuda_device):
    x = torch.randn(5, 7, 96, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    ln = LayerNorm(96).to(cuda_device)
    y = ln.differentiable(x)
    assert torch.equal(y, ln(x)) and not ln(x).requires_grad  # the inference forward builds no graph, as before
    y.float().sum().backward()
    assert x.grad.dtype == torch.bfloat16 and ln.weight.grad.dtype == torch.float32
    assert torch.equal(ln.bias.grad, torch.full_like(ln.bias, 35.0))
    half = LayerNorm(96, create_offset=False).to(cuda_device).to(torch.bfloat16)
    half.differentiable(x.detach()).float().sum().backward()  # only the parameter needs a gradient
    assert half.weight.grad.dtype == torch.bfloat16
    with torch.no_grad():
        assert not ln.differentiable(x).requires_grad


def test_relative_position_head_bias(cuda_device):
    n, heads = 45, 3
    ids = token_ids(n, 2, cuda_device)
    relpe = RelativePositionEncoding(r_max=32, s_max=2, c_z=heads).to(cuda_device)
    names = ("asym_id", "residue_index", "entity_id", "token_index", "sym_id")
    feats = relpe.generate_relp(dict(zip(names, ids)))["relp"]
    bias = relpe.head_bias(feats)
    hot = relpos_columns(ids, slice(0, n), slice(0, n), 32, 2)
    w = relpe.linear_no_bias.weight
    want = torch.einsum("ijf,hf->hij", hot, w.double())
    assert ((bias.double() - want).abs() <= 8 * U * w.abs().max()).all()
    g = torch.randn(heads, n, n, device=cuda_device)
    bias.backward(g.transpose(1, 2))  # a gradient whose columns are not contiguous
    ref = torch.einsum("ijf,hji->hf", hot, g.double())
    assert ((w.grad.double() - ref).abs() <= n * n * U * torch.einsum("ijf,hji->hf", hot, g.double().abs()) + 1e-30).all()
    part = relpe.head_bias(feats, tile=(10, 20, 5, 33), dtype=torch.bfloat16)
    assert torch.equal(part, bias.detach()[:, 10:30, 5:38].to(torch.bfloat16))
    other = RelativePositionEncoding(r_max=16, s_max=2, c_z=heads).to(cuda_device)
    with pytest.raises(ValueError, match="r_max"):
        other.head_bias(feats)


def test_broadcast_inputs_and_layouts(cuda_device):
    """A bias shared by heads and batch, expanded keys, channels that are not contiguous: gradients are sums over what
    was expanded, as autograd makes them."""
    B, n, H, d = 3, 21, 4, 32
    g = torch.Generator().manual_seed(1)
    q = torch.randn(B, n, d, H, generator=g).to(cuda_device).requires_grad_()
    k = torch.randn(B, n, 1, d, generator=g).to(cuda_device).requires_grad_()
    bias = torch.randn(1, 1, n, n, generator=g).to(cuda_device).requires_grad_()
    do = torch.randn(B, n, H, d, generator=g).to(cuda_device)

    def call(q, k, bias, f):
        kk = k.expand(B, n, H, d)
        return f(q.transpose(2, 3), kk, kk, bias.expand(B, H, n, n).transpose(2, 3))

    def plain(q, k, v, bias):
        t = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(d) + bias
        return torch.einsum("bhij,bjhd->bihd", torch.softmax(t, -1), v)
    got = torch.autograd.grad(call(q, k, bias, autograd.attention), (q, k, bias), do)
    q6, k6, b6 = (t.detach().double().requires_grad_() for t in (q, k, bias))
    want = torch.autograd.grad(call(q6, k6, b6, plain), (q6, k6, b6), do.double())
    for a, b in zip(got, want):
        assert ((a.double() - b).norm() / b.norm()).item() <= 400 * 20 * U


def test_refusals(cuda_device):
    x = torch.randn(4, 32, device=cuda_device, requires_grad=True)
    with pytest.raises(ValueError, match="weight and bias"):
        autograd.layer_norm(x, torch.ones(31, device=cuda_device))
    y = autograd.layer_norm(x)
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivatives
        gx.sum().backward()


def test_autograd_is_refused_in_a_capture(cuda_device):
    """A call that needs a gradient is refused while capturing, also next to a live eager graph of the same leaf; the
    capture of calls without gradients goes on working."""
    x = torch.randn(8, 32, device=cuda_device, requires_grad=True)
    live = autograd.layer_norm(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        g.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="not captured"):
                autograd.layer_norm(x)
            q = x.view(1, 8, 1, 32)
            with pytest.raises(RuntimeError, match="not captured"):
                autograd.attention(q, q, q)
            with torch.no_grad():
                y = autograd.layer_norm(x)
            dx = kernels.layernorm_bwd(x, y, None)[0]
        finally:
            g.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    g.replay()
    assert torch.equal(y, live.detach())
    live.backward(y)
    assert torch.equal(x.grad, dx)
