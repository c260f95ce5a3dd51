"""The modules' differentiable forms next to their forward, and on masks that are not 0 and 1."""
import pytest
import torch

from oracle import pairformer_oracle as O
from opendde_b200 import autograd
from opendde_b200.model import AttentionPairBias, LayerNorm, RelativePositionEncoding, TriangleAttention
from opendde_b200.model.trunk_init import trunk_pair_init
from opendde_b200.utils import make_inputs, ragged_pair_mask, seeded_init_
from test_gpu_autograd import TOL, _compare
from train_ops_support import U, relpos_columns, token_ids

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _pair_mask(n, device):
    """Holes; a row that is masked, one of equal fractions, one of several; a fraction beside full keys; a value
    above 1."""
    mask = ragged_pair_mask(n, seed=8, drop=0.2, full_rows=[4])
    mask[0, ::3] = 0.5
    mask[0, 1] = 1.0
    mask[7] = 0.25
    mask[9] = torch.arange(n) % 4 * 0.125
    mask[11, 2] = 1.5
    mask[11, 3] = 1.0
    return mask.to(device)


def _triangle_attention(z, mask, p, heads, starting, uniform):
    """The update in z's type: each row's keys are those of its largest mask value; a row whose largest is below 1
    is a softmax over its scores, or the plain mean of v over its keys."""
    if not starting:
        z, mask = z.transpose(0, 1), mask.t()
    n = z.shape[0]
    x = O.layer_norm(z, p["layer_norm.weight"], p["layer_norm.bias"], 1e-5)
    q, k, v, g = (O.linear(x, p[f"mha.linear_{m}.weight"]).view(n, n, heads, -1).transpose(1, 2) for m in "qkvg")
    t = q @ k.transpose(2, 3) / q.shape[-1] ** 0.5 + O.linear(x, p["linear.weight"]).permute(2, 0, 1)
    m = mask.clamp(max=1)
    top = m.amax(-1, keepdim=True)
    if uniform:
        t = t.masked_fill((top < 1)[:, None, None], 0.0)
    o = torch.softmax(t.masked_fill((m != top)[:, None, None], float("-inf")), -1) @ v
    out = O.linear((o * torch.sigmoid(g)).transpose(1, 2).flatten(2), p["mha.linear_o.weight"])
    return out if starting else out.transpose(0, 1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("starting", [True, False])
@pytest.mark.parametrize("uniform", [True, False])
def test_triangle_attention_masks(uniform, starting, dtype, cuda_device):
    _, z, _ = make_inputs(29, c_z=64, seed=6, with_s=False)
    mask = _pair_mask(29, cuda_device)
    if not starting:
        mask = mask.t()
    mod = TriangleAttention(c_in=64, c_hidden=32, no_heads=2, starting=starting)
    # the form above is the oracle's: with its 1e9 the scores of a row without a full key survive in fp64, with 1e30
    # they vanish as they do in fp32 with 1e9
    p64 = {name: t.double() for name, t in seeded_init_(mod, seed=3, perturb_1d=True).items()}
    m64 = mask.cpu().double()
    want = O.triangle_attention(z.double(), m64.clamp(max=1), p64, 2, starting=starting, inf=1e30 if uniform else 1e9)
    same = _triangle_attention(z.double(), m64, p64, 2, starting, uniform)
    assert (want - same).norm() <= 1e-5 * want.norm()
    _compare(mod, cuda_device, dtype, [z], lambda p, z: _triangle_attention(z, mask.double(), p, 2, starting, uniform),
             lambda m, z: m.differentiable(z, mask, uniform_rows=uniform), TOL[dtype])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("starting", [True, False])
def test_triangle_attention_follows_forward(starting, dtype, cuda_device):
    """The same update as the inference forward, masked rows and fractions beside full keys included, within what both
    may be off (bf16: forward's scores are fp16 values, 2e-2 as for its parity with the reference)."""
    _, z, _ = make_inputs(40, c_z=64, seed=6, with_s=False)
    mask = ragged_pair_mask(40, seed=8, drop=0.2, full_rows=[4, 39])
    mask[0, ::3] = 0.5
    mask[0, 1] = 1.0
    mask = mask.to(cuda_device) if starting else mask.t().to(cuda_device)
    mod = TriangleAttention(c_in=64, c_hidden=32, no_heads=2, starting=starting)
    seeded_init_(mod, seed=3, perturb_1d=True)
    mod, z = mod.to(cuda_device), z.to(cuda_device, dtype)
    with torch.no_grad():
        want, got = mod(z, mask), mod.differentiable(z, mask, uniform_rows=True)
        every = mod.differentiable(z), mod(z)
    tol = TOL[F32] if dtype == F32 else 2e-2
    for a, b in ((got, want), every):
        assert ((a.double() - b.double()).norm() / b.double().norm()).item() <= tol
    with pytest.raises(ValueError, match="mask"):
        mod.differentiable(z, mask[:, :-1])


def test_no_tokens(cuda_device):
    """The forms of nothing: shapes and zero gradients, no error."""
    x = torch.zeros(0, 0, 64, device=cuda_device, requires_grad=True)
    ln = LayerNorm(64).to(cuda_device)
    ln.differentiable(x).sum().backward()
    assert x.grad.shape == x.shape and not ln.weight.grad.any()
    mod = TriangleAttention(c_in=64, c_hidden=32, no_heads=2).to(cuda_device)
    for mask in (None, torch.ones(0, 0, device=cuda_device)):
        out = mod.differentiable(x, mask, uniform_rows=True)
        out.sum().backward()
        assert out.shape == x.shape and not mod.mha.linear_q.weight.grad.any()
    apb = AttentionPairBias(has_s=False, create_offset_ln_z=True, n_heads=4, c_a=96, c_z=64).to(cuda_device)
    for dtype in (F32, BF16):
        a, z = torch.zeros(0, 96, device=cuda_device, dtype=dtype), torch.zeros(0, 0, 64, device=cuda_device, dtype=dtype)
        out = apb.differentiable(a, z)
        out.sum().backward()
        assert out.shape == a.shape and not apb.linear_nobias_z.weight.grad.any()


def test_attention_pair_bias_is_fp32(cuda_device, monkeypatch):
    """bf16 inputs: the bias that attention gets is the fp32 product of the normalised pair tensor and the weight, as
    in forward, and its gradient reaches the weight unrounded. Sums of 64 and n^2 products."""
    n = 50
    s, z, _ = make_inputs(n, c_z=64, c_s=96, seed=5)
    mod = AttentionPairBias(has_s=False, create_offset_ln_z=True, n_heads=4, c_a=96, c_z=64)
    seeded_init_(mod, seed=3, perturb_1d=True)
    mod, s, z = mod.to(cuda_device), s.to(cuda_device, BF16), z.to(cuda_device, BF16)
    w = mod.linear_nobias_z.weight
    with torch.no_grad():
        w.copy_(w.to(BF16))  # forward multiplies bf16 weights
    seen, attention = {}, autograd.attention

    def record(q, k, v, bias, *rest):
        seen["bias"] = bias.detach()
        bias.register_hook(lambda g: seen.update(grad=g))
        return attention(q, k, v, bias, *rest)
    monkeypatch.setattr(autograd, "attention", record)
    out = mod.differentiable(s, z)
    out.backward(torch.randn(out.shape, generator=torch.Generator().manual_seed(1)).to(cuda_device, BF16))
    y, w64 = mod.layernorm_z(z).double(), w.detach().double()
    assert seen["bias"].dtype == seen["grad"].dtype == F32
    far = (seen["bias"].double() - (y @ w64.t()).permute(2, 0, 1)).abs()
    assert (far <= 72 * U * (y.abs() @ w64.abs().t()).permute(2, 0, 1)).all()
    g = seen["grad"].double()
    far = (w.grad.double() - torch.einsum("hij,ijc->hc", g, y)).abs()
    assert (far <= 16 * n * U * torch.einsum("hij,ijc->hc", g.abs(), y.abs())).all()
    # forward's own bias rounds its normalised input to bf16 as well
    rel = (seen["bias"].double() - mod.pair_bias(z).double()).norm() / seen["bias"].double().norm()
    assert rel.item() <= 2.0 ** -8


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_single_update_with_a_relative_position_bias(dtype, cuda_device):
    """s + AttentionPairBias(s, z) with RelativePositionEncoding.head_bias as extra_attn_bias: outputs and gradients of
    s, z, every parameter and the table against fp64 autograd of the same formula."""
    n, heads = 37, 4
    s, z, _ = make_inputs(n, c_z=64, c_s=96, seed=5)
    ids = token_ids(n, 2, cuda_device)
    relpe = RelativePositionEncoding(r_max=8, s_max=2, c_z=heads).to(cuda_device)
    feats = relpe.generate_relp(dict(zip(("asym_id", "residue_index", "entity_id", "token_index", "sym_id"), ids)))["relp"]
    mod = AttentionPairBias(has_s=False, create_offset_ln_z=False, n_heads=heads, c_a=96, c_z=64)
    p = {k: t.double().to(cuda_device).requires_grad_() for k, t in seeded_init_(mod, seed=3, perturb_1d=True).items()}
    mod = mod.to(cuda_device)
    s, z = s.to(cuda_device, dtype).requires_grad_(), z.to(cuda_device, dtype).requires_grad_()
    table = relpe.linear_no_bias.weight
    got = s + mod.differentiable(s, z, relpe.head_bias(feats))

    s64, z64, t64 = (t.detach().double().requires_grad_() for t in (s, z, table))
    y = O.layer_norm(s64, p["layernorm_a.weight"], p["layernorm_a.bias"], 1e-5)
    q = O.linear(y, p["attention.linear_q.weight"], p["attention.linear_q.bias"])
    k, v, g = (O.linear(y, p[f"attention.linear_{m}.weight"]) for m in "kvg")
    q, k, v = (t.view(n, heads, -1).transpose(0, 1) for t in (q, k, v))
    bias = O.linear(O.layer_norm(z64, p["layernorm_z.weight"], None, 1e-5), p["linear_nobias_z.weight"]).permute(2, 0, 1)
    bias = bias + torch.einsum("ijf,hf->hij", relpos_columns(ids, slice(0, n), slice(0, n), 8, 2), t64)
    o = (torch.softmax(q @ k.transpose(1, 2) / q.shape[-1] ** 0.5 + bias, -1) @ v).transpose(0, 1).flatten(1)
    want = s64 + O.linear(o * torch.sigmoid(g), p["attention.linear_o.weight"])

    dy = torch.randn(n, 96, generator=torch.Generator().manual_seed(2)).to(cuda_device, dtype)
    names = [k for k, _ in mod.named_parameters()]
    assert set(names) == set(p)
    gg = torch.autograd.grad(got, [s, z, table] + [t for _, t in mod.named_parameters()], dy)
    gw = torch.autograd.grad(want, [s64, z64, t64] + [p[k] for k in names], dy.double())
    for name, a, b in zip(["out", "s", "z", "table"] + names, (got,) + gg, (want,) + gw):
        assert ((a.double() - b).norm() / b.norm()).item() <= TOL[dtype], name
    with torch.no_grad():  # the inference form of the same call
        want = s + mod(s, None, z, extra_attn_bias=relpe.head_bias(feats))
    assert ((got.double() - want.double()).norm() / want.double().norm()).item() <= TOL[dtype]


def test_pair_input_and_head_bias_have_the_same_features(cuda_device):
    """The trunk's pair input (of a zero single input: the relative-position term alone) and the head bias of one table
    are the same sums of columns, also for ids at the ends of int32, whose differences do not fit."""
    n, c = 50, 64
    ids = list(token_ids(n, 3, cuda_device))
    lim = torch.iinfo(torch.int32)
    at = torch.arange(n, device=cuda_device)
    ids[1] = torch.where(at % 2 == 0, lim.min, lim.max).int()
    ids[3] = torch.where(at % 5 == 0, lim.max, lim.min).int()
    ids[4] = torch.where(at % 3 == 0, lim.min, lim.max).int()
    relpe = RelativePositionEncoding(r_max=32, s_max=2, c_z=c).to(cuda_device)
    feats = relpe.generate_relp(dict(zip(("asym_id", "residue_index", "entity_id", "token_index", "sym_id"), ids)))["relp"]
    one, two, bond = (torch.nn.Linear(k, c, bias=False).to(cuda_device) for k in (96, 96, 1))
    z = trunk_pair_init(torch.zeros(n, 96, device=cuda_device), one, two, relpe, bond, feats, None)
    w = relpe.linear_no_bias.weight.detach().double()
    hot = relpos_columns(ids, slice(0, n), slice(0, n), 32, 2)
    bound = 8 * U * (hot @ w.abs().t())
    assert ((z.double() - hot @ w.t()).abs() <= bound).all()
    assert ((relpe.head_bias(feats).permute(1, 2, 0).double() - hot @ w.t()).abs() <= bound).all()
