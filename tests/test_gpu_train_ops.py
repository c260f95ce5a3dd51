"""The training operators on the GPU -- the layer norm's backward, attention with a learned bias and its
backward, the relative-position bias and its table's gradient -- against plain fp64 forms (tolerances: counted
roundings, train_ops_support.py), against differences, and in the calls a program makes of them."""
import math

import pytest
import torch

from opendde_b200 import kernels
from train_ops_support import U, attention_ref, check, half_step, layernorm_ref, relpos_columns, token_ids

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _rand(shape, dtype, device, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(device, dtype)


# ------------------------------------------------------------------------------ layer norm
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 8), (3, 7), (33, 16), (17, 24), (5, 33), (64, 64), (129, 128),
                                    (70, 257), (40, 384), (31, 449), (19, 512), (9, 768), (12, 1001), (10, 1024),
                                    (6001, 128), (2500, 31)])
def test_layernorm_bwd(rows, c, dtype, cuda_device):
    x, dy = _rand((rows, c), dtype, cuda_device, 1, 2.0), _rand((rows, c), dtype, cuda_device, 2)
    w = _rand((c,), F32, cuda_device, 3, 0.3) + 1
    val, bound = layernorm_ref(x, dy, w, 1e-5)
    for name, got in zip(("dx", "dw", "db"), kernels.layernorm_bwd(x, dy, w)):
        assert got.dtype == (dtype if name == "dx" else F32)
        check(got, val[name], bound[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layernorm_bwd_large_mean_no_scale_and_parts(dtype, cuda_device):
    """A mean far above the spread; no scale; any subset of the gradients; a row of equal values."""
    x = _rand((37, 128), dtype, cuda_device, 1) + 100
    x[5] = 3.0
    dy = _rand((37, 128), dtype, cuda_device, 2)
    val, bound = layernorm_ref(x, dy, None, 1e-3)
    full = kernels.layernorm_bwd(x, dy, None, eps=1e-3)
    for name, got in zip(("dx", "dw", "db"), full):
        check(got, val[name], bound[name], name)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        part = kernels.layernorm_bwd(x, dy, None, eps=1e-3, need=need)
        for want, a, b in zip(need, part, full):
            assert torch.equal(a, b) if want else a is None


def test_layernorm_bwd_views_batches_and_empty(cuda_device):
    big = _rand((6, 9, 80), BF16, cuda_device, 1)
    x, dy = big[:, 1:8, 3:40], _rand((7, 6, 37), BF16, cuda_device, 2).transpose(0, 1)
    w = torch.ones(37, device=cuda_device)
    val, bound = layernorm_ref(x, dy, w, 1e-5)
    for name, got in zip(("dx", "dw", "db"), kernels.layernorm_bwd(x, dy, w)):
        check(got, val[name], bound[name], name)
    e = torch.empty(0, 64, device=cuda_device)
    dx, dw, db = kernels.layernorm_bwd(e, e, None)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    # an unaligned start takes the element-wise kernel
    flat = _rand((4 * 128 + 1,), F32, cuda_device, 3)
    x, dy = flat[1:].view(4, 128), _rand((4, 128), F32, cuda_device, 4)
    val, bound = layernorm_ref(x, dy, None, 1e-5)
    check(kernels.layernorm_bwd(x, dy, None)[0], val["dx"], bound["dx"], "dx")


def test_layernorm_gradient_against_differences(cuda_device):
    """<dy, y(x + h u) - y(x - h u)> / 2h against <dx, u>, the outputs in fp64 sums. A step of 2^-6 in rows of unit
    spread: the third derivative term is below h^2 = 2^-12 of |dy||u| sums, the roundings of y are 2^-24 / h."""
    x, dy, u = (_rand((16, 128), F32, cuda_device, s) for s in (1, 2, 3))
    w, b = _rand((128,), F32, cuda_device, 4, 0.2) + 1, _rand((128,), F32, cuda_device, 5)
    h = 2.0 ** -6
    hi, lo = kernels.layernorm(x + h * u, w, b).double(), kernels.layernorm(x - h * u, w, b).double()
    num = (dy.double() * (hi - lo)).sum() / (2 * h)
    dx, dw, db = kernels.layernorm_bwd(x, dy, w)
    ana = (dx.double() * u.double()).sum()
    size = (dy.abs() * u.abs() * w.abs()).sum().item()
    assert abs(num - ana) <= size * (4 * h * h + 16 * U / h)
    du = _rand((128,), F32, cuda_device, 6)  # y is linear in the scale and the offset
    hi, lo = kernels.layernorm(x, w + h * du, b + h * du).double(), kernels.layernorm(x, w - h * du, b - h * du).double()
    num = (dy.double() * (hi - lo)).sum() / (2 * h)
    ana = ((dw + db).double() * du.double()).sum()
    assert abs(num - ana) <= (dy.abs() * (4 + x.abs())).sum().item() * du.abs().max().item() * 64 * U / h


# ------------------------------------------------------------------------------ attention
def _att(B, nq, nk, H, KV, d, dtype, device, bias=None, bias_dtype=None, mask=None, seed=0):
    """Inputs of one attention call: q, k, v, do, bias, mask."""
    q, do = _rand((B, nq, H, d), dtype, device, seed + 1, 1.3), _rand((B, nq, H, d), dtype, device, seed + 2)
    k, v = _rand((B, nk, KV, d), dtype, device, seed + 3, 1.2), _rand((B, nk, KV, d), dtype, device, seed + 4)
    bt = None
    if bias is not None:
        bt = _rand((B if bias == "batch" else 1, H, nq, nk), bias_dtype or dtype, device, seed + 5)
    mt = None
    if mask == "pad":
        mt = torch.ones(B, nk, device=device)
        mt[:, nk - max(1, nk // 5):] = 0
    elif mask == "holes":
        g = torch.Generator().manual_seed(seed + 6)
        mt = (torch.rand((B, nk), generator=g) > 0.3).float().to(device)
        mt[B - 1] = 0
    return q, k, v, do, bt, mt


def _run(q, k, v, do, bias, mask, scale=None):
    o, saved = kernels.attention(q, k, v, bias, mask, scale, save=True)
    dq, dk, dv, db = kernels.attention_bwd(do, q, k, v, o, saved, bias, mask, scale)
    out = {"o": o, "dq": dq, "dk": dk, "dv": dv}
    if bias is not None:
        out["dbias"] = db
    return out


def _verify(args, scale=None):
    val, bound = attention_ref(*args, scale=scale)
    got = _run(*args, scale)
    assert set(got) == set(val)
    for name in val:
        assert torch.isfinite(got[name].float()).all(), name
        check(got[name], val[name], bound[name], name)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,d,H", [(1, 24, 2), (2, 32, 4), (13, 24, 16), (63, 24, 3), (64, 32, 2), (65, 32, 1),
                                   (129, 16, 2), (200, 24, 16)])
def test_attention_single(n, d, H, dtype, cuda_device):
    """One sequence, a bias per head, as AttentionPairBias has it."""
    _verify(_att(1, n, n, H, H, d, dtype, cuda_device, "batch", F32))


@pytest.mark.parametrize("dtype,bias_dtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("n,H,mask", [(2, 4, None), (17, 4, "holes"), (67, 2, "pad"), (96, 4, "holes")])
def test_attention_shared_bias(n, H, mask, dtype, bias_dtype, cuda_device):
    """n rows share one bias plane, as triangle attention has it; the last row of "holes" sees nothing."""
    got = _verify(_att(n, n, n, H, H, 32, dtype, cuda_device, "shared", bias_dtype, mask))
    if mask == "holes":
        assert not got["o"][-1].any() and not got["dq"][-1].any() and not got["dv"][-1].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,nq,nk,H,KV,d,mask,bias_dtype", [
    (40, 100, 130, 4, 4, 24, "holes", BF16), (37, 64, 255, 8, 2, 20, None, F32), (150, 40, 33, 4, 4, 32, "pad", BF16),
    (9, 130, 832, 4, 4, 32, "pad", F32), (9, 130, 833, 4, 4, 32, None, BF16), (21, 97, 65, 16, 16, 3, "holes", F32),
    (6, 200, 190, 4, 2, 64, "pad", BF16), (5, 1, 400, 4, 4, 32, None, F32)])
def test_attention_shared_bias_over_a_long_batch(B, nq, nk, H, KV, d, mask, bias_dtype, dtype, cuda_device):
    """The plane's gradient as a sum over the batch, in one pass with dq or by itself, whole and in parts; the keys up
    to and past what one pass holds; a batch larger than its parts."""
    args = _att(B, nq, nk, H, KV, d, dtype, cuda_device, "shared", bias_dtype, mask)
    got = _verify(args)
    q, k, v, do, bias, mt = args
    o, saved = kernels.attention(q, k, v, bias, mt, save=True)
    alone = kernels.attention_bwd(do, q, k, v, o, saved, bias, mt, need=(False, False, False, True))
    assert alone[:3] == (None, None, None) and torch.equal(alone[3], got["dbias"])
    again = _run(*args)
    assert all(torch.equal(again[name], got[name]) for name in got)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,nq,nk,H,KV,d,mask,bias_dtype", [
    (96, 130, 149, 4, 4, 24, "holes", F32), (100, 65, 256, 6, 3, 32, "pad", BF16), (99, 70, 257, 4, 4, 32, None, F32),
    (100, 67, 512, 4, 1, 30, "holes", F32), (100, 65, 513, 4, 4, 32, "pad", F32)])
def test_attention_shared_bias_with_blocks_for_every_sm(B, nq, nk, H, KV, d, mask, bias_dtype, dtype, cuda_device):
    """As above where the batch's parts fill the machine, which fp32 takes for its one pass: up to 256, up to 512 and
    above 512 keys."""
    test_attention_shared_bias_over_a_long_batch(B, nq, nk, H, KV, d, mask, bias_dtype, dtype, cuda_device)


@pytest.mark.parametrize("dtype,bias_dtype", [(F32, F32), (BF16, BF16), (BF16, F32)])
def test_attention_large_shared_bias_of_any_alignment(dtype, bias_dtype, cuda_device):
    """Enough scores (2^24) that a plane with rows off four elements is copied: odd strides, a base off 16 bytes, and
    one plane expanded over the batch; the plane itself stays as it was."""
    B, n, H = 47, 301, 4
    q, k, v, do, bias, mask = _att(B, n, n, H, H, 16, dtype, cuda_device, "shared", bias_dtype, "pad")
    buf = torch.full((H * n * 303 + 1,), float("nan"), device=cuda_device, dtype=bias_dtype)
    odd = torch.as_strided(buf, (1, H, n, n), (1, n * 303, 303, 1), 1)
    odd.copy_(bias)
    kept = buf.clone()
    got = _verify((q, k, v, do, odd, mask))
    assert torch.equal(buf.view(torch.uint8), kept.view(torch.uint8))
    o, saved = kernels.attention(q, k, v, odd.expand(B, H, n, n), mask, save=True)
    assert torch.equal(o, got["o"])
    each = kernels.attention_bwd(do, q, k, v, o, saved, odd[0], mask)[3]
    assert each.shape == (H, n, n) and torch.equal(each, got["dbias"][0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [1, 3, 8, 33, 40, 64, 65, 96, 100, 128])
def test_attention_head_dims(d, dtype, cuda_device):
    _verify(_att(2, 70, 45, 2, 1, d, dtype, cuda_device, "batch", dtype, "holes"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,nq,nk,H,KV,bias,mask", [(1, 1, 300, 8, 2, "batch", None), (3, 1, 1, 4, 4, "shared", None),
                                                    (2, 130, 1, 2, 2, "batch", None), (2, 3, 257, 6, 1, None, "pad"),
                                                    (4, 191, 66, 4, 2, "shared", "holes"),
                                                    (3, 64, 128, 4, 4, None, None), (1, 1, 5000, 2, 1, None, None),
                                                    (1, 900, 3, 2, 2, "batch", None), (2, 33, 700, 2, 2, "batch", "pad")])
def test_attention_lengths_and_shared_heads(B, nq, nk, H, KV, bias, mask, dtype, cuda_device):
    _verify(_att(B, nq, nk, H, KV, 32, dtype, cuda_device, bias, F32, mask))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,nq,nk,H,KV,d,bias,mask", [
    (1, 70, 130, 8, 1, 128, "batch", "pad"), (2, 65, 67, 16, 2, 96, None, "holes"), (1, 100, 64, 6, 2, 40, "batch", None),
    (1, 33, 200, 12, 2, 24, "shared", "pad"), (1, 1, 1, 16, 1, 8, "batch", None), (2, 129, 90, 4, 1, 64, "shared", None),
    (1, 64, 65, 32, 2, 32, "batch", "pad"), (3, 301, 517, 8, 2, 64, None, "holes"), (2, 0, 70, 8, 2, 32, None, None)])
def test_attention_key_heads_of_many_query_heads(B, nq, nk, H, KV, d, bias, mask, dtype, cuda_device):
    """dk and dv add up to sixteen query heads, shared out to blocks in twos, fours and eights or not at all (three)."""
    args = _att(B, nq, nk, H, KV, d, dtype, cuda_device, bias, F32, mask)
    got = _verify(args) if nq else _run(*args)
    again = _run(*args)
    assert all(torch.equal(again[name], got[name]) for name in got)
    if nq == 0:
        assert not got["dk"].any() and not got["dv"].any()
    q, k, v, do, bt, mt = args
    views = torch.zeros(B, nk, KV, 3 * d, device=cuda_device, dtype=dtype)
    views[..., d:2 * d], views[..., 2 * d:] = k, v
    o, saved = kernels.attention(q, views[..., d:2 * d], views[..., 2 * d:], bt, mt, save=True)
    far = kernels.attention_bwd(do, q, views[..., d:2 * d], views[..., 2 * d:], o, saved, bt, mt,
                                need=(False, True, True, False))
    assert torch.equal(far[1], got["dk"]) and torch.equal(far[2], got["dv"])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_one_visible_key_has_no_score_gradient(dtype, cuda_device):
    q, k, v, do, bias, _ = _att(2, 40, 33, 2, 2, 24, dtype, cuda_device, "batch", F32)
    mask = torch.zeros(2, 33, device=cuda_device)
    mask[0, 7] = mask[1, 32] = 1
    got = _verify((q, k, v, do, bias, mask))
    assert not got["dq"].any() and not got["dk"].any() and not got["dbias"].any()
    assert torch.equal(got["o"][0], v[0, 7].expand(40, 2, 24))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_strides(dtype, cuda_device):
    """Packed projections, transposed batches, odd offsets (no 16-byte accesses), expanded heads and batches,
    a bias inside a wider plane with odd rows."""
    B, n, H, d = 3, 50, 4, 24
    qkv = _rand((B, n, 3, H, d), dtype, cuda_device, 1)
    do = _rand((n, B, H, d), dtype, cuda_device, 2).transpose(0, 1)
    wide = _rand((B, H, n + 3, n + 5), F32, cuda_device, 3)
    mask = torch.ones(n, B, device=cuda_device).t()
    _verify((qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], do, wide[:, :, 2:n + 2, 1:n + 1], mask))
    odd = _rand((B, n, H, d + 5), dtype, cuda_device, 4)
    one = _rand((B, n, 1, d), dtype, cuda_device, 5)
    q, k, v = odd[..., 3:d + 3], one.expand(B, n, H, d), one[:1].expand(B, n, 1, d).expand(B, n, H, d)
    _verify((q, k, v, do, wide[:1, :, :n, :n], None))
    plane = wide[:1, :, 1:n + 1, 2:n + 2]
    got = _run(q, k, v, do, plane.expand(B, H, n, n), None)   # one plane expanded: a gradient for each entry
    want = _run(q, k, v, do, plane.repeat(B, 1, 1, 1), None)
    assert all(torch.equal(got[name], want[name]) for name in want)
    got = _run(q[0], k[0], v[0], do[0], wide[0, :, :n, :n], None)  # without a batch
    want = _run(q[:1], k[:1], v[:1], do[:1], wide[:1, :, :n, :n], None)
    assert all(torch.equal(got[name], want[name].view(got[name].shape)) for name in got)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_masked_places_may_hold_anything(dtype, cuda_device):
    """NaN and infinities at masked keys and in their bias change no bit."""
    q, k, v, do, bias, mask = _att(3, 70, 80, 2, 2, 32, dtype, cuda_device, "batch", F32, "holes")
    want = _run(q, k, v, do, bias, mask)
    k2, v2, b2 = k.clone(), v.clone(), bias.clone()
    gone = mask == 0
    k2[gone], v2[gone] = float("nan"), float("inf")
    b2.masked_fill_(gone[:, None, None, :], float("nan"))
    got = _run(q, k2, v2, do, b2, mask)
    for name in want:
        assert torch.equal(got[name], want[name]), name


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_bias_as_a_mask(dtype, cuda_device):
    """-inf in the bias hides a key (a row of them sees nothing); a row of the type's lowest value is uniform over
    its keys, as fp32 sums have it (the scores vanish next to it)."""
    q, k, v, do, bias, _ = _att(1, 40, 75, 2, 2, 32, dtype, cuda_device, "batch", F32)
    bias[:, :, :, 60:] = -math.inf
    bias[:, :, 3] = -math.inf
    got = _verify_inf((q, k, v, do, bias, None))
    assert not got["o"][0, 3].any() and not got["dbias"][0, :, 3].any()
    low = torch.finfo(F32).min
    bias = torch.full_like(bias, low)
    o, saved = kernels.attention(q, k, v, bias, save=True)
    want = v.double().mean(1, keepdim=True).expand(1, 40, 2, 32)
    bound = v.double().abs().mean(1, keepdim=True) * (2 * 75 * U + 2.0 ** -8 * (dtype == BF16)) + want.abs() * half_step(dtype)
    check(o, want, bound, "o")
    dv = kernels.attention_bwd(do, q, k, v, o, saved, bias)[2]
    want = (do.double().mean(1, keepdim=True) * 40 / 75).expand(1, 75, 2, 32)
    bound = do.double().abs().sum(1, keepdim=True) / 75 * (200 * U + 2.0 ** -8 * (dtype == BF16)) + want.abs() * half_step(dtype)
    check(dv, want, bound, "dv")


def _verify_inf(args):
    q, k, v, do, bias, mask = args
    finite = torch.where(bias == -math.inf, torch.full_like(bias, -1e4), bias)  # exp(-1e4) is 0 in fp64 too
    val, bound = attention_ref(q, k, v, do, finite, mask)
    empty = (bias == -math.inf).all(-1)  # [B, H, n_q]: these rows see nothing
    got = _run(*args)
    keep = ~empty.transpose(1, 2)[..., None]
    for name in ("o", "dq"):
        check(got[name] * keep, val[name] * keep, bound[name], name)
        assert not got[name].masked_fill(keep.expand_as(got[name]), 0).any()
    alive = torch.where(empty[..., None], torch.zeros_like(bias), finite)
    do0 = do * keep
    val, bound = attention_ref(q, k, v, do0, alive, mask)
    for name in ("dk", "dv"):
        check(got[name], val[name], bound[name], name)
    check(got["dbias"], val["dbias"] * ~empty[..., None], bound["dbias"], "dbias")
    return got


def test_attention_large_logits(cuda_device):
    """Logits of several hundred: one key takes each row; nothing overflows."""
    q, k, v, do, bias, _ = _att(1, 50, 60, 2, 2, 32, F32, cuda_device, "batch", F32)
    _verify((q * 20, k * 10, v, do, bias, None))
    _verify((q, k, v, do, bias * 300, None))


def test_attention_peaked_rows_keep_small_gradients(cuda_device):
    """Rows whose probability is 1 in fp32 at one key: its ds is 0, the other keys keep theirs, however small."""
    for dtype in (F32, BF16):
        q, k, v, do, bias, _ = _att(3, 66, 70, 2, 2, 32, dtype, cuda_device, "shared", F32)
        bias[:, :, ::2, 5] += 30.0  # every other row
        _verify((q, k, v, do, bias, None))


def test_attention_parts_scale_and_repeat(cuda_device):
    """Subsets of the gradients, a given scale, and equal bits in two runs."""
    args = _att(5, 45, 50, 4, 2, 32, BF16, cuda_device, "shared", BF16, "pad")
    _verify(args, scale=0.3)
    q, k, v, do, bias, mask = args
    o, saved = kernels.attention(q, k, v, bias, mask, save=True)
    assert torch.equal(o, kernels.attention(q, k, v, bias, mask))
    full = kernels.attention_bwd(do, q, k, v, o, saved, bias, mask)
    for need in ((True, True, True, True), (True, False, False, False), (False, True, False, False),
                 (False, False, True, False), (False, False, False, True)):
        part = kernels.attention_bwd(do, q, k, v, o, saved, bias, mask, need=need)
        for want, a, b in zip(need, part, full):
            assert torch.equal(a, b) if want else a is None


@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.int64, BF16])
def test_attention_mask_types(mask_dtype, cuda_device):
    q, k, v, do, bias, mask = _att(2, 20, 30, 2, 2, 24, F32, cuda_device, None, None, "pad")
    want = _run(q, k, v, do, bias, mask)
    got = _run(q, k, v, do, bias, mask.to(mask_dtype))
    assert all(torch.equal(got[name], want[name]) for name in want)


@pytest.mark.parametrize("B,nq,nk", [(0, 5, 6), (2, 0, 6), (2, 5, 0)])
def test_attention_empty(B, nq, nk, cuda_device):
    for bias in (None, "shared", "batch"):
        q, k, v, do, bt, _ = _att(B, nq, nk, 2, 2, 32, BF16, cuda_device, bias, F32)
        got = _run(q, k, v, do, bt, None)
        for name, like in (("o", q), ("dq", q), ("dk", k), ("dv", v)):
            assert got[name].shape == like.shape and not got[name].any()
        if bias:
            assert got["dbias"].shape == bt.shape and not got["dbias"].any()


def test_attention_gradients_against_differences(cuda_device):
    """Central differences of <do, o> along random directions, in fp32 with fp64 sums. Steps of 2^-6: the third-order
    term is at most (2 |t'|)^3 h^2 / 6 of the loss's size for logit changes |t'| h, the roundings U n / h."""
    q, k, v, do, bias, mask = _att(2, 30, 40, 2, 1, 32, F32, cuda_device, "shared", F32, "pad")
    got = _run(q, k, v, do, bias, mask)
    h = 2.0 ** -6

    def loss(q, k, v, bias):
        return (do.double() * kernels.attention(q, k, v, bias, mask).double()).sum()

    val, _ = attention_ref(q, k, v, do, bias, mask)
    size = (do.double().abs() * 4.0).sum().item()  # |o| is at most the largest |v|, near 4
    for i, name in enumerate(("dq", "dk", "dv", "dbias")):
        args = [q, k, v, bias]
        u = _rand(args[i].shape, F32, cuda_device, 50 + i, 0.2)
        plus, minus = list(args), list(args)
        plus[i], minus[i] = args[i] + h * u, args[i] - h * u
        num = (loss(*plus) - loss(*minus)) / (2 * h)
        ana = (got[name].double() * u.double()).sum()
        assert abs(num - ana) <= size * (8 * h * h / 6 + 100 * U / h), (name, num.item(), ana.item())


# ------------------------------------------------------------------------------ relative-position bias
def _table(heads, r_max, s_max, dtype, device):
    return _rand((heads, 4 * r_max + 2 * s_max + 7), dtype, device, 9, 0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,heads,chains,r_max,s_max,tile", [
    (1, 1, 1, 32, 2, None), (40, 3, 2, 4, 1, None), (65, 16, 1, 32, 2, None), (300, 5, 4, 8, 2, None),
    (257, 4, 3, 32, 2, (100, 57, 31, 201)), (90, 2, 5, 0, 0, (0, 90, 89, 1)), (130, 6, 2, 200, 3, None),
    (700, 4, 6, 32, 2, None)])
def test_relpos_bias(n, heads, chains, r_max, s_max, tile, dtype, cuda_device):
    ids = token_ids(n, chains, cuda_device)
    row0, rows, col0, cols = tile or (0, n, 0, n)
    hot = relpos_columns(ids, slice(row0, row0 + rows), slice(col0, col0 + cols), r_max, s_max)
    for w_dtype in (F32, BF16):
        w = _table(heads, r_max, s_max, w_dtype, cuda_device)
        out = torch.full((heads, rows, cols), float("nan"), device=cuda_device, dtype=dtype)
        kernels.relpos_bias(w, ids, out, row0, col0, r_max, s_max)
        want = torch.einsum("ijf,hf->hij", hot, w.double())
        size = torch.einsum("ijf,hf->hij", hot, w.double().abs())
        check(out, want, 4 * U * size + want.abs() * half_step(dtype) + 1e-30, "bias")
    g = _rand((heads, rows, cols), dtype, cuda_device, 11)
    dw = kernels.relpos_bias_bwd(g, ids, row0, col0, r_max, s_max)
    want = torch.einsum("ijf,hij->hf", hot, g.double())
    size = torch.einsum("ijf,hij->hf", hot, g.double().abs())
    check(dw, want, (rows * cols + 8) * U * size + 1e-30, "dw")
    assert torch.equal(dw, kernels.relpos_bias_bwd(g, ids, row0, col0, r_max, s_max))


def test_relpos_bias_strided_planes_and_extreme_ids(cuda_device):
    """Planes inside wider ones are written and read in place, their surroundings left alone; ids at the ends of
    int32 do not wrap around."""
    n, heads = 50, 3
    ids = list(token_ids(n, 3, cuda_device))
    lim = torch.iinfo(torch.int32)
    ids[1] = torch.where(torch.arange(n, device=cuda_device) % 2 == 0, lim.min, lim.max).int()
    ids[4] = torch.where(torch.arange(n, device=cuda_device) % 3 == 0, lim.min, lim.max).int()
    hot = relpos_columns(ids, slice(0, n), slice(0, n), 32, 2)
    w = _table(heads, 32, 2, F32, cuda_device)
    wide = torch.full((heads, n + 2, n + 7), 5.0, device=cuda_device)
    kernels.relpos_bias(w, ids, wide[:, 1:n + 1, 3:n + 3], 0, 0, 32, 2)
    want = torch.einsum("ijf,hf->hij", hot, w.double())
    check(wide[:, 1:n + 1, 3:n + 3], want, 4 * U * torch.einsum("ijf,hf->hij", hot, w.double().abs()) + 1e-30, "bias")
    wide[:, 1:n + 1, 3:n + 3] = 5.0
    assert (wide == 5.0).all()
    g = _rand((heads, n + 2, n + 7), F32, cuda_device, 3)[:, 1:n + 1, 3:n + 3]
    dw = kernels.relpos_bias_bwd(g, ids, 0, 0, 32, 2)
    want = torch.einsum("ijf,hij->hf", hot, g.double())
    check(dw, want, (n * n + 8) * U * torch.einsum("ijf,hij->hf", hot, g.double().abs()) + 1e-30, "dw")
    row = _rand((heads, 1, 1), F32, cuda_device, 4).expand(heads, n, 1)  # a broadcast gradient
    dw = kernels.relpos_bias_bwd(row.expand(heads, n, 1), ids, 0, 7, 32, 2)
    want = torch.einsum("ijf,hij->hf", hot[:, 7:8], row.double())
    check(dw, want, 64 * U * torch.einsum("ijf,hij->hf", hot[:, 7:8], row.double().abs()) + 1e-30, "dw")


def test_relpos_gradient_against_differences(cuda_device):
    """The bias is linear in its table, so a difference is exact but for roundings."""
    ids, h = token_ids(60, 2, cuda_device), 0.5
    w, u = _table(4, 32, 2, F32, cuda_device), _rand((4, 139), F32, cuda_device, 1)
    g = _rand((4, 60, 60), F32, cuda_device, 2)
    hi, lo = torch.empty_like(g), torch.empty_like(g)
    kernels.relpos_bias(w + h * u, ids, hi, 0, 0, 32, 2)
    kernels.relpos_bias(w - h * u, ids, lo, 0, 0, 32, 2)
    num = (g.double() * (hi.double() - lo.double())).sum() / (2 * h)
    ana = (kernels.relpos_bias_bwd(g, ids, 0, 0, 32, 2).double() * u.double()).sum()
    assert abs(num - ana) <= g.abs().sum().item() * 16 * (60 * 60 + 16) * U


def test_relpos_empty(cuda_device):
    ids = token_ids(5, 1, cuda_device)
    out = torch.empty(2, 0, 5, device=cuda_device)
    kernels.relpos_bias(_table(2, 32, 2, F32, cuda_device), ids, out, 0, 0, 32, 2)
    assert not kernels.relpos_bias_bwd(out, ids, 0, 0, 32, 2).any()


# ------------------------------------------------------------------------------ streams, graphs, far offsets
def _step(x, w, ids, table, do):
    """Layer norm, relative-position bias, attention and their gradients, as one training step uses them."""
    n, heads, d = x.shape[1], table.shape[0], x.shape[2] // table.shape[0]
    y = kernels.layernorm(x, w, None)
    bias = torch.empty(heads, n, n, device=x.device, dtype=x.dtype)
    kernels.relpos_bias(table, ids, bias, 0, 0, 32, 2)
    qkv = y.view(x.shape[0], n, heads, d)
    o, saved = kernels.attention(qkv, qkv, qkv, bias, save=True)
    dq, dk, dv, db = kernels.attention_bwd(do, qkv, qkv, qkv, o, saved, bias)
    dtable = kernels.relpos_bias_bwd(db, ids, 0, 0, 32, 2)
    dx, dw, _ = kernels.layernorm_bwd(x, (dq + dk + dv).view(x.shape), w, need=(True, True, False))
    return o, dx, dw, dtable


def _step_inputs(dtype, device, seed=0):
    x, w = _rand((6, 70, 128), dtype, device, seed + 1), _rand((128,), F32, device, seed + 2, 0.1) + 1
    return x, w, token_ids(70, 2, device), _table(4, 32, 2, F32, device), _rand((6, 70, 4, 32), dtype, device, seed + 3)


def test_operators_together_against_autograd(cuda_device):
    """The chain in fp32 against fp64 autograd of the same chain; each link's relative error is a few thousand U
    (sums of 70 to 420 terms, logits near 40), and the gradients pass three links."""
    x, w, ids, table, do = _step_inputs(F32, cuda_device)
    X, W, T = (t.double().requires_grad_() for t in (x, w, table))
    xc = X - X.mean(-1, keepdim=True)
    y = xc / torch.sqrt((xc * xc).mean(-1, keepdim=True) + 1e-5) * W
    h = y.view(6, 70, 4, 32).transpose(1, 2)
    bias = torch.einsum("ijf,hf->hij", relpos_columns(ids, slice(0, 70), slice(0, 70), 32, 2), T)
    o = (torch.softmax(h @ h.transpose(2, 3) / math.sqrt(32) + bias, -1) @ h).transpose(1, 2)
    want = (o,) + torch.autograd.grad(o, (X, W, T), do.double())
    for name, got, ref in zip(("o", "dx", "dw", "dtable"), _step(x, w, ids, table, do), want):
        rel = ((got.double() - ref).norm() / ref.norm()).item()
        assert rel <= 4096 * U, (name, rel)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_operators_in_a_graph_and_on_a_stream(dtype, cuda_device):
    """Captured and replayed with new inputs in place; two graphs that share a pool; another stream."""
    ins = _step_inputs(dtype, cuda_device)
    new = _step_inputs(dtype, cuda_device, seed=40)
    first, second = _step(*ins), _step(*new)
    torch.cuda.synchronize()
    live = tuple(t.clone() if torch.is_tensor(t) else t for t in ins)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out1 = _step(*live)
    with torch.cuda.graph(g2, pool=g1.pool()):
        out2 = _step(*new)
    g1.replay()
    assert all(torch.equal(a, b) for a, b in zip(out1, first))
    g2.replay()
    assert all(torch.equal(a, b) for a, b in zip(out2, second))
    for a, b in zip(live, new):
        if torch.is_tensor(a):
            a.copy_(b)
    g1.replay()
    assert all(torch.equal(a, b) for a, b in zip(out1, second))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out3 = _step(*ins)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(out3, first))


def test_offsets_past_32_bits(cuda_device):
    """Keys, a bias and planes whose elements lie more than 2^31 elements apart."""
    buf = torch.zeros((1 << 31) + (1 << 20), device=cuda_device, dtype=BF16)
    n, H, d = 40, 2, 32
    q, k, v, do, bias, _ = _att(2, n, n, H, H, d, BF16, cuda_device, "batch", BF16)
    far = torch.as_strided(buf, (2, n, H, d), (1 << 31, H * d, d, 1))
    far.copy_(k)
    want = _run(q, k, v, do, bias, None)
    got = _run(q, far, v, do, bias, None)
    assert all(torch.equal(got[name], want[name]) for name in want)
    far = torch.as_strided(buf, (2, H, n, n), (1 << 31, n * n, n, 1))
    far.copy_(bias)
    got = _run(q, k, v, do, far, None)
    assert all(torch.equal(got[name], want[name]) for name in want)
    ids, w = token_ids(n, 2, cuda_device), _table(2, 32, 2, F32, cuda_device)
    near, far = torch.empty(2, n, n, device=cuda_device, dtype=BF16), torch.as_strided(buf, (2, n, n), (1 << 31, n, 1))
    kernels.relpos_bias(w, ids, near, 0, 0, 32, 2)
    kernels.relpos_bias(w, ids, far, 0, 0, 32, 2)
    assert torch.equal(near, far)
    assert torch.equal(kernels.relpos_bias_bwd(near, ids, 0, 0, 32, 2), kernels.relpos_bias_bwd(far, ids, 0, 0, 32, 2))
