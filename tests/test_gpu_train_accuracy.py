"""Attention and its gradients against fp64 in the 2-norm (bounds: train_accuracy_support.py)."""
import pytest
import torch

from test_gpu_train_ops import _att, _run
from train_accuracy_support import BF16_TOL, FP32_TOL, distance
from train_ops_support import attention_ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("B,nq,nk,H,KV,d,bias,bias_dtype,mask", [
    (160, 160, 160, 4, 4, 32, "shared", BF16, "pad"),     # dq and the plane's gradient in one pass
    (40, 100, 900, 4, 4, 32, "shared", F32, None),        # apart, the plane past what one pass holds
    (1, 700, 700, 16, 16, 24, "batch", F32, None), (64, 200, 190, 4, 2, 32, None, None, "holes"),
    (6, 300, 257, 8, 8, 64, "batch", BF16, "pad"), (5, 200, 320, 8, 2, 96, None, None, None),
    (4, 300, 300, 8, 8, 128, "shared", F32, "pad"), (1, 40, 45, 2, 2, 32, "batch", BF16, None)])
def test_bf16_outputs_are_rounded_once(B, nq, nk, H, KV, d, bias, bias_dtype, mask, cuda_device):
    """Whatever the size of the problem and the kernels that it takes: nothing but the rounding to bf16 shows."""
    args = _att(B, nq, nk, H, KV, d, BF16, cuda_device, bias, bias_dtype, mask)
    val, _ = attention_ref(*args)
    got = _run(*args)
    far = {name: distance(got[name], val[name]) for name in val}
    tol = {name: FP32_TOL if got[name].dtype == F32 else BF16_TOL for name in far}
    assert all(far[name] <= tol[name] for name in far), far


@pytest.mark.parametrize("B,nq,nk,H,KV,d,bias,bias_dtype,mask", [
    (1, 13, 13, 16, 16, 24, "batch", F32, None), (60, 149, 149, 4, 4, 32, "shared", F32, "holes"),
    (20, 70, 600, 4, 4, 32, "shared", F32, "pad"), (1, 900, 1500, 2, 2, 32, "batch", F32, None),
    (3, 200, 190, 4, 2, 64, "batch", BF16, "pad"), (10, 65, 70, 2, 1, 64, "shared", F32, None),
    (2, 90, 130, 4, 4, 128, "batch", F32, None), (9, 100, 67, 2, 2, 96, "shared", F32, "holes"),
    (2, 130, 200, 8, 2, 100, None, None, None)])
def test_fp32_outputs(B, nq, nk, H, KV, d, bias, bias_dtype, mask, cuda_device):
    """Every output keeps fp32's bits: a lost term of a split or product is off by several times the bound."""
    args = _att(B, nq, nk, H, KV, d, F32, cuda_device, bias, bias_dtype, mask)
    val, _ = attention_ref(*args)
    got = _run(*args)
    # a bf16 bias's gradient is rounded to bf16: a border is crossed with probability |error| / step
    far = {name: distance(got[name], val[name]) / (FP32_TOL if got[name].dtype == F32 else (2.0 ** -7 * FP32_TOL) ** 0.5)
           for name in val}
    assert all(x <= 1 for x in far.values()), far


def test_fp32_outputs_of_small_operands(cuda_device):
    """Operands keep their 24 bits down to 2^-110 and an absolute error of 2^-134 below, half of bf16's least step."""
    q, k, v, do, bias, mask = _att(2, 70, 80, 2, 2, 32, F32, cuda_device, "batch", F32, "pad")
    for args in ((q, k, v, do * 2.0 ** -108, bias, mask), (q, k, v * 2.0 ** -108, do, bias, mask),
                 (q, k * 2.0 ** -108, v, do, bias, mask)):
        val, _ = attention_ref(*args)
        got = _run(*args)
        # ds has the spread of p in it: its smaller values lie 2^-6 and more below do
        assert all(distance(got[name], val[name]) <= FP32_TOL for name in val)
    args = (q, k, v * 2.0 ** -118, do, bias, mask)
    val, bound = attention_ref(*args)
    # o is a mean of v; its own rounding to a subnormal number is below 2^-149
    assert ((_run(*args)["o"].double() - val["o"]).abs() <= bound["o"] - 1e-30 + 2.0 ** -134 + 2.0 ** -149).all()
