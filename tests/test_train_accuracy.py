"""The bounds of train_accuracy_support.py on the CPU: an emulation of the split operands passes with three terms and
fails with two, in every output."""
import pytest
import torch

from train_accuracy_support import FP32_TOL, distance, split_attention
from train_ops_support import attention_ref


@pytest.mark.parametrize("n,d,H", [(13, 24, 4), (67, 32, 2), (200, 64, 2), (90, 128, 1)])
def test_a_lost_term_is_noticed(n, d, H):
    g = torch.Generator().manual_seed(n)
    q, k, v, do = (torch.randn(2, n, H, d, generator=g) * s for s in (1.3, 1.2, 1.0, 1.0))
    bias = torch.randn(2, H, n, n, generator=g)
    val, _ = attention_ref(q, k, v, do, bias)
    for terms, passes in ((3, True), (2, False)):
        got = split_attention(*(t.transpose(1, 2) for t in (q, k, v, do)), bias, terms)
        for name, x in got.items():
            x = x if name == "dbias" else x.transpose(1, 2)
            assert (distance(x.float(), val[name]) <= FP32_TOL) == passes, (terms, name)
