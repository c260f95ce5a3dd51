"""How far attention's outputs may be from fp64 in the 2-norm, and where a lost term of a split shows.

The elementwise bounds of train_ops_support.py count every rounding at its worst, which leaves room for an operand cut
to half of its bits. Errors that are independent add as squares, so the norm of a whole output is far tighter.
"""
import math

import torch

U = 2.0 ** -24

# fp32, and the fp32 gradient of a bias: a score is a sum of d products (each off by at most three dropped products of
# order U) next to a bias, with errors of order U of its size, here a few units; p, dp, D and the second sums each add
# an error of order U. Eight such sources of at most 4 U, independent: sqrt(8) 4 U = 11 U, and 16 U with the scores'
# size. An operand of two terms is off by 2^-17 = 128 U at most, by a third of that on average.
FP32_TOL = 16 * U

# bf16: an output that is off by a relative error e before its rounding (2-norm) differs from the rounded fp64 value
# where a border between two bf16 values lies between them: with probability |error| / step, and then by a step of at
# most 2^-7. The square of the distance is therefore 2^-7 e on average. p and ds of two terms are off by at most
# 2^-17, o's error in D by as much: e <= 2^-15. One term (2^-9 or more on average, e = 1.6e-3) gives 3.5e-3.
BF16_TOL = math.sqrt(2.0 ** -7 * 2.0 ** -15)


def distance(got, val):
    """2-norm of ``got`` less the fp64 ``val`` rounded to its type, relative to val's."""
    return ((got.double() - val.to(got.dtype).double()).norm() / val.norm().clamp_min(1e-300)).item()


def split(x, terms):
    """x as a list of ``terms`` bf16 values (held in fp64) that add up to it as far as they can."""
    out, rest = [], x.double()
    for _ in range(terms):
        out.append(rest.to(torch.bfloat16).double())
        rest = rest - out[-1]
    return out


def product(a, b, terms):
    """a @ b of operands split into ``terms`` bf16 values, products past the ``terms``-th order left out."""
    a, b = split(a, terms), split(b, terms)
    return sum(a[i] @ b[j] for i in range(terms) for j in range(terms) if i + j < terms)


def split_attention(q, k, v, do, bias, terms):
    """o, dq, dk, dv, dbias [B, H, N, d] with every operand of a product split; all else in fp64."""
    scale = 1.0 / math.sqrt(q.shape[-1])
    p = torch.softmax(product(q, k.transpose(2, 3), terms) * scale + bias.double(), -1)
    o = product(p, v, terms)
    ds = p * (product(do, v.transpose(2, 3), terms) - (do.double() * o).sum(-1, keepdim=True))
    return {"o": o, "dq": product(ds, k, terms) * scale, "dk": product(ds.transpose(2, 3), q, terms) * scale,
            "dv": product(p.transpose(2, 3), do, terms), "dbias": ds}
