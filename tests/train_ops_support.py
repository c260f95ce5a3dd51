"""Plain fp64 forms of the training operators, with bounds on what fp32 and bf16 arithmetic may lose.

A bound counts roundings: U = 2^-24 is half a step of fp32, H = 2^-8 half a step of bf16, each relative to the
value that is rounded. A sum of n terms adds at most n U of the sum of its terms' magnitudes, so every bound is a
count times the same formula with absolute values in it.
"""
import math

import torch

U = 2.0 ** -24
H = 2.0 ** -8


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention_ref(q, k, v, do, bias=None, mask=None, scale=None):
    """fp64 o, dq, dk, dv, dbias and elementwise bounds on their errors, [B, N, H, d] inputs."""
    dt = q.dtype
    bdt = None if bias is None else bias.dtype
    B, nq, heads, d = q.shape
    nk, kv = k.shape[1], k.shape[2]
    rep = heads // kv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    Q, G = (t.double().transpose(1, 2) for t in (q, do))
    K, V = (t.double().transpose(1, 2).repeat_interleave(rep, 1) for t in (k, v))
    seen = torch.ones(B, 1, 1, nk, dtype=torch.bool, device=q.device)
    if mask is not None:
        seen = (mask.reshape(-1, nk) != 0)[:, None, None, :].expand(B, 1, 1, nk)
    K, V = K.masked_fill(~seen.transpose(2, 3), 0.0), V.masked_fill(~seen.transpose(2, 3), 0.0)
    bs = None
    if bias is not None:
        bs = bias.double()
        bs = (bs[None] if bs.dim() == 3 else bs).masked_fill(~seen, 0.0)
    t = Q @ K.transpose(2, 3) * scale
    at = Q.abs() @ K.abs().transpose(2, 3) * scale
    if bs is not None:
        t, at = t + bs, at + bs.abs().masked_fill(bs.abs() == math.inf, 0.0)
    t = t.masked_fill(~seen, -math.inf)
    m = t.amax(-1, keepdim=True) if nk else torch.full((B, heads, nq, 1), -math.inf, device=q.device).double()
    e = torch.exp(t - m.masked_fill(m == -math.inf, 0.0))
    l = e.sum(-1, keepdim=True)
    p = e / l.masked_fill(l == 0, 1.0)
    o = p @ V
    dp = G @ V.transpose(2, 3)
    D = (G * o).sum(-1, keepdim=True)
    ds = p * (dp - D)
    ds_abs = p * (G.abs() @ V.abs().transpose(2, 3) + (G.abs() * (p @ V.abs())).sum(-1, keepdim=True))

    def back(x):   # add the query heads of a key head, [B, N, H, d]
        return x.view(B, kv, rep, nk, d).sum(2).transpose(1, 2)

    def plane(x):  # the bias's own shape
        if bias.dim() == 3 or bias.shape[0] == 1:
            return x.sum(0).view(bias.shape)
        return x

    val = {"o": o.transpose(1, 2), "dq": (ds @ K * scale).transpose(1, 2),
           "dk": back(ds.transpose(2, 3) @ Q * scale), "dv": back(p.transpose(2, 3) @ G)}
    # logits: d products and sums, the scale and the bias; then the exponential (its argument's difference and
    # factor; a few steps of the function) and the row's sum
    top = float(at.masked_fill(~seen, 0.0).max()) if at.numel() else 0.0
    logit = 2 * (d + 6) * U * top
    base = 2 * logit + (2 * nk + 2 * d + 64) * U
    op = H if dt == torch.bfloat16 else 0.0  # p and ds as operands of the second product
    eps = base + op + (nk + nq * rep) * U
    absv = {"o": (p @ V.abs()).transpose(1, 2), "dq": (ds_abs @ K.abs() * scale).transpose(1, 2),
            "dk": back(ds_abs.transpose(2, 3) @ Q.abs() * scale), "dv": back(p.transpose(2, 3) @ G.abs())}
    bound = {n: absv[n] * eps + val[n].abs() * half_step(dt) + 1e-30 for n in val}
    if bias is not None:
        val["dbias"] = plane(ds)
        bound["dbias"] = plane(ds_abs) * (base + B * U) + val["dbias"].abs() * half_step(bdt) + 1e-30
    return val, bound


def layernorm_ref(x, dy, w, eps):
    """fp64 dx, dw, db and bounds on their errors."""
    X, G = x.double(), dy.double()
    X, G = X.reshape(-1, X.shape[-1]), G.reshape(-1, G.shape[-1])
    rows, c = X.shape
    W = torch.ones(c, device=x.device, dtype=torch.float64) if w is None else w.double()
    mean = X.mean(-1, keepdim=True)
    xc = X - mean
    s = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xh = xc * s
    g = G * W
    dx = s * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    # the mean is off by c U of the largest element, which moves every xh by that times s; the rest is relative
    shift = 2 * (c + 8) * U * X.abs().amax(-1, keepdim=True) * s
    rel = (4 * c + 64) * U
    ah = xh.abs() + shift
    dx_abs = s * (g.abs() + g.abs().mean(-1, keepdim=True) + ah * (g.abs() * ah).mean(-1, keepdim=True))
    move = s * shift * ((g.abs() * ah).mean(-1, keepdim=True) + ah * g.abs().mean(-1, keepdim=True))
    move = move + dx.abs() * shift  # rstd moves with the mean
    val = {"dx": dx.view(x.shape), "dw": (G * xh).sum(0), "db": G.sum(0)}
    bound = {"dx": (dx_abs * rel + move).view(x.shape) + val["dx"].abs() * half_step(x.dtype) + 1e-30,
             "dw": (G.abs() * (xh.abs() * (rows + rel / U) * U + shift * (1 + ah))).sum(0) + 1e-30,
             "db": G.abs().sum(0) * (rows + 4) * U + 1e-30}
    return val, bound


def relpos_columns(ids, rows, cols, r_max, s_max):
    """The one-hot features [R, C, F] (fp64) of the pairs, from the definition."""
    asym, res, ent, tok, sym = (t.long() for t in ids)

    def diff(t):
        return t[rows][:, None] - t[cols][None, :]

    def hot(at, n):
        return torch.nn.functional.one_hot(at, n).double()

    chain, entity = diff(asym) == 0, diff(ent) == 0
    a = torch.where(chain, diff(res).clamp(-r_max, r_max) + r_max, 2 * r_max + 1)
    b = torch.where(chain & (diff(res) == 0), diff(tok).clamp(-r_max, r_max) + r_max, 2 * r_max + 1)
    s = torch.where(entity, diff(sym).clamp(-s_max, s_max) + s_max, 2 * s_max + 1)
    return torch.cat([hot(a, 2 * r_max + 2), hot(b, 2 * r_max + 2), entity[..., None].double(),
                      hot(s, 2 * s_max + 2)], -1)


def check(got, val, bound, what=""):
    """Every element of ``got`` within its bound of ``val``."""
    assert got.shape == val.shape, (what, got.shape, val.shape)
    if got.numel() == 0:
        return
    far = (got.double() - val).abs()
    bad = ~(far <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} elements, worst {float((far / bound).max()):.2f} "
                           f"bounds at {tuple(int(i) for i in bad.nonzero()[0])}")


def token_ids(n, chains, device, seed=0):
    """Random chains of tokens: ids of several chains, entities and symmetry copies, multi-token residues."""
    g = torch.Generator().manual_seed(seed)
    asym = torch.sort(torch.randint(0, chains, (n,), generator=g)).values
    res = torch.cumsum(torch.randint(0, 2, (n,), generator=g), 0)
    tok = torch.arange(n)
    return tuple(t.to(device=device, dtype=torch.int32) for t in (asym, res, asym // 2, tok, asym % 2))
