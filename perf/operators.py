"""Training operators of the pair stack, as calls to measure and check.

Three operators that are used together when a Pairformer layer is trained: the layer norm with its
backward pass, attention with a learned bias and its backward pass (which recomputes the
probabilities), and the relative-position bias with the gradient of its table. One pass of a case is
the forward call followed by the backward call.

``own`` selects between the plain form (elementary torch operations in fp32 or fp64, rounded once at
the end) and this package's kernels. ``exact`` is the definition in fp64, written separately.
"""

import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_DEV = "cuda"


# ------------------------------------------------------------------------------ cases

def _ln(rows, c, dtype, affine):
    return {"op": "layernorm", "rows": rows, "c": c, "dtype": dtype, "affine": affine}


def _att(batch, n_q, n_k, heads, kv_heads, d, dtype, bias, bias_dtype, mask, packed):
    return {"op": "attention", "batch": batch, "n_q": n_q, "n_k": n_k, "heads": heads, "kv_heads": kv_heads, "d": d,
            "dtype": dtype, "bias": bias, "bias_dtype": bias_dtype, "mask": mask, "packed": packed}


def _rel(n, row0, rows, col0, cols, heads, chains, copies, dtype):
    return {"op": "relpos", "n": n, "row0": row0, "rows": rows, "col0": col0, "cols": cols, "heads": heads,
            "chains": chains, "copies": copies, "dtype": dtype}


def listed():
    cases = [
        # the single representation of a small complex (c_s = 384): launch latency
        ("ln_single_n64_c384_f32", _ln(64, 384, "f32", "full")),
        # the pair representation of a 384-token training crop (c_z = 128)
        ("ln_pair_n384_c128_bf16", _ln(384 * 384, 128, "bf16", "full")),
        # the 449 input features of a ragged batch of tokens: rows that are no whole 16-byte vectors
        ("ln_features_n20011_c449_f32", _ln(20011, 449, "f32", "scale")),
        # the pair representation of the 1536-token benchmark input
        ("ln_pair_n1536_c128_bf16", _ln(1536 * 1536, 128, "bf16", "full")),
        # single attention of a tiny chain (16 heads of 24), fp32: launch latency
        ("att_single_n13_h16_d24_f32", _att(1, 13, 13, 16, 16, 24, "f32", "batch", "f32", "none", False)),
        # single attention of the 1536-token input with its fp32 pair bias: bound by the bias
        ("att_single_n1536_h16_d24_bf16", _att(1, 1536, 1536, 16, 16, 24, "bf16", "batch", "f32", "none", False)),
        # triangle attention of a 256-token crop: 256 rows share one bias, the last tenth is padding
        ("att_tri_n256_h4_d32_bf16", _att(256, 256, 256, 4, 4, 32, "bf16", "shared", "bf16", "pad", False)),
        # triangle attention of the 768-token input: the largest
        ("att_tri_n768_h4_d32_bf16", _att(768, 768, 768, 4, 4, 32, "bf16", "shared", "bf16", "pad", False)),
        # triangle attention of the structural refiner's width (12 heads of 32) in fp32, an odd length
        ("att_tri_n149_h12_d32_f32", _att(149, 149, 149, 12, 12, 32, "f32", "shared", "f32", "holes", False)),
        # a padded batch of sequences over one packed projection, no bias, two key heads for eight
        ("att_batch3_n301_517_h8_kv2_d64_bf16", _att(3, 301, 517, 8, 2, 64, "bf16", "none", "f32", "pad", True)),
        # the relative-position bias of a small complex: launch latency
        ("relpos_n64_h16_f32", _rel(64, 0, 64, 0, 64, 16, 1, 1, "f32")),
        # the 1536-token input, four chains in two symmetric copies
        ("relpos_n1536_h16_f32", _rel(1536, 0, 1536, 0, 1536, 16, 4, 2, "f32")),
    ]
    return [dict(case, name=name) for name, case in cases]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layernorm", "attention", "attention", "relpos"])
    if op == "layernorm":
        c = rng.choice([16, 37, 64, 128, 128, 139, 256, 384, 449, 512, 768, 1001, 1024, rng.randint(1, 1024)])
        dtype = rng.choice(["f32", "bf16", "bf16"])
        most = 1536 * 1536 * (128 if dtype == "bf16" else 64)
        return _ln(_log(rng, 1, min(1 << 21, most // max(c, 64))), c, dtype,
                   rng.choice(["full", "full", "scale", "none"]))
    if op == "attention":
        dtype = rng.choice(["f32", "bf16", "bf16"])
        most = (768 ** 3) * 4 * 32 if dtype == "bf16" else (256 ** 3) * 4 * 32
        form = rng.choice(["single", "triangle", "triangle", "batch"])
        if form == "single":     # one sequence, a bias per head, many heads
            heads = rng.choice([4, 8, 16])
            d = rng.choice([24, 32, 48])
            n = _log(rng, 1, 2000)
            n_q = n if rng.random() < 0.6 else rng.randint(1, n)
            case = _att(1, n_q, n, heads, heads, d, dtype, "batch", rng.choice(["f32", "f32", "bf16"]),
                        rng.choice(["none", "none", "holes"]), False)
        elif form == "triangle":  # n rows of n tokens share one bias
            heads, d = rng.choice([(4, 32), (4, 32), (2, 32), (12, 32), (8, 16)])
            n = _log(rng, 2, 640)
            case = _att(n, n, n, heads, heads, d, dtype, "shared", rng.choice([dtype, "f32"]),
                        rng.choice(["none", "pad", "holes"]), False)
        else:                    # a padded batch of sequences, with or without shared key heads
            kv = rng.choice([1, 2, 4])
            heads = kv * rng.choice([1, 2, 4])
            case = _att(rng.randint(1, 6), _log(rng, 1, 1500), _log(rng, 1, 1500), heads, kv,
                        rng.choice([8, 40, 64, 96, 128]), dtype, rng.choice(["none", "shared", "batch"]),
                        rng.choice(["f32", dtype]), rng.choice(["none", "pad", "holes"]), False)
        while (case["batch"] * case["n_q"] * case["n_k"] * case["heads"] * case["d"] > most
               or case["bias"] == "batch" and case["batch"] * case["n_q"] * case["n_k"] * case["heads"] > 1 << 27):
            for k in ("batch", "n_q", "n_k"):
                case[k] = max(1, (case[k] * 3) // 4)
        if form == "triangle":
            case["batch"] = case["n_q"] = case["n_k"]
        return case
    n = _log(rng, 1, 1536)
    heads = rng.choice([1, 4, 4, 12, 16, 16])
    if rng.random() < 0.6:
        row0, rows, col0, cols = 0, n, 0, n
    else:                        # the tile of a mesh position
        rows, cols = rng.randint(1, n), rng.randint(1, n)
        row0, col0 = rng.randint(0, n - rows), rng.randint(0, n - cols)
    return _rel(n, row0, rows, col0, cols, heads, rng.randint(1, min(6, n)), rng.randint(1, 3),
                rng.choice(["f32", "f32", "bf16"]))


# ------------------------------------------------------------------------------ inputs

_R_MAX, _S_MAX = 32, 2


def _token_ids(case, gen):
    """asym_id, residue_index, entity_id, token_index, sym_id of ``chains`` chains, every ``copies``
    of them copies of one entity; some residues are modified and span several tokens."""
    n, chains = case["n"], case["chains"]
    cuts = sorted((torch.randperm(n - 1, generator=gen)[:chains - 1] + 1).tolist()) if chains > 1 else []
    bounds = [0] + cuts + [n]
    span = torch.rand(n, generator=gen)
    asym, res, ent, tok, sym = [], [], [], [], []
    for ch in range(chains):
        r, left = 0, 0
        for t in range(bounds[ch], bounds[ch + 1]):
            if left == 0:
                r += 1
                left = 1 if span[t] > 0.05 else 7  # an atomised residue of seven tokens
            left -= 1
            asym.append(ch)
            res.append(r)
            ent.append(ch // case["copies"])
            tok.append(t)
            sym.append(ch % case["copies"])
    return tuple(torch.tensor(v, dtype=torch.int32, device=_DEV) for v in (asym, res, ent, tok, sym))


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=_DEV).manual_seed(seed)

    def rand(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(shape, generator=g, device=_DEV, dtype=torch.float32) * std).to(dtype)

    op = case["op"]
    if op == "layernorm":
        dt, rows, c = _DT[case["dtype"]], case["rows"], case["c"]
        st = {"x": rand(rows, c, dtype=dt, std=1.5), "dy": rand(rows, c, dtype=dt), "w": None, "b": None}
        st["x"] += 0.25
        if case["affine"] != "none":
            st["w"] = 1.0 + rand(c, std=0.1)
        if case["affine"] == "full":
            st["b"] = rand(c, std=0.1)
    elif op == "attention":
        dt, bdt = _DT[case["dtype"]], _DT[case["bias_dtype"]]
        B, nq, nk, H, KV, d = (case[k] for k in ("batch", "n_q", "n_k", "heads", "kv_heads", "d"))
        st = {"q": rand(B, nq, H, d, dtype=dt, std=1.2), "do": rand(B, nq, H, d, dtype=dt)}
        if case["packed"]:       # keys and values side by side, as one projection writes them
            kv = rand(B, nk, 2, KV, d, dtype=dt, std=1.1)
            st["k"], st["v"] = kv[:, :, 0], kv[:, :, 1]
        else:
            st["k"], st["v"] = rand(B, nk, KV, d, dtype=dt, std=1.2), rand(B, nk, KV, d, dtype=dt)
        st["bias"] = None
        if case["bias"] != "none":
            st["bias"] = rand(1 if case["bias"] == "shared" else B, H, nq, nk, dtype=bdt)
        st["mask"] = None
        if case["mask"] == "pad":      # padded tokens: the last tenth of the keys, and the rows past it
            mask = torch.ones(B, nk, device=_DEV)
            mask[:, nk - nk // 10:] = 0
            if case["bias"] == "shared":
                mask[B - B // 10:] = 0
            st["mask"] = mask
        elif case["mask"] == "holes":  # unresolved positions; one row of the batch sees nothing
            mask = (torch.rand((B, nk), generator=g, device=_DEV) >= 0.1).float()
            if B > 1:
                mask[B // 2] = 0
            st["mask"] = mask
    else:
        H = case["heads"]
        st = {"ids": _token_ids(case, gen), "w": rand(H, 4 * _R_MAX + 2 * _S_MAX + 7, std=0.3),
              "dbias": rand(H, case["rows"], case["cols"], dtype=_DT[case["dtype"]])}
    st["case"] = case
    return st


# ------------------------------------------------------------------------------ plain forms

def _plain_layernorm(st):
    x, dy, c = st["x"].float(), st["dy"].float(), st["x"].shape[-1]
    dt = st["x"].dtype
    mean = x.sum(-1, keepdim=True) / c
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).sum(-1, keepdim=True) / c + 1e-5)
    xh = xc * rstd
    y = xh if st["w"] is None else xh * st["w"]
    if st["b"] is not None:
        y = y + st["b"]
    g = dy if st["w"] is None else dy * st["w"]
    m1 = g.sum(-1, keepdim=True) / c
    m2 = (g * xh).sum(-1, keepdim=True) / c
    out = [y.to(dt), ((g - m1 - xh * m2) * rstd).to(dt)]
    if st["w"] is not None:
        out.append((dy * xh).sum(0, dtype=torch.float64).float())
    if st["b"] is not None:
        out.append(dy.sum(0, dtype=torch.float64).float())
    return out


def _plain_attention(st):
    q, k, v, do, bias, mask = (st[n] for n in ("q", "k", "v", "do", "bias", "mask"))
    B, nq, H, d = q.shape
    nk, KV = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d)
    o, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.empty(k.shape, dtype=k.dtype, device=k.device), \
        torch.empty(v.shape, dtype=v.dtype, device=v.device)
    db = None if bias is None else torch.zeros(bias.shape, device=q.device)
    step = max(1, min(B, (1 << 29) // max(1, H * nq * nk)))  # rows of the batch at a time: 2 GB a score tensor
    for b0 in range(0, B, step):
        s = slice(b0, min(B, b0 + step))
        qs, gs = q[s].float().transpose(1, 2), do[s].float().transpose(1, 2)
        ks = k[s].float().transpose(1, 2).repeat_interleave(H // KV, dim=1)
        vs = v[s].float().transpose(1, 2).repeat_interleave(H // KV, dim=1)
        t = torch.matmul(qs, ks.transpose(2, 3)) * scale
        shared = bias is not None and bias.shape[0] == 1
        if bias is not None:
            t = t + (bias if shared else bias[s]).float()
        if mask is not None:
            t = torch.where((mask[s] != 0)[:, None, None, :], t, -math.inf)
        m = t.amax(-1, keepdim=True)
        p = torch.exp(t - torch.where(m == -math.inf, 0.0, m))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        o[s] = torch.matmul(p, vs).transpose(1, 2).to(o.dtype)
        dp = torch.matmul(gs, vs.transpose(2, 3))
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        dq[s] = (torch.matmul(ds, ks) * scale).transpose(1, 2).to(dq.dtype)
        n = ds.shape[0]
        dkf = torch.matmul(ds.transpose(2, 3), qs) * scale
        dvf = torch.matmul(p.transpose(2, 3), gs)
        dk[s] = dkf.view(n, KV, H // KV, nk, d).sum(2).transpose(1, 2).to(dk.dtype)
        dv[s] = dvf.view(n, KV, H // KV, nk, d).sum(2).transpose(1, 2).to(dv.dtype)
        if shared:
            db += ds.sum(0, keepdim=True)
        elif bias is not None:
            db[s] = ds
    out = [o, dq, dk, dv]
    if bias is not None:
        out.append(db.to(bias.dtype))
    return out


def _features(case, ids):
    """The residue, token and symmetry-copy columns of each pair of the tile, and its same-entity bit."""
    R, S = _R_MAX, _S_MAX
    asym, res, ent, tok, sym = (t.long() for t in ids)
    i = slice(case["row0"], case["row0"] + case["rows"])
    j = slice(case["col0"], case["col0"] + case["cols"])

    def diff(t):
        return t[i][:, None] - t[j][None, :]

    chain, same_ent = diff(asym) == 0, diff(ent) == 0
    f_res = torch.where(chain, (diff(res) + R).clamp(0, 2 * R), 2 * R + 1)
    f_tok = torch.where(chain & (diff(res) == 0), (diff(tok) + R).clamp(0, 2 * R), 2 * R + 1) + 2 * R + 2
    f_sym = torch.where(same_ent, (diff(sym) + S).clamp(0, 2 * S), 2 * S + 1) + 4 * R + 5
    return f_res, f_tok, f_sym, same_ent


def _plain_relpos(st):
    case, w, g = st["case"], st["w"], st["dbias"]
    H, F = w.shape
    R = _R_MAX
    f_res, f_tok, f_sym, same = _features(case, st["ids"])
    bias = w[:, f_res] + w[:, f_tok] + w[:, f_sym] + w[:, 4 * R + 4][:, None, None] * same
    dw = torch.zeros(H, F, dtype=torch.float64, device=w.device)
    cols = torch.arange(F, device=w.device)
    for r in range(0, case["rows"], 64):
        s = slice(r, min(case["rows"], r + 64))
        hot = sum((f[s].reshape(-1)[:, None] == cols).double() for f in (f_res, f_tok, f_sym))
        hot[:, 4 * R + 4] = same[s].reshape(-1).double()
        dw += torch.matmul(g[:, s].reshape(H, -1).double(), hot)
    return [bias.to(g.dtype), dw.float()]


# ------------------------------------------------------------------------------ the measured pass

def run(state):
    op = state["case"]["op"]
    if not own:
        return {"layernorm": _plain_layernorm, "attention": _plain_attention, "relpos": _plain_relpos}[op](state)
    from opendde_b200 import kernels
    if op == "layernorm":
        y = kernels.layernorm(state["x"], state["w"], state["b"])
        grads = kernels.layernorm_bwd(state["x"], state["dy"], state["w"], need=(True, state["w"] is not None,
                                                                              state["b"] is not None))
        return [y] + [t for t in grads if t is not None]
    if op == "attention":
        q, k, v, bias, mask = (state[n] for n in ("q", "k", "v", "bias", "mask"))
        o, saved = kernels.attention(q, k, v, bias, mask, save=True)
        grads = kernels.attention_bwd(state["do"], q, k, v, o, saved, bias, mask)
        return [o] + [t for t in grads if t is not None]
    case, g = state["case"], state["dbias"]
    bias = torch.empty_like(g)
    kernels.relpos_bias(state["w"], state["ids"], bias, case["row0"], case["col0"], _R_MAX, _S_MAX)
    return [bias, kernels.relpos_bias_bwd(g, state["ids"], case["row0"], case["col0"], _R_MAX, _S_MAX)]


def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "f32" else 2
    if op == "layernorm":        # x, dy in; y, dx out
        return {"bytes": 4 * case["rows"] * case["c"] * size, "flops": 16 * case["rows"] * case["c"]}
    if op == "attention":        # q, k, v, do, bias, mask in; o, dq, dk, dv, dbias out; two products, then five
        B, nq, nk, H, KV, d = (case[k] for k in ("batch", "n_q", "n_k", "heads", "kv_heads", "d"))
        nbytes = size * B * d * (4 * nq * H + 4 * nk * KV)
        if case["bias"] != "none":
            nbytes += 2 * (1 if case["bias"] == "shared" else B) * H * nq * nk * (4 if case["bias_dtype"] == "f32" else 2)
        if case["mask"] != "none":
            nbytes += 4 * B * nk
        return {"bytes": nbytes, "flops": 7 * 2 * B * H * nq * nk * d}
    pairs = case["rows"] * case["cols"]  # dbias in, bias out
    return {"bytes": 2 * size * case["heads"] * pairs + 2 * 4 * case["heads"] * (4 * _R_MAX + 2 * _S_MAX + 7),
            "flops": 7 * case["heads"] * pairs}


# ------------------------------------------------------------------------------ the definition in fp64

def _exact_layernorm(st):
    x = st["x"].double().requires_grad_()
    w = None if st["w"] is None else st["w"].double().requires_grad_()
    b = None if st["b"] is None else st["b"].double().requires_grad_()
    var, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
    y = (x - mean) * (var + 1e-5).rsqrt()
    y = y if w is None else y * w
    y = y if b is None else y + b
    leaves = [t for t in (x, w, b) if t is not None]
    return [y.detach()] + list(torch.autograd.grad(y, leaves, st["dy"].double()))


def _exact_attention(st):
    case = st["case"]
    B, H, KV, d = case["batch"], case["heads"], case["kv_heads"], case["d"]
    step = max(1, min(B, (1 << 28) // max(1, H * case["n_q"] * case["n_k"])))
    bias = None if st["bias"] is None else st["bias"].double().requires_grad_()
    outs, grads = [], []
    db = None if bias is None else torch.zeros_like(bias)
    for b0 in range(0, B, step):
        s = slice(b0, min(B, b0 + step))
        q, k, v = (st[n][s].double().requires_grad_() for n in ("q", "k", "v"))
        n = q.shape[0]
        qg = q.view(n, case["n_q"], KV, H // KV, d)
        t = torch.einsum("bigrd,bjgd->bgrij", qg, k).reshape(n, H, case["n_q"], case["n_k"]) / math.sqrt(d)
        if bias is not None:
            t = t + (bias if bias.shape[0] == 1 else bias[s])
        if st["mask"] is not None:
            seen = (st["mask"][s] != 0)[:, None, None, :]
            p = torch.softmax(t.masked_fill(~seen, -1e300), dim=-1) * seen  # a row that sees nothing: all zero
        else:
            p = torch.softmax(t, dim=-1)
        o = torch.einsum("bgrij,bjgd->bigrd", p.reshape(n, KV, H // KV, case["n_q"], case["n_k"]), v)
        o = o.reshape(n, case["n_q"], H, d)
        leaves = [q, k, v] + ([] if bias is None else [bias])
        got = torch.autograd.grad(o, leaves, st["do"][s].double())
        outs.append(o.detach())
        grads.append(got[:3])
        if bias is not None:
            db += got[3]
    res = [torch.cat(outs)] + [torch.cat([g[i] for g in grads]) for i in range(3)]
    return res if bias is None else res + [db]


def _exact_relpos(st):
    case, w, g = st["case"], st["w"].double(), st["dbias"].double()
    R, S = _R_MAX, _S_MAX
    H, F = w.shape
    asym, res, ent, tok, sym = (t.double() for t in st["ids"])
    rows = torch.arange(case["row0"], case["row0"] + case["rows"], device=w.device)
    cols = torch.arange(case["col0"], case["col0"] + case["cols"], device=w.device)
    i, j = torch.meshgrid(rows, cols, indexing="ij")
    apart = asym[i] != asym[j]
    table = torch.zeros(H, F, dtype=torch.float64, device=w.device)
    bias = torch.zeros_like(g)
    off = 0
    for val, other, reach in ((res, apart, R), (tok, apart | (res[i] != res[j]), R), (None, ent[i] == ent[j], 0),
                              (sym, ent[i] != ent[j], S)):
        if val is None:
            bias += w[:, off, None, None] * other
            table[:, off] = (g * other).sum((1, 2))
            off += 1
            continue
        at = torch.minimum(torch.maximum(val[i] - val[j], torch.tensor(-float(reach), device=w.device)),
                           torch.tensor(float(reach), device=w.device)) + reach
        at = torch.where(other, 2.0 * reach + 1, at).long().reshape(-1)
        for h in range(H):
            table[h, off:off + 2 * reach + 2] = torch.bincount(at, weights=g[h].reshape(-1), minlength=2 * reach + 2)
            bias[h] += w[h, off + at].view(bias[h].shape)
        off += 2 * reach + 2
    return [bias, table]


def exact(case, seed):
    st = prepare(case, seed)
    return {"layernorm": _exact_layernorm, "attention": _exact_attention, "relpos": _exact_relpos}[case["op"]](st)
