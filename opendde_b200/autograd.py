"""Differentiable forms of the training operators: layer norm, attention with a learned bias, and the
relative-position bias.

Each is one autograd node over a forward and a backward kernel of :mod:`opendde_b200.kernels` (no CPU fallback,
no second derivatives). The rest of this package stays an inference forward: its modules' ``forward`` builds no
graph, and their ``differentiable`` forms (:class:`~opendde_b200.model.LayerNorm`,
:class:`~opendde_b200.model.AttentionPairBias`, :class:`~opendde_b200.model.TriangleAttention`,
:meth:`~opendde_b200.model.RelativePositionEncoding.head_bias`) are built from these.

A backward pass that autograd runs uses the streams its leaves were first used on, which a CUDA graph capture
cannot follow, so a call that would need a gradient is refused while its stream is being captured: capture the
``kernels`` forward and backward calls themselves, which take their streams from the caller.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import kernels


def _wants_grad(*ts: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _refuse_capture(what: str) -> None:
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: autograd is not captured into a CUDA graph; capture the opendde_b200.kernels "
                           "forward and backward calls instead")


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        ctx.types = tuple(None if p is None else p.dtype for p in (weight, bias))
        with torch.cuda.device(x.device):
            return kernels.layernorm(x, weight, bias, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture("layer_norm")
        x, weight = ctx.saved_tensors
        dx, dw, db = kernels.layernorm_bwd(x, dy, weight, ctx.eps, need=ctx.needs_input_grad[:3])
        return dx, None if dw is None else dw.to(ctx.types[0]), None if db is None else db.to(ctx.types[1]), None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """:func:`kernels.layernorm` with gradients of x [..., c], ``weight`` and ``bias`` [c]."""
    kernels.require_cuda(x, weight, bias)
    for p in (weight, bias):
        if p is not None and (tuple(p.shape) != (x.shape[-1],) or p.device != x.device):
            raise ValueError(f"weight and bias must be [{x.shape[-1]}] on {x.device}")
    if not _wants_grad(x, weight, bias):
        with torch.cuda.device(x.device):
            return kernels.layernorm(x, weight, bias, eps)
    _refuse_capture("layer_norm")
    return _LayerNorm.apply(x, weight, bias, eps)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, mask, scale):
        o, saved = kernels.attention(q, k, v, bias, mask, scale, save=True)
        ctx.save_for_backward(q, k, v, bias, mask, o, *saved)
        ctx.scale = scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        _refuse_capture("attention")
        q, k, v, bias, mask, o, stats, o_lo = ctx.saved_tensors
        do = do if do.stride(-1) == 1 else do.contiguous()
        grads = kernels.attention_bwd(do, q, k, v, o, kernels.AttentionSaved(stats, o_lo), bias, mask, ctx.scale,
                                      need=ctx.needs_input_grad[:4])
        return (*grads, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bias: Optional[torch.Tensor] = None,
              mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """:func:`kernels.attention` with gradients of q, k, v and ``bias`` (any layout: one that the kernels do not
    read in place is copied first)."""
    kernels.require_cuda(q, k, v, bias, mask)
    q, k, v = (t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous() for t in (q, k, v))
    if bias is not None and bias.stride(-1) != 1 and bias.shape[-1] > 1:
        bias = bias.contiguous()
    if not _wants_grad(q, k, v, bias):
        return kernels.attention(q, k, v, bias, mask, scale)
    _refuse_capture("attention")
    return _Attention.apply(q, k, v, bias, None if mask is None else mask.detach(), scale)


class _RelposBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, tile, r_max, s_max, dtype):
        row0, n_rows, col0, n_cols = tile
        out = torch.empty((weight.shape[0], n_rows, n_cols), device=weight.device, dtype=dtype)
        kernels.relpos_bias(weight, ids, out, row0, col0, r_max, s_max)
        ctx.save_for_backward(*ids)
        ctx.args = (row0, col0, r_max, s_max)
        ctx.w_dtype = weight.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        _refuse_capture("relative_position_bias")
        dout = dout if dout.stride(-1) == 1 else dout.contiguous()
        dw = kernels.relpos_bias_bwd(dout, ctx.saved_tensors, *ctx.args)
        return dw.to(ctx.w_dtype), None, None, None, None, None


def relative_position_bias(weight: torch.Tensor, ids, r_max: int, s_max: int, tile=None,
                           dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[H, R, C] bias of attention heads from the relative-position features of the tokens ``ids`` (int32 CUDA
    vectors asym_id, residue_index, entity_id, token_index, sym_id), with the gradient of its table ``weight``
    [H, 4 r_max + 2 s_max + 7]. ``tile`` = (row0, R, col0, C) selects a part of the plane."""
    kernels.require_cuda(weight, *ids)
    n = ids[0].shape[0]
    tile = (0, n, 0, n) if tile is None else tuple(int(t) for t in tile)
    if not _wants_grad(weight):
        with torch.no_grad():
            return _RelposBias.apply(weight, tuple(ids), tile, r_max, s_max, dtype)
    _refuse_capture("relative_position_bias")
    return _RelposBias.apply(weight, tuple(ids), tile, r_max, s_max, dtype)
