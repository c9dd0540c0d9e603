"""The residual block around the routed layer: x + gate * N(moe(N(x) * (1 + scale) + shift)), the second half of the
reference's denoiser block (aurora/model.py:191-210) with MoESwiGLU as its mlp.

  norm_modulate   the RMS norm before a block with its weight and per-sample scale / shift, differentiable
  norm_residual   the RMS norm behind a block (or none), the gate and the scaled residual, differentiable
  moe_residual    both around the routed layer as one autograd node: the sum over the routed slots is taken inside the norm
                  behind (no combined copy of the layer's output), and the gradient of the residual joins the backward of
                  the norm before
  MoEResidual     the module

Rows come as (T, d), or (..., d) with leading dimensions that are flattened; per-sample parameters are (B, d) for equal runs
of rows -- (B, L, d) inputs, whose first dimensions they have to match -- or with starts (B + 1,) int32 for packed samples of
unequal lengths, (d,) for all rows.
Rows outside the samples are padding: their residual passes through and nothing else does."""
from __future__ import annotations

from dataclasses import replace

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import ops
from .layer import MoESwiGLU, _check_checkpoint, _experts_backward, _experts_forward, _experts_infer, _few, _few_infer, _recorded


def _flat(x):
    """x's rows as a matrix the kernels take: a view where its rows lie in one stride of a multiple of 8, else a copy."""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1 or x2.shape[0] > 1 and (x2.stride(0) < x2.shape[1] or x2.stride(0) % 8):
        x2 = x2.contiguous()
    return x2 if x2.data_ptr() % 16 == 0 else x2.clone(memory_format=torch.contiguous_format)


def _dense(t):
    """A contiguous, 16-byte aligned tensor with t's values."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _par(t):
    return None if t is None else _dense(t.detach())


def _check_samples(x, starts, **params):
    """Refuses parameters whose samples are not x's: for (B, L, d) one set, B, or one for each of the B * L rows."""
    if starts is not None or x.dim() < 3:
        return
    for name, p in params.items():
        if p is not None and p.dim() == 2 and p.shape[0] != x.shape[0]:
            n, runs = 1, {1}
            for s in x.shape[:-1]:
                n *= s
                runs.add(n)
            if p.shape[0] not in runs:
                raise ValueError(f"{name} {tuple(p.shape)} does not go with the leading dimensions of x {tuple(x.shape)}")


def _want(*flags):
    return tuple(n for n, f in flags if f)


class _NormModulate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, scale, shift, starts, eps, dtype):
        x2, w, sc, sh = _flat(x), _par(weight), _par(scale), _par(shift)
        h = ops.norm_modulate(x2, w, sc, sh, starts, eps, dtype)
        ctx.save_for_backward(x2, w, sc, sh, starts)
        ctx.eps, ctx.shape = eps, x.shape
        return h.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x2, w, sc, sh, starts = ctx.saved_tensors
        n = ctx.needs_input_grad
        want = _want(("weight", n[1]), ("scale", n[2]), ("shift", n[3]))
        dx, dw, dsc, dsh = ops.norm_modulate_bwd(_dense(dh.reshape(x2.shape)), x2, w, sc, sh, starts, ctx.eps, want=want)
        return dx.view(ctx.shape) if n[0] else None, dw, dsc, dsh, None, None, None


class _NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, weight, norm, starts, eps, alpha):
        y2, g, w = _dense(y.reshape(-1, y.shape[-1])), _par(gate), _par(weight)
        out = ops.norm_residual(y2, _flat(x), g, w, norm, starts, eps, alpha)
        ctx.save_for_backward(y2, g, w, starts)
        ctx.norm, ctx.eps, ctx.alpha, ctx.shape = norm, eps, alpha, y.shape
        return out.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        y2, g, w, starts = ctx.saved_tensors
        n = ctx.needs_input_grad
        dy = dg = dw = None
        if n[1] or n[2] or n[3]:
            dy, dg, dw = ops.norm_residual_bwd(_dense(dout.reshape(y2.shape)), y2, g, w, ctx.norm, starts, ctx.eps,
                                               want=_want(("gate", n[2]), ("weight", n[3])))
            dy = dy.view(ctx.shape) if n[1] else None
        dx = (dout if ctx.alpha == 1.0 else ctx.alpha * dout) if n[0] else None
        return dx, dy, dg, dw, None, None, None, None


def norm_modulate(x, weight=None, scale=None, shift=None, starts=None, eps=1e-6, dtype=None):
    """h = n * weight * (1 + scale_b) + shift_b with n = x / sqrt(mean(x^2) + eps), of x's shape: ops.norm_modulate with
    gradients to x, weight, scale and shift."""
    _check_samples(x, starts, scale=scale, shift=shift)
    return _NormModulate.apply(x, weight, scale, shift, starts, eps, dtype)


def norm_residual(x, y, gate=None, weight=None, norm=True, starts=None, eps=1e-6, alpha=1.0):
    """alpha * x + gate_b * weight * n with n = y / sqrt(mean(y^2) + eps) (y itself without norm), of x's shape and type:
    ops.norm_residual for one slot with gradients to x, y, gate and weight.  (The stream x comes first here, the block's output
    y in ops.norm_residual.)"""
    if x.shape != y.shape:
        raise ValueError(f"x {tuple(x.shape)} and y {tuple(y.shape)} must have one shape")
    _check_samples(x, starts, gate=gate)
    return _NormResidual.apply(x, y, gate, weight, norm, starts, eps, alpha)


class _MoEResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wr, wgu, wd, pre_w, scale, shift, post_w, res_gate, cfg):
        (bias, k, renorm, gate, select_bias, norm, starts, eps, alpha, checkpoint) = cfg
        need = any(ctx.needs_input_grad[:9])
        pw, sc, sh, qw, rg = _par(pre_w), _par(scale), _par(shift), _par(post_w), _par(res_gate)
        h = ops.norm_modulate(x, pw, sc, sh, starts, eps, torch.bfloat16)
        y, ids, tw, state = _experts_forward(h, wr, wgu, wd, bias, k, renorm, gate, select_bias, need, checkpoint)
        out = ops.norm_residual(y, x, rg, qw, norm, starts, eps, alpha, k)
        if need:
            ctx.save_for_backward(x, y, pw, sc, sh, qw, rg, starts, *state.saved)
            state.saved = None
        ctx.state, ctx.cfg = state, (norm, eps, alpha, k)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return out, ids, tw

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _dids, dtw_out):
        if dout is None and dtw_out is None:
            return (None,) * 10
        norm, eps, alpha, k = ctx.cfg
        x, y, pw, sc, sh, qw, rg, starts, *saved = ctx.saved_tensors
        state = replace(ctx.state, saved=tuple(saved))
        n = ctx.needs_input_grad
        if dout is None:  # a loss on the routing weights alone
            dout = torch.zeros_like(x, memory_format=torch.contiguous_format)
        dout = _dense(dout)
        dy, drg, dqw = ops.norm_residual_bwd(dout, y, rg, qw, norm, starts, eps, k,
                                             want=_want(("gate", n[8]), ("weight", n[7])))
        below = n[0] or n[4] or n[5] or n[6]
        dh, dwr, dwgu, dwd = _experts_backward(state, dy, dtw_out, below, n[1], n[2], n[3])
        dx = dpw = dsc = dsh = None
        if below:
            dx, dpw, dsc, dsh = ops.norm_modulate_bwd(dh, x, pw, sc, sh, starts, eps, dres=dout, dres_scale=alpha,
                                                      want=_want(("weight", n[4]), ("scale", n[5]), ("shift", n[6])))
        return dx if n[0] else None, dwr, dwgu, dwd, dpw, dsc, dsh, dqw, drg, None


def moe_residual(x, router_weight, w_gu, w_d, top_k, pre_weight=None, scale=None, shift=None, post_weight=None, gate=None,
                 post_norm=True, starts=None, eps=1e-6, alpha=1.0, logit_bias=None, renorm=True, router=None,
                 select_bias=None, checkpoint=None, few_tokens=0):
    """out (T, d) = alpha * x + gate_b * post_weight * N(moe(N(x) * pre_weight * (1 + scale_b) + shift_b)) of x (T, d), bf16 or
    fp32 (the routed layer runs in bf16), N the RMS norm (post_norm=False: the layer's output itself) -> (out of x's type,
    topk_ids, topk_weight).  The routed layer and its options are moe_swiglu's (`router` its Gate; with few_tokens, the layer's
    output is rounded to bf16 ahead of the norm behind it); the other arguments are norm_modulate's and norm_residual's."""
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"x must be a (T, d) matrix in bf16 or fp32 (got {tuple(x.shape)} {x.dtype})")
    _check_checkpoint(checkpoint)
    few = _few(x.shape[0], top_k, few_tokens)
    if not _recorded(x, router_weight, w_gu, w_d, pre_weight, scale, shift, post_weight, gate):
        x2 = _flat(x)
        h = ops.norm_modulate(x2, _par(pre_weight), _par(scale), _par(shift), starts, eps, torch.bfloat16)
        layer = (h, router_weight, w_gu, w_d, logit_bias, top_k, renorm, router, select_bias)
        slots, inv = top_k, None
        if few:
            (y, ids, tw), slots = _few_infer(*layer), 1
        else:
            y, ids, tw, inv = _experts_infer(*layer)
        out = ops.norm_residual(y, x2, _par(gate), _par(post_weight), post_norm, starts, eps, alpha, slots, inv)
        return out, ids, tw
    cfg = (logit_bias, top_k, renorm, router, select_bias, post_norm, starts, eps, alpha, checkpoint)
    return _MoEResidual.apply(_flat(x), router_weight, w_gu, w_d, pre_weight, scale, shift, post_weight, gate, cfg)


class MoEResidual(nn.Module):
    """x -> alpha * x + gate * N(mlp(N(x) * (1 + scale) + shift)) with mlp = MoESwiGLU(dim, hidden, experts, top_k, ...): the
    second half of a denoiser block, its modulation (scale, shift, gate: (B, d) each) from outside.  norm_weight and, with
    post_norm, post_weight are learned (ones at first; affine=False: none).  x (B, L, d), or packed rows (T, d) with starts, in
    bf16 or fp32; the output has its shape and type.  The routing of the last call is kept in mlp.last_topk_ids /
    mlp.last_topk_weight, padding rows included: all of them have h = 0 and so the same experts.  mlp holds the parameters and is
    not called: hooks on it do not run, and what gathers sharded weights wraps this module, not mlp."""

    def __init__(self, dim: int, hidden: int, experts: int, top_k: int = 2, post_norm: bool = False, affine: bool = True,
                 eps: float = 1e-6, alpha: float = 1.0, device=None, norm_dtype=torch.float32, **mlp):
        super().__init__()
        self.mlp = MoESwiGLU(dim, hidden, experts, top_k, device=device, **mlp)
        self.post_norm, self.eps, self.alpha = post_norm, eps, alpha
        f = dict(device=device, dtype=norm_dtype)
        self.norm_weight = nn.Parameter(torch.ones(dim, **f)) if affine else None
        self.post_weight = nn.Parameter(torch.ones(dim, **f)) if affine and post_norm else None

    def forward(self, x, scale=None, shift=None, gate=None, starts=None):
        _check_samples(x, starts, scale=scale, shift=shift, gate=gate)
        m = self.mlp
        out, ids, tw = moe_residual(x.reshape(-1, x.shape[-1]), m.router_weight, m.w_gu, m.w_d, m.top_k, self.norm_weight,
                                    scale, shift, self.post_weight, gate, self.post_norm, starts, self.eps, self.alpha,
                                    m.logit_bias, m.renorm, m.gate, m.select_bias, m.checkpoint, m.few_tokens)
        m.last_topk_ids, m.last_topk_weight = ids, tw
        return out.view(x.shape)
