"""Trainable MoE-SwiGLU layer: a drop-in for the reference's dense FFN `DenoiserBlock.mlp = SwiGLU(dim, hidden)`
(aurora/model.py:102-110, called as self.mlp(h) on (B, T, dim) at :210), with a softmax top-k router and a full
backward pass -- neither exists in the reference (its MoE path is inference-only, aurora/hf_compat.py:62).

Forward (all hmoe HIP kernels, one stream, no host sync):
  route_topk -> dispatch (stable counting sort, the routed rows of x as row-group tiles for the GEMM's copies; with
  a backward to follow, also the row-major permuted copy) -> gate/up GEMM with fused SwiGLU ->
  down GEMM x routing weight, scattered to (token, slot) order -> combine over the k slots.
Backward:
  combine_bwd (weighted dY for the down wgrad) -> down wgrad -> down dgrad (dY rows gathered, routing weight
  applied in fp32) with fused SwiGLU backward and the routing-weight gradients -> gate/up dgrad (fp32 rows) ->
  gate/up wgrad -> router backward (softmax + renormalisation Jacobian, dWr) -> un-permute (sum over
  the k slots) + router input gradient.

The kernels compute in bf16 with fp32 accumulation.  fp32 weights (master weights) are rounded to bf16 for the
products, as torch.autocast does for the reference's nn.Linear layers, and receive fp32 gradients; fp16 weights
are rounded to bf16 the same way and receive their fp32 gradients rounded once to fp16.
"""
from __future__ import annotations

from dataclasses import dataclass, replace

import torch
import torch.autograd.forward_ad as fwd
import torch.nn as nn

from . import ops

_WDTYPES = (torch.bfloat16, torch.float32, torch.float16)


def _grad_dtype(param_dtype):
    """dtype a weight gradient is computed in: the parameter's own for bf16 / fp32, fp32 for fp16 parameters (the
    kernels write bf16 or fp32; the fp32 sum is then rounded once to fp16)."""
    return torch.float32 if param_dtype == torch.float16 else param_dtype


def _to_param(g, param_dtype):
    return g if g is None or g.dtype == param_dtype else g.to(param_dtype)


def _check_layer_args(x, wr, wgu, wd, bias, k):
    """Every shape the kernels rely on, cross-checked before the first launch: one expert count E (router rows,
    expert stacks, bias) and one model width d.  A router with more rows than there are expert stacks would route
    tokens to experts that do not exist."""
    if x.dim() != 2 or x.dtype != torch.bfloat16:
        raise TypeError(f"x must be a (T, d) bf16 matrix (got {tuple(x.shape)} {x.dtype})")
    if wr.dim() != 2 or wgu.dim() != 3 or wd.dim() != 3:
        raise ValueError("router_weight (E, d), w_gu (E, d, 2h) and w_d (E, h, d) expected")
    T, d = x.shape
    E, h = wgu.shape[0], wd.shape[1]
    for t, name, shape in ((wr, "router_weight", (E, d)), (wgu, "w_gu", (E, d, 2 * h)), (wd, "w_d", (E, h, d))):
        if tuple(t.shape) != shape:
            raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {shape} (E={E}, d={d}, h={h})")
        if t.dtype not in _WDTYPES:
            raise TypeError(f"{name}: dtype {t.dtype}; the layer takes bf16, fp32 or fp16 weights")
    if bias is not None and tuple(bias.shape) != (E,):
        raise ValueError(f"logit_bias: shape {tuple(bias.shape)}, expected ({E},)")
    if not 1 <= k <= E:
        raise ValueError(f"top_k = {k} must lie in [1, {E}]")


def _bf16(t):
    return t if t.dtype == torch.bfloat16 else t.to(torch.bfloat16)


def _recorded(*tensors):
    """Whether a call has to go through its autograd node: it has a gradient to record, or an input with a forward-mode
    tangent, which the nodes refuse (the one-call forms would drop it)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return fwd._current_level >= 0 and any(t is not None and fwd.unpack_dual(t).tangent is not None for t in tensors)


@dataclass(frozen=True)
class Gate:
    """How a layer's gate scores and selects experts (ops.route_scores): softmax over all experts or a sigmoid each, the
    experts in n_group groups of which the topk_group with the largest sums of their group_top best values are kept, and the
    factor on the weights.  The default is the plain softmax top-k, which the layer's own router serves in one kernel."""

    score: str = "softmax"
    n_group: int = 1
    topk_group: int = 1
    group_top: int = 2
    scaling: float = 1.0


def _route(x, wr, bias, k, renorm, gate, select_bias):
    """(logits, topk_ids, topk_weight) of x's rows."""
    if gate is None and select_bias is None:
        return ops.route_topk(x, wr, k, bias=bias, renorm=renorm)
    g = gate or Gate()
    logits, _, _ = ops.route_topk(x, wr, 1, bias=bias)
    if select_bias is not None:  # (a module cast to another type casts its buffers too)
        select_bias = select_bias.detach().to(torch.float32).contiguous()
    ids, tw = ops.route_scores(logits, k, g.score, select_bias, g.n_group, g.topk_group, g.group_top, renorm, g.scaling)
    return logits, ids, tw


@dataclass
class _Experts:
    """What the backward of a routed layer needs of its forward, besides the tensors in `saved`."""

    saved: tuple
    k: int
    renorm: bool
    gate: Gate | None
    select: bool  # the routing took a selection bias
    w_dtypes: tuple
    packed: bool = False  # [g | u] is kept in 8 bits, and neither the activation nor the permuted rows


def _check_checkpoint(checkpoint):
    if checkpoint not in (None, "fp8"):
        raise ValueError(f"checkpoint = {checkpoint!r}: None or 'fp8'")
    return checkpoint is not None


def _few(T, top_k, few_tokens):
    """Whether a call of T tokens without a gradient takes the two kernels for few of them."""
    if not 0 <= few_tokens <= ops.FEW_TOKENS:
        raise ValueError(f"few_tokens = {few_tokens}: 0 to {ops.FEW_TOKENS}")
    return 0 < T <= few_tokens and top_k <= 16


def _experts_forward(x, wr, wgu, wd, bias, k, renorm, gate, select_bias, need_grad, checkpoint=None):
    """Routing, dispatch and both projections of x (T, d) bf16 -> (y (T*k, d) in (token, slot) order, ids, weights, state)."""
    _check_layer_args(x, wr, wgu, wd, bias, k)
    if select_bias is not None and tuple(select_bias.shape) != (wgu.shape[0],):
        raise ValueError(f"select_bias: shape {tuple(select_bias.shape)}, expected ({wgu.shape[0]},)")
    M = x.shape[0] * k
    w_dtypes = (wr.dtype, wgu.dtype, wd.dtype)
    wr, wgu, wd = _bf16(wr), _bf16(wgu), _bf16(wd)
    logits, ids, tw = _route(x, wr, bias, k, renorm, gate, select_bias)
    packed = _check_checkpoint(checkpoint) and need_grad
    if packed:
        # [g | u] by the plain product, then act and the 8-bit copy in one pass over it: the same bytes as the fused epilogue
        # with a copy of [g | u], and nothing 16 bits wide stays behind
        disp = ops.dispatch(ids, wgu.shape[0], topk_w=tw, want_xs=False, dtype=x.dtype)
        act, kept = ops.swiglu_pack(ops.grouped_mm(x, wgu, disp.counts, M, a_idx=disp.a_idx))
        y, _ = ops.down_scatter(act, wd, disp.counts, M, disp.w_sorted, disp.order)
        saved = (x, wr, wgu, wd, logits, ids, disp.counts, disp.order, disp.a_idx, disp.inv_pos, disp.w_sorted, kept.q, kept.s)
        if gate is not None or select_bias is not None:
            saved += (tw,)
        return y, ids, tw, _Experts(saved, k, renorm, gate, select_bias is not None, w_dtypes, True)
    # The dispatch writes the routed rows as row-group tiles for the gate/up GEMM; with a backward to follow,
    # also the row-major permuted copy xs (the gate/up weight gradient reads it).
    disp, act, gu = ops.routed_gate_up(x, ids, wgu.shape[0], wgu, topk_w=tw, keep_gu=need_grad, want_xs=need_grad,
                                       want_inv=need_grad)
    y, _ = ops.down_scatter(act, wd, disp.counts, M, disp.w_sorted, disp.order)
    state = None
    if need_grad:
        saved = (x, wr, wgu, wd, logits, ids, disp.counts, disp.order, disp.a_idx, disp.inv_pos, disp.w_sorted, disp.xs, gu, act)
        if gate is not None or select_bias is not None:  # (else not kept: a program may change the weights in place)
            saved += (tw,)
        state = _Experts(saved, k, renorm, gate, select_bias is not None, w_dtypes)
    return y, ids, tw, state


def _experts_backward(state, dout, dtw_out, need_x, need_wr, need_wgu, need_wd):
    """(dx, dwr, dwgu, dwd), None where not needed, from dout (T, d) bf16, the gradient of every slot of y, and dtw_out
    (T, k), that of the returned weights, or None."""
    x, wr, wgu, wd, logits, ids, counts, order, a_idx, inv_pos, w_sorted, xs, gu, *rest = state.saved
    act, tw = (None, rest) if state.packed else (rest[0], rest[1:])  # (packed: xs and gu are the checkpoint's q and s)
    k = state.k
    T = x.shape[0]
    E = wgu.shape[0]
    M = T * k
    wr_dt, wgu_dt, wd_dt = state.w_dtypes
    disp = ops.Dispatch(counts, None, None, order, a_idx, inv_pos, w_sorted, xs)
    # One stream: every GEMM is a persistent launch sized to own all CUs, so two of them side by side only
    # queue each other's workgroups behind long-running tiles.
    dys = dwd = dwgu = dgu = dtw = None
    if state.packed:
        kept = ops.PackedGU(xs, gu, torch.bfloat16)
        dgu, act, dtw = ops.swiglu_pack_bwd(ops.down_dgrad(dout, wd, counts, M, a_idx=a_idx), kept, w_sorted, order, want_act=need_wd)
        dtw = dtw.view(T, k)
        xs = ops.dispatch(ids, E, x=x, want_inv=False).xs if need_wgu else None
    if need_wd:
        dys, _ = ops.combine_bwd(dout, None, disp, k)
        dwd = _to_param(ops.grouped_wgrad(act, dys, counts, E, dtype=_grad_dtype(wd_dt)), wd_dt)
    if not state.packed:
        # dgu, and the routing-weight gradient <dout[t], act[r] @ wd[e]> from the same fp32 product
        dgu, dtw = ops.down_dgrad_swiglu_dw(dout, wd, counts, M, gu, order, k, a_idx=a_idx, w_sorted=w_sorted)
    if dtw_out is not None:  # the returned routing weights are outputs too: their gradient joins the combine's
        dtw = dtw + dtw_out.to(torch.float32)
    if need_wgu:
        dwgu = _to_param(ops.grouped_wgrad(xs, dgu, counts, E, dtype=_grad_dtype(wgu_dt)), wgu_dt)
    # (for a few thousand rows its reduction is split, and the un-permute adds the parts)
    dxs = ops.gate_up_dgrad(dgu, wgu, counts, M, parts=ops.dgrad_parts(M, wgu))
    if state.gate is None and not state.select:
        dl, dwr = ops.router_bwd(logits, ids, dtw, x, renorm=state.renorm, dwr_dtype=_grad_dtype(wr_dt), want_dwr=need_wr)
    else:
        g = state.gate or Gate()
        dl = ops.route_scores_bwd(dtw, tw[0], logits, ids, g.score, state.renorm, g.scaling)
        dwr = ops.router_wgrad(dl, x, dtype=_grad_dtype(wr_dt)) if need_wr else None
    dwr = _to_param(dwr, wr_dt)
    dx = ops.unpermute_bwd(dxs, inv_pos, T, k, dlogits=dl, wr=wr) if need_x else None
    return dx, dwr, dwgu, dwd


class _MoEFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wr, wgu, wd, bias, k, renorm, gate=None, select_bias=None, checkpoint=None):
        need_grad = any(ctx.needs_input_grad[:4])
        y, ids, tw, state = _experts_forward(x, wr, wgu, wd, bias, k, renorm, gate, select_bias, need_grad, checkpoint)
        out = ops.combine(y, x.shape[0], k)
        if need_grad:
            ctx.save_for_backward(*state.saved)
            state.saved = None
        ctx.state = state
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)  # absent output gradients stay None (no zero-filled tensors)
        return out, ids, tw

    @staticmethod
    def backward(ctx, dout, _dids, dtw_out):
        none = (None,) * 6
        if dout is None and dtw_out is None:
            return (None,) * 4 + none
        state = replace(ctx.state, saved=ctx.saved_tensors)
        x = state.saved[0]
        if dout is None:  # a loss on the routing weights alone: the expert path carries no gradient
            dout = torch.zeros(x.shape, device=x.device, dtype=torch.bfloat16)
        dout = dout.contiguous().to(torch.bfloat16)
        return _experts_backward(state, dout, dtw_out, *ctx.needs_input_grad[:4]) + none


def moe_swiglu(x, router_weight, w_gu, w_d, top_k, logit_bias=None, renorm=True, gate=None, select_bias=None, checkpoint=None,
               few_tokens=0):
    """Functional form: x (T, d) bf16 -> (out (T, d) bf16, topk_ids (T, k) int32, topk_weight (T, k) fp32).

    router_weight (E, d), w_gu (E, d, 2h) = [gate | up], w_d (E, h, d): bf16, or fp32 / fp16 (rounded to bf16 for
    the products, gradients in the weights' dtype).  logit_bias (E,) fp32 is added to the router logits (no gradient).  Gradients reach
    x and the three weights from `out` and from `topk_weight` (softmax + renormalisation Jacobian).  gate: a Gate for sigmoid
    scores, groups or a factor on the weights; select_bias (E,) fp32 joins the scores for the selection only (a bias for
    balance; no gradient).  checkpoint="fp8" keeps [g | u] for the backward in 8 bits (ops.swiglu_pack), and neither the
    activation nor the permuted rows: about a third of the memory; the forward is the same but for act's single rounding, the
    gradients are those at the kept g and u.  few_tokens: without a gradient, calls of at most that many tokens (up to 16) run as
    two kernels (ops.few_forward, ops.few_experts), rounded once, so that their last bits differ from a larger call's.  Without a
    gradient to record (grad mode off, or no input requiring one) the forward runs as one C call
    (ops.moe_forward; with a gate or a selection bias, the routing and ops.moe_experts): the same kernels and outputs, a
    fraction of the host time."""
    _check_checkpoint(checkpoint)
    few = _few(x.shape[0], top_k, few_tokens)
    if not _recorded(x, router_weight, w_gu, w_d):
        if few:
            return _few_infer(x, router_weight, w_gu, w_d, logit_bias, top_k, renorm, gate, select_bias)
        if gate is None and select_bias is None:
            _check_layer_args(x, router_weight, w_gu, w_d, logit_bias, top_k)
            out, ids, tw, _ = ops.moe_forward(x, _bf16(router_weight), _bf16(w_gu), _bf16(w_d), top_k, bias=logit_bias,
                                              renorm=renorm)
            return out, ids, tw
        y, ids, tw, inv = _experts_infer(x, router_weight, w_gu, w_d, logit_bias, top_k, renorm, gate, select_bias)
        return ops.combine(y, x.shape[0], top_k, inv_pos=inv), ids, tw
    return _MoEFunction.apply(x, router_weight, w_gu, w_d, logit_bias, top_k, renorm, gate, select_bias, checkpoint)


def _experts_infer(x, wr, wgu, wd, bias, k, renorm, gate, select_bias):
    """_experts_forward without anything kept for a backward, the experts in one C call -> (y, ids, weights, inv_pos)."""
    _check_layer_args(x, wr, wgu, wd, bias, k)
    if select_bias is not None and tuple(select_bias.shape) != (wgu.shape[0],):
        raise ValueError(f"select_bias: shape {tuple(select_bias.shape)}, expected ({wgu.shape[0]},)")
    _, ids, tw = _route(x, _bf16(wr), bias, k, renorm, gate, select_bias)
    y, inv, _ = ops.moe_experts(x, ids, tw, _bf16(wgu), _bf16(wd))
    return y, ids, tw, inv


def _few_infer(x, wr, wgu, wd, bias, k, renorm, gate, select_bias):
    """The layer on a few tokens in two kernels -> (out, ids, weights)."""
    _check_layer_args(x, wr, wgu, wd, bias, k)
    if select_bias is not None and tuple(select_bias.shape) != (wgu.shape[0],):
        raise ValueError(f"select_bias: shape {tuple(select_bias.shape)}, expected ({wgu.shape[0]},)")
    wr, wgu, wd = _bf16(wr), _bf16(wgu), _bf16(wd)
    if gate is None and select_bias is None:
        return ops.few_forward(x, wr, wgu, wd, k, bias=bias, renorm=renorm)
    _, ids, tw = _route(x, wr, bias, k, renorm, gate, select_bias)
    return ops.few_experts(x, ids, tw, wgu, wd), ids, tw


class _ExpertStackProj:
    """What the reference's initialisation code reads of the dense SwiGLU's nn.Linear projections
    (aurora/model.py:308-312 and 393-396: `lin.weight`, `lin.in_features`; train_pp.py:1420-1421 zeroes
    `mlp.out_proj.weight`): here `weight` is the stacked expert parameter itself, so nn.init.normal_(..., std=
    in_features ** -0.5) gives every expert the fan-in initialisation and nn.init.zeros_ zeroes every expert."""

    __slots__ = ("weight", "in_features", "out_features")

    def __init__(self, weight, in_features, out_features):
        self.weight, self.in_features, self.out_features = weight, in_features, out_features


def _result_dtype(h: torch.Tensor) -> torch.dtype:
    """The dtype the reference's nn.Linear-based SwiGLU returns for input h: the autocast dtype inside an autocast
    region of h's device type, else h's own dtype."""
    dev = h.device.type
    if torch.is_autocast_enabled(dev):
        return torch.get_autocast_dtype(dev)
    return h.dtype


class MoESwiGLU(nn.Module):
    """MoE replacement for aurora/model.py:102-110 `SwiGLU(dim, hidden)`: same call shape ((..., dim) -> (..., dim)).

    Parameters: router_weight (E, dim); w_gu (E, dim, 2*hidden) = [gate | up] per expert (the stacked layout of
    aurora/hf_compat.py:154, gate first as in aurora/model.py:109); w_d (E, hidden, dim).  Buffer logit_bias (E,)
    fp32 is added to the router logits (zero by default; -inf disables an expert).

    `in_proj` / `out_proj` expose w_gu / w_d with the nn.Linear attributes the reference's init code uses, so
    Denoiser.init_weights / init_block and the zeroed output projection of train_pp --init run unchanged.  The
    default initialisation is theirs: N(0, in_features ** -0.5) per projection (dim for w_gu and the router, hidden
    for w_d); `init_std` overrides it with one std for all three.

    `gate` (a Gate) chooses sigmoid scores, groups or a factor on the weights; `balance` adds the buffer select_bias (E,)
    fp32, which joins the scores for the selection only: a training script that balances its experts without a loss raises
    it for experts that got too few tokens and lowers it for the others.

    `few_tokens` (up to 16): calls of at most that many tokens without a gradient run as two kernels (moe_swiglu).
    `checkpoint="fp8"` keeps [g | u] for the backward in 8 bits and nothing else of the experts' activations (moe_swiglu).

    The products run in bf16 (any other input dtype is rounded to bf16 first); the output has the dtype the
    reference's SwiGLU would return: the autocast dtype inside autocast, else the input's dtype.  The routing of the
    last call is kept in `last_topk_ids` / `last_topk_weight` (the weights carry gradient)."""

    def __init__(self, dim: int, hidden: int, experts: int, top_k: int = 2, renorm: bool = True,
                 init_std: float | None = None, device=None, dtype=torch.bfloat16, gate: Gate | None = None,
                 balance: bool = False, checkpoint: str | None = None, few_tokens: int = 0):
        super().__init__()
        _check_checkpoint(checkpoint)
        self.checkpoint, self.few_tokens = checkpoint, few_tokens
        self.dim, self.hidden, self.experts, self.top_k, self.renorm = dim, hidden, experts, top_k, renorm
        self.gate = gate
        f = dict(device=device, dtype=dtype)
        self.router_weight = nn.Parameter(torch.empty(experts, dim, **f))
        self.w_gu = nn.Parameter(torch.empty(experts, dim, 2 * hidden, **f))
        self.w_d = nn.Parameter(torch.empty(experts, hidden, dim, **f))
        self.register_buffer("logit_bias", torch.zeros(experts, device=device, dtype=torch.float32))
        if balance:
            self.register_buffer("select_bias", torch.zeros(experts, device=device, dtype=torch.float32))
        else:
            self.select_bias = None
        self.init_std = init_std
        self.reset_parameters()
        self.last_topk_ids = None
        self.last_topk_weight = None

    def __setstate__(self, state):
        super().__setstate__(state)
        self.__dict__.setdefault("gate", None)  # (pickled before the layer had gates)
        self.__dict__.setdefault("checkpoint", None)
        self.__dict__.setdefault("few_tokens", 0)
        if "select_bias" not in self._buffers:
            self.__dict__.setdefault("select_bias", None)

    @property
    def in_proj(self) -> _ExpertStackProj:
        return _ExpertStackProj(self.w_gu, self.dim, 2 * self.hidden)

    @property
    def out_proj(self) -> _ExpertStackProj:
        return _ExpertStackProj(self.w_d, self.hidden, self.dim)

    @torch.no_grad()
    def reset_parameters(self):
        for p, fan_in in ((self.router_weight, self.dim), (self.w_gu, self.dim), (self.w_d, self.hidden)):
            nn.init.normal_(p, std=self.init_std if self.init_std is not None else fan_in ** -0.5)

    def forward(self, h: torch.Tensor) -> torch.Tensor:
        shape = h.shape
        out_dtype = _result_dtype(h)
        x = h.reshape(-1, shape[-1])
        if x.dtype != torch.bfloat16:
            x = x.to(torch.bfloat16)
        out, ids, tw = moe_swiglu(x, self.router_weight, self.w_gu, self.w_d, self.top_k, self.logit_bias,
                                  self.renorm, self.gate, self.select_bias, self.checkpoint, self.few_tokens)
        self.last_topk_ids, self.last_topk_weight = ids, tw
        out = out.view(shape)
        return out if out.dtype == out_dtype else out.to(out_dtype)


def moe_param_groups(module: nn.Module, lr: float, weight_decay: float, router_lr: float | None = None):
    """Optimizer groups for every MoESwiGLU inside `module`, for a training script whose grouping rule sends 2-D
    matrices under `.blocks.` to Muon and everything else to AdamW (train.py:305-338 of the reference).  Left to that
    rule, a MoESwiGLU standing in for a block's dense SwiGLU would have its router (E, dim), a 2-D matrix, updated by
    Muon and its 3-D expert stacks w_gu / w_d put in the AdamW "other" group (no weight decay, the Adam learning
    rate), while the dense in_proj / out_proj they replace were Muon's hidden matrices.

    Returns (groups, ids).  groups: AdamW parameter groups (`params`, `lr`, `base_lr`, `weight_decay`, `name`):
      - "moe_experts": every w_gu and w_d, at `lr` (the hidden-matrix learning rate) with `weight_decay`;
      - "moe_router": every router_weight, at `router_lr` (default `lr`) without weight decay, kept out of Muon (an
        orthogonalised update would mix the experts' logit directions).
    ids: the id() of each parameter placed, to remove from the list the script's own rule groups (its `named=`
    argument), so that no parameter is in two groups."""
    experts, routers = [], []
    for m in module.modules():
        if isinstance(m, MoESwiGLU):
            experts += [p for p in (m.w_gu, m.w_d) if p.requires_grad]
            if m.router_weight.requires_grad:
                routers.append(m.router_weight)
    rlr = lr if router_lr is None else router_lr
    groups = [dict(params=experts, lr=lr, base_lr=lr, weight_decay=weight_decay, name="moe_experts"),
              dict(params=routers, lr=rlr, base_lr=rlr, weight_decay=0.0, name="moe_router")]
    groups = [g for g in groups if g["params"]]
    return groups, {id(p) for g in groups for p in g["params"]}


def clip_grad_norm(grads, max_norm, out=None):
    """Clips a list of gradient tensors by their global norm: each becomes itself times min(1, max_norm / (norm + 1e-6)), in
    place, or in `out` (tensors of the same shapes and strides, of the gradients' types or fp32, such as an optimizer's fp32
    gradients; the gradients then stay as they are).  Tensors written by a call that overlap others of it are refused.  bf16, fp16 and fp32 tensors of
    any size and alignment may be mixed, None entries are skipped.  Returns the norm before clipping, a () fp32 tensor on the
    device; nothing waits for the GPU.
    A gradient spread over several processes: all-reduce ops.grad_sq_norm's sum before ops.grad_clip.  Autograd does not see
    the change in place: where gradients are themselves part of a graph (create_graph=True), clip after its last backward."""
    grads = list(grads)
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"{len(out)} outputs for {len(grads)} gradients")
    if not all([g is not None for g in grads]):
        if out is not None:
            out = [o for g, o in zip(grads, out) if g is not None]
        grads = [g for g in grads if g is not None]
    gl = ops.GradList(grads, out)
    return ops.grad_clip(gl, ops.grad_sq_norm(gl), max_norm)
