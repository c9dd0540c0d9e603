"""Plain 64-bit restatements (CPU, torch float64) of the operators around the routed block, for their tests: the norms,
routing from logits and gradient clipping.  Gradients come from differentiating these."""
import math

import torch

EPS24 = 2.0 ** -24


def half_step(dtype):
    """The largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of dtype's smallest step: the absolute error of a rounding among its subnormal values."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2


def sample_rows(T, B, starts):
    """(T,) sample of each row, -1 for padding."""
    if starts is None:
        return torch.arange(T) // max(T // B, 1)
    b = torch.full((T,), -1, dtype=torch.long)
    for i in range(B):
        b[starts[i]:starts[i + 1]] = i
    return b


def rms(v, eps):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def _per_row(p, b):
    p = p if p.dim() == 2 else p.unsqueeze(0).expand(int(b.max()) + 1 if b.numel() else 1, -1)
    return p[b.clamp(min=0)]


def norm_modulate(x, weight, scale, shift, b, eps):
    live = (b >= 0).unsqueeze(1)
    h = rms(torch.where(live, x, torch.zeros((), dtype=x.dtype)), eps)
    if weight is not None:
        h = h * weight
    if scale is not None:
        h = h * (1 + _per_row(scale, b))
    if shift is not None:
        h = h + _per_row(shift, b)
    return torch.where(live, h, torch.zeros((), dtype=x.dtype))


def slot_sum(y, T, k, inv_pos, add):
    s = y.reshape(T, k, -1)
    if inv_pos is not None:
        s = torch.where((inv_pos.reshape(T, k, 1) < 0), torch.zeros((), dtype=s.dtype), s)
    s = s.sum(1)
    return s if add is None else s + add


def norm_residual(s, x, gate, weight, norm, b, eps, alpha):
    live = (b >= 0).unsqueeze(1)
    z = torch.where(live, s, torch.zeros((), dtype=s.dtype))
    if norm:
        z = rms(z, eps)
    if weight is not None:
        z = z * weight
    if gate is not None:
        z = z * _per_row(gate, b)
    return alpha * x + torch.where(live, z, torch.zeros((), dtype=s.dtype))


def route(logits, k, score, bias, n_group, topk_group, group_top, renorm, scaling, live):
    """ids (T, k), weights (T, k): one token after the other, in Python floats' precision."""
    T, E = logits.shape
    lg = logits.double()
    if score == "softmax":
        m = lg.amax(1, keepdim=True) if E else lg
        ex = torch.where(lg == -math.inf, torch.zeros_like(lg), torch.exp(lg - m))
        tot = ex.sum(1, keepdim=True)
        s = torch.where(tot == 0, torch.zeros_like(ex), ex / tot)
    else:
        s = 1 / (1 + torch.exp(-lg))
    key = s if bias is not None or topk_group < n_group else lg
    key = key + (0 if bias is None else bias.double())
    dead = ~(lg > -math.inf)
    if bias is not None:
        dead = dead | ~(bias.double() > -math.inf)
    key = torch.where(dead | torch.isnan(key), torch.full_like(key, -math.inf), key)
    ids = torch.empty(T, k, dtype=torch.int32)
    w = torch.zeros(T, k, dtype=torch.float64)
    eg = E // n_group
    for t in range(T):
        row = key[t].tolist()
        if topk_group < n_group:
            val = [sum(sorted(row[g * eg:(g + 1) * eg], reverse=True)[:group_top]) for g in range(n_group)]
            kept = sorted(range(n_group), key=lambda g: (-val[g], g))[:topk_group]
            row = [v if e // eg in kept else -math.inf for e, v in enumerate(row)]
        best = sorted(range(E), key=lambda e: (-row[e], e))[:k]
        for j, e in enumerate(best):
            ids[t, j] = e
            w[t, j] = 0.0 if row[e] == -math.inf else s[t, e]
            if score == "softmax" and torch.isnan(s[t]).any():
                w[t, j] = math.nan
    if renorm:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    w = w * scaling
    if live is not None:
        ids[~live] = -1
        w[~live] = 0
    return ids, w


def route_weights(lg, ids, w, score, renorm, scaling):
    """The weights of given ids as a differentiable function of float64 logits (slots of weight 0 stay 0)."""
    s = torch.softmax(lg, 1) if score == "softmax" else torch.sigmoid(lg)
    on = (ids >= 0) & (w != 0)
    v = torch.where(on, s.gather(1, ids.long().clamp(min=0)), torch.zeros((), dtype=lg.dtype))
    if renorm:
        v = v / (v.sum(1, keepdim=True) + 1e-20)
    return v * scaling
