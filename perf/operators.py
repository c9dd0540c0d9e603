"""Operators around the routed block that their speed is measured on, with their plain forms.

Kinds:
  norm_in   the RMS norm before the block with its weight and per-sample scale and shift; with train, its backward too
  norm_out  the sum over the routed slots, the RMS norm after the block, the gate and the scaled residual; with train,
            the backward too
  route     experts chosen from given logits: softmax or sigmoid scores, selection bias, groups, top-k, renormalised
            weights; with train, the logits' gradient too
  clip      the global norm of a list of gradients, and the clipped gradients

Where `own` is false, `run` computes the plain form (elementary torch operations in 32 bits, selection keys and long
sums in 64); where it is true it calls the framework's operators.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SZ = {"bf16": 2, "fp16": 2, "fp32": 4, "none": 0}


def listed():
    return [
        # the norm before the text encoder's block on a handful of tokens: one launch, latency counts
        dict(name="norm_in_8", kind="norm_in", T=8, d=2048, B=0, ragged=False, stream="bf16", block="bf16",
             weight="bf16", mods="none", train=False),
        # packed images of several resolutions with padding behind them, an fp32 residual stream, widths off 512
        dict(name="norm_in_3001_ragged", kind="norm_in", T=3001, d=760, B=7, ragged=True, stream="fp32", block="bf16",
             weight="fp32", mods="fp32", train=True),
        # a training step on four 1024 px images
        dict(name="norm_in_16384", kind="norm_in", T=16384, d=1536, B=4, ragged=False, stream="bf16", block="bf16",
             weight="bf16", mods="bf16", train=True),
        # the text encoder's block on one short prompt: eight slots and the shared expert per token
        dict(name="norm_out_64", kind="norm_out", T=64, d=2048, B=0, ragged=False, stream="bf16", block="bf16",
             weight="bf16", gate="none", k=8, shared=True, dropped=False, alpha=1.0, train=False),
        # a packed batch in fp16 on an fp32 stream, some expert ids out of range
        dict(name="norm_out_5000_fp16", kind="norm_out", T=5000, d=1024, B=9, ragged=True, stream="fp32",
             block="fp16", weight="fp32", gate="fp32", k=4, shared=False, dropped=True, alpha=0.7, train=False),
        # a training step on four 1024 px images
        dict(name="norm_out_16384", kind="norm_out", T=16384, d=1536, B=4, ragged=False, stream="bf16", block="bf16",
             weight="bf16", gate="bf16", k=2, shared=False, dropped=False, alpha=1.0, train=True),
        # one short prompt through the text encoder's gate
        dict(name="route_64", kind="route", T=64, E=128, k=8, score="sigmoid", n_group=8, topk_group=2, bias=True,
             renorm=True, logits="fp32", padded=False, train=False),
        # a training step of the softmax gate on four 1024 px images
        dict(name="route_16384", kind="route", T=16384, E=16, k=2, score="softmax", n_group=1, topk_group=1,
             bias=True, renorm=True, logits="fp32", padded=False, train=True),
        # a training step of a wide grouped sigmoid gate on a padded batch
        dict(name="route_8192_groups", kind="route", T=8192, E=256, k=8, score="sigmoid", n_group=8, topk_group=4,
             bias=True, renorm=True, logits="fp32", padded=True, train=True),
        # the vectors and small matrices of a model: many views of a bucket, odd sizes, norm below the bound, in place
        dict(name="clip_small", kind="clip", n=300, E=0, d=1536, h=0, layers=0, dtype="bf16", out="inplace",
             clipped=False),
        # four small layers with fp32 master weights, clipped
        dict(name="clip_layers_fp32", kind="clip", n=24, E=8, d=760, h=1352, layers=4, dtype="fp32", out="same",
             clipped=True),
        # the gradients of one large layer, clipped into the optimiser's fp32 gradients: the largest
        dict(name="clip_layer_bf16", kind="clip", n=6, E=16, d=1536, h=4096, layers=1, dtype="bf16", out="fp32",
             clipped=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm_in", "norm_out", "route", "clip"))
    if kind in ("norm_in", "norm_out"):
        d = 8 * rng.randint(16, 512)
        T = min(_log_int(rng, 1, 16384), 16384 * 1536 // d)
        stream, block = rng.choice((("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "bf16"), ("fp32", "fp16"),
                                    ("fp32", "fp32")))
        B = rng.choice((0, 1, rng.randint(1, 40)))
        ragged = B > 0 and rng.random() < 0.5
        if B and not ragged:  # equal runs of rows
            B = min(B, T)
            T -= T % B
        p = rng.choice((stream, "fp32"))
        c = dict(kind=kind, T=T, d=d, B=B, ragged=ragged, stream=stream, block=block,
                 weight=rng.choice((p, p, "none")), train=rng.random() < 0.6)
        if kind == "norm_in":
            c["mods"] = p if B else "none"
        else:
            k = rng.choice((1, 2, 4, 6, 8, 3))
            c["T"] = T if k < 3 else max(1, B, T // k - (T // k) % max(B, 1) if not ragged else T // k)
            c.update(gate=p if B else "none", k=k, shared=rng.random() < 0.3, dropped=k > 1 and rng.random() < 0.4,
                     alpha=rng.choice((1.0, 1.0, 0.5)))
        return c
    if kind == "route":
        n_group, eg = rng.choice(((1, 0), (1, 0), (4, 0), (8, 0), (6, 0)))
        if n_group == 1:
            E = rng.randint(4, 300)
            topk_group = 1
            k = rng.randint(1, min(12, E))
        else:
            eg = rng.randint(2, 40)
            E = n_group * eg
            topk_group = rng.randint(1, n_group - 1)
            k = rng.randint(1, min(12, topk_group * eg))
        # (renormalised over one expert the weight is constant and the logits have no gradient)
        return dict(kind=kind, T=min(_log_int(rng, 1, 16384), 8192 * 256 // E), E=E, k=k,
                    score=rng.choice(("softmax", "sigmoid")), n_group=n_group, topk_group=topk_group,
                    bias=rng.random() < 0.6, renorm=k > 1 and rng.random() < 0.7, logits=rng.choice(("fp32", "fp32", "bf16")),
                    padded=rng.random() < 0.4, train=rng.random() < 0.6)
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    clipped = rng.random() < 0.6
    E, d, h = rng.randint(2, 16), 8 * rng.randint(32, 192), 8 * rng.randint(32, 400)
    layers = rng.randint(1, 4)
    while layers * E * d * h * 3 > 16 * 1536 * 4096 * 3 // 2:
        E, h = max(1, E // 2), max(64, h // 2)
    return dict(kind=kind, n=rng.randint(0, 200), E=E, d=d, h=h, layers=layers, dtype=dtype,
                out=rng.choice(("same", "fp32")) if clipped else "inplace", clipped=clipped)


# ---------------------------------------------------------------------------------------------------------------
# What a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------
def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)


def _starts(T, B, g):
    """(B + 1,) row offsets of B packed samples of unequal lengths (one of them empty where there are several), with
    padding rows behind the last."""
    end = T - min(T // 16, 40)
    cuts = torch.randint(0, end + 1, (B - 1,), generator=g, device=DEV).sort().values
    if B > 2:
        cuts[1] = cuts[0]
    z = torch.zeros(1, dtype=cuts.dtype, device=DEV)
    return torch.cat([z, cuts, z + end]).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = case
    s = dict(case=c)
    if c["kind"] in ("norm_in", "norm_out"):
        T, d, B = c["T"], c["d"], c["B"]
        st, bt = _DT[c["stream"]], _DT[c["block"]]
        # a residual stream: unit rows of unequal size, a few channels far above the rest
        x = torch.randn(T, d, generator=g, device=DEV) * (0.5 + torch.rand(T, 1, generator=g, device=DEV))
        x[:, :: max(d // 4, 1)] *= 8
        s["x"] = x.to(st)
        s["weight"] = None if c["weight"] == "none" else _randn(g, d, std=0.1, mean=1.0, dtype=_DT[c["weight"]])
        s["starts"] = _starts(T, B, g) if c["ragged"] else None
        if c["kind"] == "norm_in":
            mods = None if c["mods"] == "none" else _DT[c["mods"]]
            s["scale"] = None if mods is None else _randn(g, B, d, std=0.3, dtype=mods)
            s["shift"] = None if mods is None else _randn(g, B, d, std=0.5, dtype=mods)
            if c["train"]:
                s["dh"] = _randn(g, T, d, std=0.02, dtype=bt)
                s["dres"] = _randn(g, T, d, std=0.02, dtype=st)
        else:
            k = c["k"]
            s["y"] = _randn(g, T * k, d, std=0.3, dtype=bt)
            s["add"] = _randn(g, T, d, std=0.3, dtype=bt) if c["shared"] else None
            s["inv_pos"] = None
            if c["dropped"]:  # slots routed nowhere: their rows of y are never written
                off = torch.rand(T * k, generator=g, device=DEV) < 0.02
                s["inv_pos"] = torch.where(off, -1, torch.arange(T * k, device=DEV)).to(torch.int32)
                s["y"][off] = math.nan
            s["gate"] = None if c["gate"] == "none" else _randn(g, B, d, std=0.3, dtype=_DT[c["gate"]])
            if c["train"]:
                s["dout"] = _randn(g, T, d, std=0.02, dtype=st)
    elif c["kind"] == "route":
        T, E, k = c["T"], c["E"], c["k"]
        s["logits"] = _randn(g, T, E, std=1.5, dtype=_DT[c["logits"]])
        s["bias"] = _randn(g, E, std=0.05, dtype=torch.float32) if c["bias"] else None
        s["live"] = torch.rand(T, generator=g, device=DEV) < 0.9 if c["padded"] else None
        if c["train"]:
            s["dw"] = _randn(g, T, k, std=0.1, dtype=torch.float32)
    else:
        shapes = []
        for _ in range(c["layers"]):
            shapes += [(c["E"], c["d"]), (c["E"], c["d"], 2 * c["h"]), (c["E"], c["h"], c["d"])]
        dt = _DT[c["dtype"]]
        s["grads"] = [_randn(g, *sh, std=10.0 ** -(2 + i % 3), dtype=dt) for i, sh in enumerate(shapes)]
        sq = sum(math.prod(sh) * 10.0 ** (-2 * (2 + i % 3)) for i, sh in enumerate(shapes))
        # the small ones are views of one flat bucket, as data-parallel gradients are, packed without gaps
        small = [1 + (37 * i) % (2 * c["d"]) if i % 3 else c["d"] * (1 + i % 7) for i in range(c["n"])]
        s["bucket"] = _randn(g, sum(small), std=1e-3, dtype=dt)
        sq += sum(small) * 1e-6
        s["n_large"] = len(s["grads"])
        s["grads"] += list(s["bucket"].split(small)) if small else []
        s["max_norm"] = math.sqrt(sq) * 0.25 if c["clipped"] else math.sqrt(sq) * 4 + 1
        s["out"] = None
        if c["out"] != "inplace":
            ot = dt if c["out"] == "same" else torch.float32
            s["out"] = [torch.empty_like(t, dtype=ot) for t in s["grads"][:s["n_large"]]]
            s["out_bucket"] = torch.empty_like(s["bucket"], dtype=ot)
            s["out"] += list(s["out_bucket"].split(small)) if small else []
    return s


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)[s["case"]["kind"]](s)


def _own_norm_in(s):
    from trenowanie_generatora_obrazkow_amd import ops
    c = s["case"]
    h = ops.norm_modulate(s["x"], weight=s["weight"], scale=s["scale"], shift=s["shift"], starts=s["starts"], eps=EPS,
                          dtype=_DT[c["block"]])
    if not c["train"]:
        return {"h": h}
    dx, dw, dsc, dsh = ops.norm_modulate_bwd(s["dh"], s["x"], weight=s["weight"], scale=s["scale"], shift=s["shift"],
                                             starts=s["starts"], eps=EPS, dres=s["dres"])
    return _some(h=h, dx=dx, dweight=dw, dscale=dsc, dshift=dsh)


def _own_norm_out(s):
    from trenowanie_generatora_obrazkow_amd import ops
    c = s["case"]
    kw = dict(gate=s["gate"], weight=s["weight"], starts=s["starts"], eps=EPS, k=c["k"], inv_pos=s["inv_pos"],
              add=s["add"])
    out = ops.norm_residual(s["y"], s["x"], alpha=c["alpha"], **kw)
    if not c["train"]:
        return {"out": out}
    dy, dgate, dw = ops.norm_residual_bwd(s["dout"], s["y"], **kw)
    return _some(out=out, dy=dy, dgate=dgate, dweight=dw)


def _own_route(s):
    from trenowanie_generatora_obrazkow_amd import ops
    c = s["case"]
    ids, w = ops.route_scores(s["logits"], c["k"], score=c["score"], bias=s["bias"], n_group=c["n_group"],
                              topk_group=c["topk_group"], renorm=c["renorm"], scaling=2.5, live=s["live"])
    if not c["train"]:
        return {"ids": ids, "w": w}
    dl = ops.route_scores_bwd(s["dw"], w, s["logits"], ids, score=c["score"], renorm=c["renorm"], scaling=2.5)
    return {"ids": ids, "w": w, "dlogits": dl}


def _own_clip(s):
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    norm = clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])
    return _clip_outputs(s, norm)


def _clip_outputs(s, norm):
    out, bucket = (s["grads"], s["bucket"]) if s["out"] is None else (s["out"], s["out_bucket"])
    return {"norm": norm, "grads": out[:s["n_large"]], "bucket": bucket}


_run_own = {"norm_in": _own_norm_in, "norm_out": _own_norm_out, "route": _own_route, "clip": _own_clip}


def _some(**kw):
    return {k: v for k, v in kw.items() if v is not None}


def _samples(s):
    """The sample of every row (None: one for all) and which rows belong to one (None: all)."""
    c = s["case"]
    T, B = c["T"], c["B"]
    if B == 0:
        return None, None
    row = torch.arange(T, device=DEV)
    if s["starts"] is None:
        return row // (T // B), None
    b = torch.searchsorted(s["starts"].long(), row, right=True) - 1
    live = (b >= 0) & (b < B)
    return b.clamp(0, B - 1), live.unsqueeze(1)


def _f(t):
    return None if t is None else t.float()


def _rows(p, b):
    """Rows of a per-sample (B, d) parameter, one for each row of the batch."""
    return p.float()[b]


def _per_sample(v, b, live, s):
    """(B, d) sums of the rows v over each sample."""
    c = s["case"]
    if live is not None:
        v = torch.where(live, v, 0.0)
    if s["starts"] is None:
        return v.view(c["B"], -1, c["d"]).sum(1)
    return (torch.arange(c["B"], device=DEV).unsqueeze(1) == b).float() @ v


def _plain_norm_in(s):
    c = s["case"]
    b, live = _samples(s)
    x, w = s["x"].float(), _f(s["weight"])
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    n = x * r
    m = n if w is None else n * w
    sc = None if s["scale"] is None else 1 + _rows(s["scale"], b)
    h = m if sc is None else m * sc
    if s["shift"] is not None:
        h = h + _rows(s["shift"], b)
    if live is not None:
        h = torch.where(live, h, 0.0)
    h = h.to(_DT[c["block"]])
    if not c["train"]:
        return {"h": h}
    dh = s["dh"].float()
    if live is not None:
        dh = torch.where(live, dh, 0.0)
    dm = dh if sc is None else dh * sc
    dn = dm if w is None else dm * w
    dx = r * (dn - n * (dn * n).mean(1, keepdim=True)) + s["dres"].float()
    out = dict(h=h, dx=dx.to(s["x"].dtype), dweight=None, dscale=None, dshift=None)
    if w is not None:
        out["dweight"] = (dm * n).sum(0).to(s["weight"].dtype)
    if sc is not None:
        out["dscale"] = _per_sample(dh * m, b, live, s).to(s["scale"].dtype)
    if s["shift"] is not None:
        out["dshift"] = _per_sample(dh, b, live, s).to(s["shift"].dtype)
    return _some(**out)


def _plain_norm_out(s):
    c = s["case"]
    T, d = c["T"], c["d"]
    b, live = _samples(s)
    y = s["y"].float()
    if s["inv_pos"] is not None:
        y = torch.where(s["inv_pos"].unsqueeze(1) < 0, 0.0, y)
    y = y.view(T, c["k"], d).sum(1)
    if s["add"] is not None:
        y = y + s["add"].float()
    w, gate = _f(s["weight"]), None if s["gate"] is None else _rows(s["gate"], b)
    r = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + EPS)
    n = y * r
    m = n if w is None else n * w
    z = m if gate is None else m * gate
    if live is not None:
        z = torch.where(live, z, 0.0)
    res = {"out": (c["alpha"] * s["x"].float() + z).to(s["x"].dtype)}
    if not c["train"]:
        return res
    dz = s["dout"].float()
    if live is not None:
        dz = torch.where(live, dz, 0.0)
    dm = dz if gate is None else dz * gate
    dn = dm if w is None else dm * w
    res["dy"] = (r * (dn - n * (dn * n).mean(1, keepdim=True))).to(s["y"].dtype)
    if gate is not None:
        res["dgate"] = _per_sample(dz * m, b, live, s).to(s["gate"].dtype)
    if w is not None:
        res["dweight"] = (dm * n).sum(0).to(s["weight"].dtype)
    return res


def _plain_route(s):
    c = s["case"]
    T, E, k, G = c["T"], c["E"], c["k"], c["n_group"]
    lg = s["logits"].double()
    if c["score"] == "softmax":
        ex = torch.exp(lg - lg.amax(1, keepdim=True))
        sc = ex / ex.sum(1, keepdim=True)
    else:
        sc = 1 / (1 + torch.exp(-lg))
    key = sc if s["bias"] is None else sc + s["bias"].double()
    if c["topk_group"] < G:
        grp = key.view(T, G, E // G).sort(dim=2, descending=True).values[:, :, :2].sum(2)
        best = grp.sort(dim=1, descending=True, stable=True).indices[:, :c["topk_group"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=DEV).scatter_(1, best, True)
        key = torch.where(keep.repeat_interleave(E // G, 1), key, -math.inf)
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :k]
    sc = sc.float()
    sel = sc.gather(1, ids)
    den = sel.sum(1, keepdim=True) + 1e-20 if c["renorm"] else 1.0
    w = sel / den * 2.5
    if s["live"] is not None:
        off = ~s["live"].unsqueeze(1)
        w = torch.where(off, 0.0, w)
    res = {"ids": (ids if s["live"] is None else torch.where(off, -1, ids)).to(torch.int32), "w": w}
    if not c["train"]:
        return res
    dw = 2.5 * s["dw"]
    if s["live"] is not None:
        dw = torch.where(off, 0.0, dw)
    ds = (dw - (dw * sel).sum(1, keepdim=True) / den) / den if c["renorm"] else dw
    if c["score"] == "sigmoid":
        dl = torch.zeros(T, E, device=DEV).scatter_(1, ids, ds * sel * (1 - sel))
    else:
        dp = torch.zeros(T, E, device=DEV).scatter_(1, ids, ds)
        dl = sc * (dp - (sc * dp).sum(1, keepdim=True))
    res["dlogits"] = dl.to(s["logits"].dtype)
    return res


def _plain_clip(s):
    sq = sum((g.float() * g.float()).sum(dtype=torch.float64) for g in s["grads"])
    norm = torch.sqrt(sq)
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    out = s["grads"] if s["out"] is None else s["out"]
    for g, o in zip(s["grads"], out):
        o.copy_(g.float() * coef)
    return _clip_outputs(s, norm.float())


_run_plain = {"norm_in": _plain_norm_in, "norm_out": _plain_norm_out, "route": _plain_route, "clip": _plain_clip}


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] in ("norm_in", "norm_out"):
        T, d, B = c["T"], c["d"], c["B"]
        sx, sh, pw = _SZ[c["stream"]], _SZ[c["block"]], _SZ[c["weight"]]
        if c["kind"] == "norm_in":
            par = d * pw + 2 * B * d * _SZ[c["mods"]]
            b = T * d * (sx + sh) + par
            if c["train"]:
                b += T * d * (sh + 2 * sx) + par
            return {"bytes": b, "flops": T * d * (20 if c["train"] else 7)}
        par = d * pw + B * d * _SZ[c["gate"]]
        b = T * d * (c["k"] * sh + (sh if c["shared"] else 0) + 2 * sx) + par
        if c["train"]:
            b += T * d * (sx + sh) + par
        return {"bytes": b, "flops": T * d * (c["k"] + (18 if c["train"] else 8))}
    if c["kind"] == "route":
        T, E, k = c["T"], c["E"], c["k"]
        b = T * E * _SZ[c["logits"]] + T * k * 8
        if c["train"]:
            b += T * E * _SZ[c["logits"]] + T * k * 4
        return {"bytes": b, "flops": T * E * (12 + k) + (6 * T * E if c["train"] else 0)}
    n = c["layers"] * c["E"] * (c["d"] + 3 * c["d"] * c["h"])
    n += sum(1 + (37 * i) % (2 * c["d"]) if i % 3 else c["d"] * (1 + i % 7) for i in range(c["n"]))  # the bucket
    si = _SZ[c["dtype"]]
    so = 0 if c["out"] == "inplace" else si if c["out"] == "same" else 4  # (below the bound nothing is to be written)
    return {"bytes": n * (si + so), "flops": 2 * n + (n if so else 0)}


# ---------------------------------------------------------------------------------------------------------------
# The same results from the definitions in 64 bits: gradients by differentiation of the forward
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"norm_in": _exact_norm_in, "norm_out": _exact_norm_out, "route": _exact_route,
                "clip": _exact_clip}[case["kind"]](s)


def _leaf(t):
    return None if t is None else t.double().requires_grad_(True)


def _sample_rows(s):
    """[(sample, first row, end row)] of the batch."""
    c = s["case"]
    if c["B"] == 0:
        return [(None, 0, c["T"])]
    if s["starts"] is None:
        L = c["T"] // c["B"]
        return [(i, i * L, (i + 1) * L) for i in range(c["B"])]
    st = s["starts"].tolist()
    return [(i, st[i], st[i + 1]) for i in range(c["B"])]


def _rms64(v):
    return v * (v.square().sum(-1, keepdim=True) / v.shape[-1] + EPS).rsqrt()


def _grads64(loss, leaves):
    names = [k for k, v in leaves.items() if v is not None]
    got = torch.autograd.grad(loss, [leaves[k] for k in names], allow_unused=True)
    return {k: torch.zeros_like(leaves[k]) if v is None else v for k, v in zip(names, got)}


def _exact_norm_in(s):
    c = s["case"]
    lv = dict(x=_leaf(s["x"]), weight=_leaf(s["weight"]), scale=_leaf(s["scale"]), shift=_leaf(s["shift"]))
    parts, end = [], 0
    for i, a, e in _sample_rows(s):
        v = _rms64(lv["x"][a:e])
        if lv["weight"] is not None:
            v = lv["weight"] * v
        if lv["scale"] is not None:
            v = v + lv["scale"][i] * v
        if lv["shift"] is not None:
            v = v + lv["shift"][i]
        parts.append(v)
        end = e
    parts.append(torch.zeros(c["T"] - end, c["d"], dtype=torch.float64, device=DEV))
    h = torch.cat(parts)
    if not c["train"]:
        return {"h": h.detach()}
    loss = (h * s["dh"].double()).sum() + (lv["x"] * s["dres"].double()).sum()
    g = _grads64(loss, lv)
    return _some(h=h.detach(), dx=g["x"], dweight=g.get("weight"), dscale=g.get("scale"), dshift=g.get("shift"))


def _exact_norm_out(s):
    c = s["case"]
    T, d, k = c["T"], c["d"], c["k"]
    y = s["y"].double()
    if s["inv_pos"] is not None:
        y[(s["inv_pos"] < 0).nonzero().squeeze(1)] = 0
    total = sum(y[j::k] for j in range(k))
    if s["add"] is not None:
        total = total + s["add"].double()
    lv = dict(y=total.requires_grad_(True), gate=_leaf(s["gate"]), weight=_leaf(s["weight"]))
    parts, end = [], 0
    for i, a, e in _sample_rows(s):
        v = _rms64(lv["y"][a:e])
        if lv["weight"] is not None:
            v = lv["weight"] * v
        parts.append(v if lv["gate"] is None else v * lv["gate"][i])
        end = e
    parts.append(torch.zeros(T - end, d, dtype=torch.float64, device=DEV))
    out = torch.cat(parts) + c["alpha"] * s["x"].double()
    if not c["train"]:
        return {"out": out.detach()}
    g = _grads64((out * s["dout"].double()).sum(), lv)
    return _some(out=out.detach(), dy=g["y"], dgate=g.get("gate"), dweight=g.get("weight"))


def _exact_route(s):
    c = s["case"]
    T, E, k, G = c["T"], c["E"], c["k"], c["n_group"]
    lg = _leaf(s["logits"])
    score = torch.softmax(lg, 1) if c["score"] == "softmax" else torch.sigmoid(lg)
    with torch.no_grad():
        left = score + (0 if s["bias"] is None else s["bias"].double())
        if c["topk_group"] < G:
            per = left.reshape(T, G, E // G).clone()
            first = per.amax(2)
            per.scatter_(2, per.argmax(2, keepdim=True), -math.inf)
            val = first + per.amax(2)
            ok = torch.zeros(T, G, dtype=torch.bool, device=DEV)
            for _ in range(c["topk_group"]):
                m = (val == val.amax(1, keepdim=True)).int().argmax(1, keepdim=True)  # the first of equal ones
                ok.scatter_(1, m, True)
                val.scatter_(1, m, -math.inf)
            left = left.masked_fill(~ok.unsqueeze(2).expand(T, G, E // G).reshape(T, E), -math.inf)
        cols = []
        for _ in range(k):
            m = (left == left.amax(1, keepdim=True)).int().argmax(1, keepdim=True)
            cols.append(m)
            left = left.scatter(1, m, -math.inf)
        ids = torch.cat(cols, 1)
    w = torch.gather(score, 1, ids)
    if c["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    w = 2.5 * w
    if s["live"] is not None:
        w = w * s["live"].double().unsqueeze(1)
        ids = ids.masked_fill(~s["live"].unsqueeze(1), -1)
    res = {"ids": ids.to(torch.int32), "w": w.detach()}
    if c["train"]:
        res["dlogits"] = torch.autograd.grad((w * s["dw"].double()).sum(), lg)[0]
    return res


def _exact_clip(s):
    every = s["grads"][:s["n_large"]] + [s["bucket"]]
    norm = math.sqrt(sum(g.double().square().sum().item() for g in every))
    coef = min(1.0, s["max_norm"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64, device=DEV),
            "grads": [g.double() * coef for g in every[:-1]], "bucket": every[-1].double() * coef}
