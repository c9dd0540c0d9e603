"""Experts in 8-bit floating point, their form for a few tokens, and 8-bit checkpoints of the SwiGLU: what their speed is
measured on, with their plain forms.

Kinds:
  mm8      grouped product of rows quantised on the way (e4m3, a power-of-two scale per 128 columns) with expert stacks kept
           in e4m3 (a scale per 128 x 128 block); with train, the gradient of the rows too
  experts8 both projections of a routed SwiGLU layer over such stacks, for given routing
  few      a whole routed layer for a few tokens: bf16, fp16, int8 or 8-bit float experts
  pack     SwiGLU that keeps [g | u] in 8 bits (a scale per 32 columns), and its backward from what it kept

Where `own` is false, `run` computes the plain form (elementary torch operations in 32 bits, rounded once); where it is true
it calls the framework's operators.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_F8 = torch.float8_e4m3fn


def listed():
    return [
        # a handful of rows over small experts in fp16, gathered, scattered and scaled, one expert empty: latency
        dict(name="mm8_40_fp16", kind="mm8", M=40, E=6, K=208, N=336, dtype="fp16", extras=True, train=False),
        # a packed prompt batch, uneven experts, widths off the blocks
        dict(name="mm8_6000", kind="mm8", M=6000, E=12, K=1008, N=2000, dtype="bf16", extras=True, train=False),
        # the gate/up projection of a layer on four 1024 px images, and the gradient of its rows: the largest
        dict(name="mm8_32768_train", kind="mm8", M=32768, E=16, K=1536, N=8192, dtype="bf16", extras=False, train=True),
        # a short prompt: a few rows per expert, every expert's weights streamed once
        dict(name="experts8_48", kind="experts8", T=48, E=64, k=6, d=2048, h=1408, dtype="bf16"),
        # the text encoder's experts on a few captions
        dict(name="experts8_1500", kind="experts8", T=1500, E=128, k=8, d=2048, h=320, dtype="bf16"),
        # the layer on four 1024 px images
        dict(name="experts8_16384", kind="experts8", T=16384, E=16, k=2, d=1536, h=4096, dtype="bf16"),
        # one token through the layer with its own router
        dict(name="few_1", kind="few", T=1, E=16, k=2, d=1536, h=4096, weights="bf16", dtype="bf16", router=True,
             add=False, dropped=False),
        # one token through the text encoder's int8 experts, the shared expert's output added
        dict(name="few_1_int8", kind="few", T=1, E=128, k=8, d=2048, h=320, weights="int8", dtype="bf16", router=False,
             add=True, dropped=False),
        # sixteen sequences, a token each, over 8-bit float experts
        dict(name="few_16_fp8", kind="few", T=16, E=64, k=6, d=2048, h=1408, weights="fp8", dtype="bf16", router=False,
             add=False, dropped=False),
        # seven tokens in fp16, widths off every tile, an expert id out of range
        dict(name="few_7_fp16", kind="few", T=7, E=10, k=3, d=1000, h=712, weights="fp16", dtype="fp16", router=False,
             add=False, dropped=True),
        # a small layer's rows
        dict(name="pack_700_fp16", kind="pack", M=700, h=1352, dtype="fp16"),
        # the rows of a training step on four 1024 px images
        dict(name="pack_32768", kind="pack", M=32768, h=4096, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("mm8", "experts8", "few", "pack"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "mm8":
        train = rng.random() < 0.4
        c = dict(kind=kind, E=rng.randint(1, 40), K=16 * _log_int(rng, 4, 256), N=16 * _log_int(rng, 4, 512), dtype=dtype,
                 extras=not train, train=train)
        while c["E"] * c["K"] * c["N"] > 16 * 1536 * 8192:
            c["E"] = max(1, c["E"] // 2)
        most = 32768 * 1536 * 8192 // (c["K"] * c["N"])
        c["M"] = min(_log_int(rng, 1, 32768), most)
        return c
    if kind == "experts8":
        E = _log_int(rng, 2, 160)
        k = rng.randint(1, min(8, E))
        d, h = 16 * rng.randint(8, 144), 16 * _log_int(rng, 6, 256)
        while E * d * h > 16 * 1536 * 4096 * 2:
            E = max(k, E // 2)
            h = max(96, h // 32 * 16)
        T = min(_log_int(rng, 17, 16384), 32768 * 1536 * 4096 // (k * d * h))
        return dict(kind=kind, T=T, E=E, k=k, d=d, h=h, dtype=dtype)
    if kind == "few":
        weights = rng.choice((dtype, "int8", "fp8"))
        g = 8 if weights == dtype else 16
        E = _log_int(rng, 2, 160)
        k = rng.randint(1, min(8, E))
        router = weights == "bf16" and rng.random() < 0.5
        d, h = g * rng.randint(128 // g, 2304 // g), g * _log_int(rng, 128 // g, 4096 // g)
        while E * d * h > 16 * 1536 * 4096 * 2:
            E = max(k, E // 2)
            h = max(128, h // (2 * g) * g)
        return dict(kind=kind, T=rng.randint(1, 16), E=E, k=k, d=d, h=h, weights=weights, dtype=dtype, router=router,
                    add=rng.random() < 0.3, dropped=not router and k > 1 and rng.random() < 0.3)
    h = 8 * _log_int(rng, 8, 640)
    return dict(kind=kind, M=min(_log_int(rng, 1, 65536), 32768 * 4096 // h), h=h, dtype=dtype)


# ---------------------------------------------------------------------------------------------------------------
# Block scaling in plain torch
# ---------------------------------------------------------------------------------------------------------------
def _scale_exp(amax):
    """The least e >= -126 with amax <= 448 * 2^e."""
    m, e = torch.frexp(amax)
    return torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)


def _blocks(x, n, dim):
    """x with its axis `dim` zero-padded to whole blocks of n and split into (blocks, n)."""
    pad = -x.shape[dim] % n
    if pad:
        shape = list(x.shape)
        shape[dim] = pad
        x = torch.cat([x, x.new_zeros(shape)], dim)
    return x.unflatten(dim, (-1, n))


def _q_rows(x, n=128):
    """The values that fp32 rows x stand for in e4m3 with a scale per n columns."""
    b = _blocks(x, n, 1)
    e = _scale_exp(b.abs().amax(-1, keepdim=True))
    v = torch.ldexp(torch.ldexp(b, -e).to(_F8).float(), e)
    return v.flatten(1)[:, : x.shape[1]]


def _q_stack(w, halves=1):
    """(E, K, N) -> e4m3 values (E, K, N) and their fp32 scales (E, K blocks, N blocks), the N blocks of each of `halves`
    equal column ranges from its first column on."""
    qs, ss = [], []
    for part in w.float().chunk(halves, dim=2):
        K, N = part.shape[1:]
        b = _blocks(_blocks(part, 128, 1), 128, 3)  # (E, KB, 128, NB, 128)
        e = _scale_exp(b.abs().amax((2, 4), keepdim=True))
        q = torch.ldexp(b, -e).to(_F8)
        qs.append(q.flatten(3).flatten(1, 2)[:, :K, :N])
        ss.append(torch.ldexp(torch.ones_like(b[:, :, :1, :, :1]), e).flatten(3)[:, :, 0])
    return torch.cat(qs, 2), torch.cat(ss, 2)


def _wide(q, s, e, halves, dtype):
    """Expert e's weights (K, N) as the values they stand for."""
    K, N = q.shape[1:]
    n = N // halves
    nb = s.shape[2] // halves
    cols = torch.cat([torch.arange(n, device=q.device) // 128 + i * nb for i in range(halves)])
    rows = torch.arange(K, device=q.device) // 128
    return q[e].to(dtype) * s[e].to(dtype)[rows][:, cols]


# ---------------------------------------------------------------------------------------------------------------
# What a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------
def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _rows_in(g, R, d, dtype):
    """Rows of a residual stream behind its norm: unequal sizes, a few channels well above the rest."""
    x = torch.randn(R, d, generator=g, device=DEV) * (0.5 + torch.rand(R, 1, generator=g, device=DEV))
    x[:, :: max(d // 4, 1)] *= 6
    return x.to(dtype)


def _stack(g, E, K, N, halves=1):
    """A stack in 8 bits: what the plain form reads, and the framework's own layout of it."""
    w = _randn(g, E, K, N, std=K ** -0.5)
    q, s = _q_stack(w, halves)
    st = dict(q=q, s=s, halves=halves)
    return st, w


def _own_stack(w, halves=1, grad=False):
    from trenowanie_generatora_obrazkow_amd import F8Stack
    return F8Stack.from_weights(w, halves=halves, grad=grad)


def _gate(g, T, E, k):
    """Experts of uneven load and their renormalised weights."""
    logits = torch.randn(T, E, generator=g, device=DEV) + 0.7 * torch.randn(E, generator=g, device=DEV)
    w, ids = logits.softmax(-1).topk(k, dim=-1)
    return ids.to(torch.int32), w / w.sum(-1, keepdim=True)


def _int8(w):
    s = w.float().abs().amax(dim=1).clamp(min=1e-8) / 127
    return (w.float() / s.unsqueeze(1)).round().clamp(-127, 127).to(torch.int8), s.to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = case
    st = dict(case=c)
    dt = _DT[c["dtype"]]
    if c["kind"] == "mm8":
        M, E, K, N = c["M"], c["E"], c["K"], c["N"]
        load = torch.ones(E, device=DEV)
        load[: E // 3] = 2.0
        if E > 2:
            load[-1] = 0.0
        e = torch.multinomial(load, M, replacement=True, generator=g)
        st["counts"] = torch.bincount(e, minlength=E).to(torch.int32)
        st["w"], w = _stack(g, E, K, N)
        st["a"] = _rows_in(g, M, K, dt)
        if c["extras"]:
            order = torch.argsort(e, stable=True)
            st["a_idx"] = (order // 2).to(torch.int32)  # two rows of a token each
            st["y_idx"] = order.to(torch.int32)
            st["scale"] = torch.rand(M, generator=g, device=DEV)
        if c["train"]:
            st["dy"] = _randn(g, M, N, dtype=dt)
        if own:
            st["own"] = _own_stack(w, grad=c["train"])
            if c["train"]:
                st["a"].requires_grad_(True)
        return st
    if c["kind"] == "pack":
        M, h = c["M"], c["h"]
        st["gu"] = (torch.randn(M, 2 * h, generator=g, device=DEV) * (0.3 + torch.rand(M, 1, generator=g, device=DEV))).to(dt)
        st["dh"] = _randn(g, M, h, dtype=dt)
        st["w"] = torch.rand(M, generator=g, device=DEV)
        return st
    T, E, k, d, h = c["T"], c["E"], c["k"], c["d"], c["h"]
    st["x"] = _rows_in(g, T, d, dt)
    if c.get("router"):
        st["wr"] = _randn(g, E, d, std=d ** -0.5)
        st["bias"] = 0.3 * torch.randn(E, generator=g, device=DEV)
    else:
        st["ids"], st["tw"] = _gate(g, T, E, k)
        if c.get("dropped"):  # a gate's id for no expert
            st["ids"][T // 2, k - 1] = E + 3
    if c.get("add"):
        st["add"] = _randn(g, T, d, dtype=dt)
    kind = "fp8" if c["kind"] == "experts8" else c["weights"]
    if kind == "fp8":
        st["wgu"], w1 = _stack(g, E, d, 2 * h, 2)
        st["wd"], w2 = _stack(g, E, h, d)
        if own:
            st["own"] = (_own_stack(w1, 2), _own_stack(w2))
    else:
        w1 = _randn(g, E, d, 2 * h, std=d ** -0.5, dtype=dt)
        w2 = _randn(g, E, h, d, std=h ** -0.5, dtype=dt)
        if kind == "int8":
            (w1, st["s1"]), (w2, st["s2"]) = _int8(w1), _int8(w2)
        st["w1"], st["w2"] = w1, w2
    return st


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from trenowanie_generatora_obrazkow_amd import ops
    from trenowanie_generatora_obrazkow_amd.moe_triton import grouped_mm
    c = st["case"]
    if c["kind"] == "mm8":
        a = st["a"]
        if c["train"]:
            a.grad = None
            y = grouped_mm(a, st["own"], st["counts"])
            y.backward(st["dy"])
            return [y.detach(), a.grad]
        return [grouped_mm(a, st["own"], st["counts"], a_idx=st.get("a_idx"), y_idx=st.get("y_idx"), scale=st.get("scale"))]
    if c["kind"] == "pack":
        act, kept = ops.swiglu_pack(st["gu"])
        dgu, act_kept, dw = ops.swiglu_pack_bwd(st["dh"], kept, st["w"])
        return [act, dgu, act_kept, dw]
    if c["kind"] == "experts8":
        y, _, _ = ops.moe_experts(st["x"], st["ids"], st["tw"], *st["own"])
        return [y]
    wgu, wd = st["own"] if c["weights"] == "fp8" else (st["w1"], st["w2"])
    if c["router"]:
        return list(ops.few_forward(st["x"], st["wr"], wgu, wd, c["k"], bias=st["bias"], add=st.get("add")))
    return [ops.few_experts(st["x"], st["ids"], st["tw"], wgu, wd, wgu_s=st.get("s1"), wd_s=st.get("s2"), add=st.get("add"))]


def _run_plain(st):
    c = st["case"]
    if c["kind"] == "mm8":
        return _plain_mm8(st)
    if c["kind"] == "pack":
        return _plain_pack(st)
    x = st["x"].float()
    dt = st["x"].dtype
    ids, tw = st.get("ids"), st.get("tw")
    if c.get("router"):
        z = (st["x"].double() @ st["wr"].double().t() + st["bias"].double()).float()
        p = z.softmax(-1)
        tw, ids = p.topk(c["k"], dim=-1)
        tw = tw / tw.sum(-1, keepdim=True)
        ids = ids.to(torch.int32)
    fp8 = c["kind"] == "experts8" or c["weights"] == "fp8"
    T, d = x.shape
    y = torch.zeros(T * c["k"], d, device=DEV)
    xq = _q_rows(x) if fp8 else x
    flat = ids.reshape(-1)
    for e in range(c["E"]):
        rows = (flat == e).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        if fp8:
            w1 = _wide(st["wgu"]["q"], st["wgu"]["s"], e, 2, torch.float32)
            w2 = _wide(st["wd"]["q"], st["wd"]["s"], e, 1, torch.float32)
        else:
            w1, w2 = st["w1"][e].float(), st["w2"][e].float()
            if "s1" in st:
                w1, w2 = w1 * st["s1"][e].float(), w2 * st["s2"][e].float()
        g, u = (xq[rows // c["k"]] @ w1).chunk(2, dim=1)
        act = g / (1 + torch.exp(-g)) * u
        y[rows] = ((_q_rows(act) if fp8 else act) @ w2) * tw.reshape(-1)[rows, None]
    if c["kind"] == "experts8":
        return [y.to(dt)]
    out = y.view(T, c["k"], d).sum(1)
    if "add" in st:
        out = out + st["add"].float()
    return [out.to(dt), ids, tw] if c["router"] else [out.to(dt)]


def _plain_mm8(st):
    c, a = st["case"], st["a"].detach()
    q, s = st["w"]["q"], st["w"]["s"]
    aq = _q_rows(a.float())
    if "a_idx" in st:
        aq = aq[st["a_idx"].long()]
    y = torch.empty(c["M"], c["N"], device=DEV, dtype=a.dtype)
    da = torch.empty(c["M"], c["K"], device=DEV, dtype=a.dtype) if c["train"] else None
    dq = _q_rows(st["dy"].float()) if c["train"] else None
    r0 = 0
    for e, n in enumerate(st["counts"].tolist()):
        r = slice(r0, r0 + n)
        r0 += n
        if n == 0:
            continue
        w = _wide(q, s, e, 1, torch.float32)
        v = aq[r] @ w
        if "scale" in st:
            v = v * st["scale"][r, None]
        y[st["y_idx"][r].long() if "y_idx" in st else r] = v.to(a.dtype)
        if c["train"]:
            da[r] = (dq[r] @ w.t()).to(a.dtype)
    return [y, da] if c["train"] else [y]


def _plain_pack(st):
    gu, dh, w = st["gu"], st["dh"].float(), st["w"]
    h = dh.shape[1]
    g, u = gu.float().split(h, dim=1)
    act = (g / (1 + torch.exp(-g)) * u).to(gu.dtype)
    g, u = _q_rows(g, 32), _q_rows(u, 32)
    sg = 1 / (1 + torch.exp(-g))
    da = dh * w[:, None]
    dgu = torch.cat([da * u * (sg + g * sg * (1 - sg)), da * (g * sg)], 1)
    a = g * sg * u
    return [act, dgu.to(gu.dtype), a.to(gu.dtype), (dh * a).sum(1)]


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "mm8":
        M, E, K, N = c["M"], c["E"], c["K"], c["N"]
        hit = E * (1 - (1 - 1 / E) ** M)
        n = 2 if c["train"] else 1
        rows = 2 * M * (K + N) if not c["extras"] else 2 * (M // 2 + 1) * K + 2 * M * N + 12 * M
        return dict(bytes=int(n * (rows + hit * K * N)), flops=n * 2 * M * K * N)
    if c["kind"] == "pack":
        kept = 2 * c["M"] * c["h"] * (1 + 1 / 32)
        return dict(bytes=int(c["M"] * c["h"] * (4 + 2 + 2 + 4 + 2) + 2 * kept + 8 * c["M"]), flops=30 * c["M"] * c["h"])
    T, E, k, d, h = c["T"], c["E"], c["k"], c["d"], c["h"]
    hit = E * (1 - (1 - k / E) ** T)
    wb = 2 if c.get("weights") in ("bf16", "fp16") else 1
    out = 2 * T * k * d if c["kind"] == "experts8" else 2 * T * d
    b = 2 * T * d + out + hit * 3 * d * h * wb + 8 * T * k
    if c.get("router"):
        b += 2 * E * d
    if c.get("add"):
        b += 2 * T * d
    return dict(bytes=int(b), flops=6 * T * k * d * h + (2 * T * E * d if c.get("router") else 0))


# ---------------------------------------------------------------------------------------------------------------
# The same in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------------------
def _e4m3_64(x, n):
    """Rows of doubles rounded to e4m3 with a power-of-two scale per n columns, by their steps: four significant bits, 2^-9
    the smallest step."""
    out = torch.empty_like(x)
    for c0 in range(0, x.shape[1], n):
        b = x[:, c0:c0 + n]
        top = b.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 448)).clamp(min=-126)
        e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
        e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
        v = b / torch.exp2(e)
        step = torch.exp2((torch.frexp(v)[1] - 4).clamp(min=-9).double())
        out[:, c0:c0 + n] = torch.round(v / step) * step * torch.exp2(e)
    return out


def exact(case, seed):
    with torch.no_grad():
        return _exact(case, prepare(case, seed))


def _exact(c, st):
    if c["kind"] == "mm8":
        a = _e4m3_64(st["a"].detach().double(), 128)
        y = torch.empty(c["M"], c["N"], device=DEV, dtype=torch.float64)
        da = torch.empty(c["M"], c["K"], device=DEV, dtype=torch.float64)
        dy = _e4m3_64(st["dy"].double(), 128) if c["train"] else None
        ends = st["counts"].long().cumsum(0)
        expert = torch.searchsorted(ends, torch.arange(c["M"], device=DEV), right=True)
        src = st["a_idx"].long() if "a_idx" in st else torch.arange(c["M"], device=DEV)
        dst = st["y_idx"].long() if "y_idx" in st else torch.arange(c["M"], device=DEV)
        sc = st["scale"].double() if "scale" in st else torch.ones(c["M"], device=DEV, dtype=torch.float64)
        for e in expert.unique().tolist():
            r = (expert == e).nonzero()[:, 0]
            w = _wide(st["w"]["q"], st["w"]["s"], e, 1, torch.float64)
            y.index_copy_(0, dst[r], sc[r, None] * (a[src[r]] @ w))
            if c["train"]:
                da.index_copy_(0, r, dy[r] @ w.t().contiguous())
        return [y, da] if c["train"] else [y]
    if c["kind"] == "pack":
        h = c["h"]
        gu, dh, w = st["gu"].double(), st["dh"].double(), st["w"].double()[:, None]
        silu = lambda v: v * torch.sigmoid(v)
        kept_g, kept_u = _e4m3_64(gu[:, :h], 32), _e4m3_64(gu[:, h:], 32)
        s = torch.sigmoid(kept_g)
        a = silu(kept_g) * kept_u
        dgu = torch.empty_like(gu)
        dgu[:, :h] = w * dh * kept_u * s * (1 + kept_g * (1 - s))
        dgu[:, h:] = w * dh * silu(kept_g)
        return [silu(gu[:, :h]) * gu[:, h:], dgu, a, (a * dh).sum(1)]
    x = st["x"].double()
    T, d = x.shape
    k = c["k"]
    fp8 = c["kind"] == "experts8" or c["weights"] == "fp8"
    if c.get("router"):
        p = torch.softmax(x @ st["wr"].double().t() + st["bias"].double(), dim=1)
        order = torch.argsort(p, dim=1, descending=True, stable=True)[:, :k]
        tw = p.gather(1, order)
        ids, tw = order.to(torch.int32), tw / tw.sum(1, keepdim=True)
    else:
        ids, tw = st["ids"], st["tw"].double()
    if fp8:
        x = _e4m3_64(x, 128)
    y = torch.zeros(T, k, d, device=DEV, dtype=torch.float64)
    for e in ids.unique().tolist():
        if not 0 <= e < c["E"]:
            continue
        t, slot = (ids == e).nonzero(as_tuple=True)
        if fp8:
            w1, w2 = _wide(**_of(st["wgu"]), e=e), _wide(**_of(st["wd"]), e=e)
        else:
            w1, w2 = st["w1"][e].double(), st["w2"][e].double()
            if "s1" in st:
                w1, w2 = w1 * st["s1"][e].double(), w2 * st["s2"][e].double()
        gu = x[t] @ w1
        act = gu[:, :c["h"]] * torch.sigmoid(gu[:, :c["h"]]) * gu[:, c["h"]:]
        y[t, slot] = tw[t, slot, None] * ((_e4m3_64(act, 128) if fp8 else act) @ w2)
    if c["kind"] == "experts8":
        return [y.view(T * k, d)]
    out = y.sum(1) + (st["add"].double() if "add" in st else 0)
    return [out, ids, tw] if c["router"] else [out]


def _of(s):
    return dict(q=s["q"], s=s["s"], halves=s["halves"], dtype=torch.float64)
