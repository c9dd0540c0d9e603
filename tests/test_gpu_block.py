"""The residual block around the routed layer: the differentiable norms, the layer with sigmoid / grouped / balanced gates,
moe_residual and MoEResidual as one autograd node, and a whole step (norms, routing, experts, backward, clipping) eager and
captured.

Tolerances of the routed gradients.  The layer rounds to bf16 at its input h, g, u, silu(g), act, y and in the backward at dys
and dgu, eight roundings of at most 2^-8 each, less than 2^-9 in the mean.  They are independent, so they add as squares:
sqrt(8) 2^-9 = 5.7 2^-10.  Against a float64 reference with the forward's rounding points: mean error at most 8 2^-10 of the
mean, largest error at most 5 times that of the largest entry."""
import math

import pytest
import torch

from tests import block_ref as R
from tests.util import rel_errors

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32
MEAN, MAX = 8 * 2.0 ** -10, 40 * 2.0 ** -10


def _r16(t):
    """Rounded to bf16, the gradient passing through."""
    return t + (t.detach().float().bfloat16().double() - t.detach())


def _experts64(h, ids, w, wgu, wd):
    """The routed experts' slots summed, (T, d), with the layer's forward rounding points."""
    hh = wd.shape[1]
    out = torch.zeros_like(h)
    w16 = _r16(w)
    for e in range(wgu.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        gu = _r16(h[t] @ wgu[e])
        g, u = gu[:, :hh], gu[:, hh:]
        act = _r16(_r16(g * torch.sigmoid(g)) * u)
        out = out.index_add(0, t, _r16(act @ wd[e] * w16[t, j].unsqueeze(1)))
    return out


def _close(name, got, ref):
    mx, mn = rel_errors(got.detach().float().cpu().numpy(), ref.detach().cpu().numpy())
    print(f"  {name}: max {mx:.2e} mean {mn:.2e}", flush=True)
    assert mx <= MAX and mn <= MEAN, (name, mx, mn)


def _weights(g, d, E, h):
    r = lambda *s, std: (torch.randn(*s, generator=g) * std).bfloat16()
    return r(E, d, std=d ** -0.5 * 2), r(E, d, 2 * h, std=d ** -0.5), r(E, h, d, std=h ** -0.5)


GATES = [
    dict(score="sigmoid", n_group=4, topk_group=2, scaling=2.5),
    dict(score="softmax", n_group=8, topk_group=3, group_top=1),
    dict(score="sigmoid"),
    None,
]


@pytest.mark.parametrize("cfg", GATES, ids=["sig_groups", "soft_groups", "sigmoid", "default"])
@pytest.mark.parametrize("balance", [False, True])
def test_gated_layer(cfg, balance):
    from trenowanie_generatora_obrazkow_amd import Gate, moe_swiglu, ops
    g = torch.Generator().manual_seed(11)
    T, d, E, k, h = 700, 128, 32, 4, 96
    gate = None if cfg is None else Gate(**cfg)
    wr, wgu, wd = _weights(g, d, E, h)
    x = torch.randn(T, d, generator=g).bfloat16()
    sb = (torch.randn(E, generator=g) * 0.2) if balance else None
    dout, dtw = torch.randn(T, d, generator=g).bfloat16(), torch.randn(T, k, generator=g)
    leaves = [t.cuda().requires_grad_(True) for t in (x, wr, wgu, wd)]
    sbd = None if sb is None else sb.cuda()
    print("gated layer", cfg, balance, flush=True)
    out, ids, tw = moe_swiglu(*leaves, k, gate=gate, select_bias=sbd)
    # without a gradient: the same bits
    with torch.no_grad():
        o2, i2, w2 = moe_swiglu(*leaves, k, gate=gate, select_bias=sbd)
    assert torch.equal(out, o2) and torch.equal(ids, i2) and torch.equal(tw, w2)
    # the routing is that of the layer's own logits
    c = cfg or {}
    logits, _, _ = ops.route_topk(x.cuda(), wr.cuda(), 1)
    rid, _ = R.route(logits.cpu(), k, c.get("score", "softmax"), sb, c.get("n_group", 1), c.get("topk_group", 1),
                     c.get("group_top", 2), True, c.get("scaling", 1.0), None)
    assert torch.equal(ids.cpu(), rid)
    grads = torch.autograd.grad([out, tw], leaves, [dout.cuda(), dtw.cuda()])
    lv = [t.double().requires_grad_(True) for t in (x, wr, wgu, wd)]
    idl = ids.cpu().long()
    w64 = R.route_weights(lv[0] @ lv[1].t(), idl, tw.detach().cpu(), c.get("score", "softmax"), True, c.get("scaling", 1.0))
    ref = _experts64(lv[0], idl, w64, lv[2], lv[3])
    _close("out", out, ref)
    rg = torch.autograd.grad((ref * dout.double()).sum() + (w64 * dtw.double()).sum(), lv)
    for n, a, b in zip(("dx", "dwr", "dwgu", "dwd"), grads, rg):
        _close(n, a, b)


@pytest.mark.parametrize("stream,param", [(BF, BF), (FP, FP), (FP, BF)])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_moe_residual(stream, param, post, packed):
    from trenowanie_generatora_obrazkow_amd import Gate, moe_residual, norm_modulate, norm_residual, moe_swiglu
    g = torch.Generator().manual_seed(21)
    T, d, E, k, h, B = 600, 128, 16, 2, 160, 3
    wr, wgu, wd = _weights(g, d, E, h)
    r = lambda *s, std=1.0, dt=param: (torch.randn(*s, generator=g) * std).to(dt)
    x, dout = r(T, d, std=2.0, dt=stream), r(T, d, dt=stream)
    pw, qw = (1 + r(d, std=0.1, dt=FP)).to(param), (1 + r(d, std=0.1, dt=FP)).to(param) if post else None
    sc, sh, gt = r(B, d, std=0.3), r(B, d, std=0.3), r(B, d, std=0.5)
    starts = [0, 250, 250, 590] if packed else None
    std = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    b = R.sample_rows(T, B, starts)
    gate = Gate("sigmoid", 4, 2)
    names = ("x", "wr", "wgu", "wd", "pw", "sc", "sh", "qw", "gt")
    cpu = dict(zip(names, (x, wr, wgu, wd, pw, sc, sh, qw, gt)))
    lv = {n: t.cuda().requires_grad_(True) for n, t in cpu.items() if t is not None}
    call = lambda: moe_residual(lv["x"], lv["wr"], lv["wgu"], lv["wd"], k, lv["pw"], lv["sc"], lv["sh"], lv.get("qw"),
                                lv["gt"], post, std, alpha=0.75, router=gate)
    print("moe_residual", stream, param, post, packed, flush=True)
    out, ids, tw = call()
    assert out.dtype == stream
    with torch.no_grad():
        o2, i2, w2 = call()
    assert torch.equal(out, o2) and torch.equal(ids, i2) and torch.equal(tw, w2)
    grads = dict(zip(lv, torch.autograd.grad(out, list(lv.values()), dout.cuda())))
    # float64 of the whole block
    l64 = {n: t.double().requires_grad_(True) for n, t in cpu.items() if t is not None}
    hh = _r16(R.norm_modulate(l64["x"], l64["pw"], l64["sc"], l64["sh"], b, 1e-6))
    idl = ids.cpu().long()
    w64 = R.route_weights(hh @ l64["wr"].t(), idl, tw.detach().cpu(), "sigmoid", True, 1.0)
    s = _experts64(hh, idl, w64, l64["wgu"], l64["wd"])
    ref = R.norm_residual(s, l64["x"], l64["gt"], l64.get("qw"), post, b, 1e-6, 0.75)
    _close("out", out, ref)
    rg = dict(zip(l64, torch.autograd.grad((ref * dout.double()).sum(), list(l64.values()))))
    for n in lv:
        _close("d" + n, grads[n], rg[n])
    # node by node: the same up to the rounding of the combined rows and of the residual's gradient
    h2 = norm_modulate(lv["x"], lv["pw"], lv["sc"], lv["sh"], std, dtype=BF)
    y2, _, _ = moe_swiglu(h2, lv["wr"], lv["wgu"], lv["wd"], k, gate=gate)
    o3 = norm_residual(lv["x"], y2.to(BF), lv["gt"], lv.get("qw"), post, std, alpha=0.75)
    _close("out, node by node", o3, ref)
    for n, t in zip(lv, torch.autograd.grad(o3, list(lv.values()), dout.cuda())):
        _close("d" + n + ", node by node", t, rg[n])


def test_norm_functions():
    """3-D inputs, parameters for all rows, a strided stream, gradients for some inputs only."""
    from trenowanie_generatora_obrazkow_amd import norm_modulate, norm_residual
    g = torch.Generator().manual_seed(31)
    B, Lr, d = 3, 40, 72
    wide = torch.randn(B, Lr, 2 * d, generator=g)
    x = wide[:, :, d:].cuda().requires_grad_(True)
    w, sc, sh = (torch.randn(*s, generator=g).cuda().requires_grad_(True) for s in ((d,), (B, d), (B, d)))
    h = norm_modulate(x, w, sc, sh)
    assert h.shape == x.shape
    b = torch.arange(B * Lr) // Lr
    c64 = [t.detach().cpu().double().reshape(-1, d) if t.dim() == 3 else t.detach().cpu().double() for t in (x, w, sc, sh)]
    c64 = [t.requires_grad_(True) for t in c64]
    ref = R.norm_modulate(*c64, b, 1e-6)
    u = torch.randn(B, Lr, d, generator=g)
    got = torch.autograd.grad(h, (x, w, sc, sh), u.cuda())
    want = torch.autograd.grad((ref * u.double().view(-1, d)).sum(), c64)
    for a, r in zip(got, want):
        # fp32 throughout: far below 1e-5 of the largest entry (sums of 120 rows)
        assert (a.cpu().double().reshape(r.shape) - r).abs().max() <= 1e-5 * r.abs().max()
    y = torch.randn(B, Lr, d, generator=g).cuda().requires_grad_(True)
    out = norm_residual(x, y, sc, alpha=0.5)
    gx, gy = torch.autograd.grad(out, (x, y), u.cuda())
    assert torch.equal(gx, 0.5 * u.cuda()) and gy.shape == y.shape
    out = norm_residual(x.detach(), y, norm=False)
    assert torch.equal(torch.autograd.grad(out, y, u.cuda())[0], u.cuda())
    with pytest.raises(ValueError):
        norm_residual(x, y[:, :, :64])


def test_gradient_of_the_routing_weights_alone():
    from trenowanie_generatora_obrazkow_amd import Gate, moe_residual
    g = torch.Generator().manual_seed(41)
    T, d, E, k, h = 200, 64, 8, 2, 64
    wr, wgu, wd = (t.cuda().requires_grad_(True) for t in _weights(g, d, E, h))
    x = torch.randn(T, d, generator=g).cuda().requires_grad_(True)
    _, ids, tw = moe_residual(x, wr, wgu, wd, k, router=Gate("sigmoid"))
    dtw = torch.randn(T, k, generator=g)
    gx, gr, gu = torch.autograd.grad(tw, (x, wr, wgu), dtw.cuda())
    x64, r64 = x.detach().cpu().double().requires_grad_(True), wr.detach().cpu().double().requires_grad_(True)
    hh = _r16(R.norm_modulate(x64, None, None, None, torch.zeros(T, dtype=torch.long), 1e-6))
    w64 = R.route_weights(hh @ r64.t(), ids.cpu().long(), tw.detach().cpu(), "sigmoid", True, 1.0)
    rx, rr = torch.autograd.grad((w64 * dtw.double()).sum(), (x64, r64))
    _close("dx", gx, rx)
    _close("dwr", gr, rr)
    assert not gu.any()


def _module(seed, **kw):
    from trenowanie_generatora_obrazkow_amd import MoEResidual
    torch.manual_seed(seed)
    return MoEResidual(128, 192, 16, 2, device="cuda", **kw)


def test_module_parameters_and_state():
    from trenowanie_generatora_obrazkow_amd import Gate, moe_param_groups
    m = _module(1, post_norm=True, gate=Gate("sigmoid", 4, 2), balance=True)
    names = dict(m.named_parameters())
    assert set(names) == {"mlp.router_weight", "mlp.w_gu", "mlp.w_d", "norm_weight", "post_weight"}
    assert "mlp.select_bias" in m.state_dict() and "mlp.select_bias" not in _module(1).state_dict()
    groups, ids = moe_param_groups(m, lr=1e-3, weight_decay=0.1)
    assert ids == {id(names[n]) for n in ("mlp.router_weight", "mlp.w_gu", "mlp.w_d")}
    x = torch.randn(2, 30, 128, device="cuda")
    # the selection bias moves the choice and not the scores: raised for two experts, every token takes them
    with torch.no_grad():
        m.mlp.select_bias[[0, 3]] = 10.0
        m(x)
    assert (m.mlp.last_topk_ids.sort(1).values.cpu() == torch.tensor([0, 3], dtype=torch.int32)).all()
    assert (m.mlp.last_topk_weight.sum(1) - 1).abs().max() < 1e-6


@pytest.mark.parametrize("kw", [dict(), dict(post_norm=True, balance=True, dtype=torch.float32),
                                dict(affine=False, alpha=0.5)], ids=["plain", "post_fp32", "bare"])
@pytest.mark.parametrize("packed", [False, True])
def test_step_with_clipping_eager_and_captured(kw, packed):
    """Two blocks, forward, backward and clipping of every gradient: the norm and the clipped gradients against float64 of the
    unclipped ones, then the same step captured and replayed with inputs that change."""
    from trenowanie_generatora_obrazkow_amd import Gate, clip_grad_norm
    from trenowanie_generatora_obrazkow_amd.graphs import StepGraph
    g = torch.Generator().manual_seed(51)
    B, Lr, d = 4, 100, 128
    blocks = [_module(2, **kw), _module(3, gate=Gate("sigmoid", 4, 2), **kw)]
    params = [p for m in blocks for p in m.parameters()]
    r = lambda *s: torch.randn(*s, generator=g).cuda()
    x, dout = r(B * Lr, d), r(B * Lr, d)
    mods = [[r(B, d) * 0.3 for _ in range(3)] for _ in blocks]
    starts = torch.tensor([0, 90, 90, 200, 395], dtype=torch.int32, device="cuda") if packed else None

    def grads_of(x):
        for p in params:
            p.grad = None
        y = x
        for m, (sc, sh, gt) in zip(blocks, mods):
            y = m(y, sc, sh, gt, starts) if packed else m(y.view(B, Lr, d), sc, sh, gt).view(-1, d)
        y.backward(dout)
        for m in blocks:  # (it carries a gradient and so would keep this step's graph alive into the next one's capture)
            m.mlp.last_topk_weight = None
        return y.detach()

    def step():
        y = grads_of(x)
        return y, clip_grad_norm([p.grad for p in params], 1.0)

    graph = StepGraph(step)
    gg = [p.grad for p in params]  # the captured step's gradients
    for rep in range(3):
        if rep:
            x.copy_(r(B * Lr, d))
        y0 = grads_of(x)
        raw = [p.grad.double() for p in params]
        norm = math.sqrt(sum(float(t.square().sum()) for t in raw))
        y1, n1 = step()
        assert torch.equal(y0, y1) and abs(float(n1) - norm) <= 1e-6 * norm
        for p, t in zip(params, raw):
            ref = t / (norm + 1e-6)
            tol = (2 * R.EPS24 + R.half_step(p.grad.dtype)) * ref.abs() * 1.01 + 2 * R.tiny(p.grad.dtype)
            assert ((p.grad.double() - ref).abs() <= tol).all()
        want = [y1.clone(), n1.clone()] + [p.grad.clone() for p in params]
        y2, n2 = graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([y2, n2] + gg, want)), rep
        torch.ones(64, device="cuda").sum().item()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T", [0, 1])
def test_no_token_and_one(T, gated):
    from trenowanie_generatora_obrazkow_amd import Gate
    m = _module(4, post_norm=True, gate=Gate("sigmoid", 4, 2) if gated else None)
    x = torch.randn(T, 128, device="cuda").requires_grad_(True)
    y = m(x)
    y.sum().backward()
    assert y.shape == x.shape and x.grad.shape == x.shape
    for p in m.parameters():
        assert p.grad.shape == p.shape and torch.isfinite(p.grad).all() and (T > 0 or not p.grad.any())
    with torch.no_grad():
        assert torch.equal(m(x), y)
