"""SwiGLU with an 8-bit checkpoint, by itself and in the routed layer, against the formulas in 64 bits.

Bounds: what is kept is exact (tests/f8_ref.py).  act, dgu and the second activation are formed in fp32 with an approximate
exponential and reciprocal (within 2^-20 relative) and rounded once: half a step of the type.  A row's weight gradient is a sum
of h products: 2^-20 + h 2^-24 of the sum of their magnitudes."""
import pytest
import torch

import f8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALL = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half the smallest step


def ops():
    from trenowanie_generatora_obrazkow_amd import ops
    return ops


def rand(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


def near(y, ref, dtype, extra=2.0 ** -20):
    y, ref = y.double().cpu(), ref.cpu()
    tol = (HALF[dtype] + extra * (1 + HALF[dtype])) * ref.abs() + SMALL[dtype]
    assert ((y - ref).abs() <= tol).all(), float(((y - ref).abs() / tol.clamp(min=1e-300)).max())


def kept_values(gu):
    h = gu.shape[1] // 2
    return torch.cat([R.quant(gu[:, :h], 32)[0], R.quant(gu[:, h:], 32)[0]], 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,h", [(1, 8), (3, 40), (130, 64), (33, 120), (7, 264), (65, 1352), (5, 4096)])
def test_forward_and_backward(M, h, dtype):
    o = ops()
    gu = rand(M, 2 * h, seed=M + h, dtype=dtype, std=1.5)
    act, kept = o.swiglu_pack(gu)
    g, u = gu.double().cpu().split(h, 1)
    near(act, g * torch.sigmoid(g) * u, dtype)
    want = kept_values(gu)
    assert torch.equal(kept.dequant().double().cpu(), want)
    dh, w = rand(M, h, seed=1, dtype=dtype), torch.rand(M, generator=torch.Generator().manual_seed(2)).to(DEV)
    w[0] = 0.0
    dgu, act2, dw = o.swiglu_pack_bwd(dh, kept, w)
    g, u = want.split(h, 1)
    s = torch.sigmoid(g)
    d, wd = dh.double().cpu(), w.double().cpu()[:, None]
    near(act2, g * s * u, dtype)
    near(dgu[:, h:], wd * d * g * s, dtype)
    # s + g s (1 - s) cancels near its zero at g = -1.28: the error goes by its terms
    ref, tol = wd * d * u * (s + g * s * (1 - s)), wd * d.abs() * u.abs() * (s + (g * s * (1 - s)).abs())
    got = dgu[:, :h].double().cpu()
    assert ((got - ref).abs() <= HALF[dtype] * ref.abs() + 2.0 ** -20 * 2 * tol + SMALL[dtype]).all()
    ref, mag = (d * g * s * u).sum(1), (d * g * s * u).abs().sum(1)
    assert ((dw.double().cpu() - ref).abs() <= (2.0 ** -20 + h * 2.0 ** -24) * mag).all()


def test_gradient_against_differences():
    """dgu at the kept values against central differences of sum(dh w silu(g) u) in 64 bits (step 2^-10: an error of the
    order of 2^-20 of the third derivative, at most 1)."""
    o = ops()
    M, h = 9, 72
    gu = rand(M, 2 * h, seed=5, std=1.2)
    _, kept = o.swiglu_pack(gu)
    dh, w = rand(M, h, seed=6), torch.rand(M, device=DEV)
    dgu, _, _ = o.swiglu_pack_bwd(dh, kept, w)
    v, d = kept.dequant().double().cpu(), dh.double().cpu() * w.double().cpu()[:, None]
    f = lambda g, u: d * g * torch.sigmoid(g) * u
    g, u = v.split(h, 1)
    e = 2.0 ** -10
    diff = torch.cat([(f(g + e, u) - f(g - e, u)) / (2 * e), (f(g, u + e) - f(g, u - e)) / (2 * e)], 1)
    scale = torch.cat([(d * u).abs(), d.abs() * (g.abs() + 1)], 1)
    assert ((dgu.double().cpu() - diff).abs() <= 2.0 ** -8 * diff.abs() + 2.0 ** -18 * scale).all()


def test_order_and_without():
    o = ops()
    M, h = 50, 96
    _, kept = o.swiglu_pack(rand(M, 2 * h))
    dh = rand(M, h, seed=3)
    order = torch.randperm(M, generator=torch.Generator().manual_seed(1)).int().to(DEV)
    for wt in (torch.float32, torch.bfloat16, torch.float16):
        w = torch.rand(M, device=DEV).to(wt)
        dgu, act, dw = o.swiglu_pack_bwd(dh, kept, w, order)
        dgu2, none, dw2 = o.swiglu_pack_bwd(dh, kept, w.float(), want_act=False)
        assert none is None and torch.equal(dgu, dgu2) and torch.equal(dw[order.long()], dw2)
    a, _, none = o.swiglu_pack_bwd(dh, kept, want_dw=False)
    assert none is None and torch.equal(a, o.swiglu_pack_bwd(dh, kept, torch.ones(M, device=DEV))[0])


def test_strided_rows_and_what_is_not_finite():
    o = ops()
    h = 48
    big = rand(20, 160, seed=4)
    gu = big[:, 16:16 + 2 * h]
    act, kept = o.swiglu_pack(gu)
    a2, k2 = o.swiglu_pack(gu.contiguous())
    assert torch.equal(act, a2) and torch.equal(kept.q.view(torch.uint8), k2.q.view(torch.uint8))
    x = gu.contiguous()
    x[3, 5], x[4, h + 7] = float("inf"), float("nan")
    _, kept = o.swiglu_pack(x)
    v, want = kept.dequant().double().cpu(), kept_values(x)
    assert torch.equal(torch.isnan(v), torch.isnan(want)) and int(torch.isnan(v).sum()) == 2
    assert torch.equal(torch.nan_to_num(v), torch.nan_to_num(want))
    dgu, act, dw = o.swiglu_pack_bwd(rand(20, h, seed=8), kept)
    bad = torch.isnan(dw).cpu()
    assert bad.nonzero()[:, 0].tolist() == [3, 4]
    assert int(torch.isnan(act).sum()) == 2


def test_empty():
    o = ops()
    act, kept = o.swiglu_pack(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16))
    dgu, a, dw = o.swiglu_pack_bwd(torch.empty(0, 32, device=DEV, dtype=torch.bfloat16), kept)
    assert act.shape == (0, 32) and dgu.shape == (0, 64) and dw.shape == (0,)


def test_down_dgrad():
    o = ops()
    E, T, k, d, h = 3, 40, 2, 64, 72
    ids = torch.randint(0, E, (T, k), generator=torch.Generator().manual_seed(0)).int().to(DEV)
    disp = o.dispatch(ids, E, want_xs=False)
    dy, wd = rand(T, d, seed=1), rand(E, h, d, seed=2)
    dh = o.down_dgrad(dy, wd, disp.counts, T * k, a_idx=disp.a_idx)
    e = torch.repeat_interleave(torch.arange(E), disp.counts.long().cpu())
    a, w = dy.double().cpu()[disp.a_idx.long().cpu()], wd.double().cpu()
    ref = torch.stack([a[i] @ w[e[i]].t() for i in range(T * k)])
    mag = torch.stack([a[i].abs() @ w[e[i]].t().abs() for i in range(T * k)])
    assert ((dh.double().cpu() - ref).abs() <= 2.0 ** -8 * ref.abs() + (d + 8) * 2.0 ** -23 * mag).all()


# ---------------------------------------------------------------------------------------------------------------
# In the layer
# ---------------------------------------------------------------------------------------------------------------
def layer(T, d, E, k, h, dtype=torch.bfloat16, **kw):
    from trenowanie_generatora_obrazkow_amd import MoESwiGLU
    torch.manual_seed(T)
    m = MoESwiGLU(d, h, E, k, device=DEV, dtype=dtype, **kw)
    x = rand(T, d, seed=T).requires_grad_(True)
    return m, x, rand(T, d, seed=T + 1)


def step(m, x, dy):
    m.zero_grad(set_to_none=True)
    x.grad = None
    y = m(x)
    y.backward(dy)
    m.last_topk_weight = None
    return [y.detach()] + [t.grad for t in (x, m.router_weight, m.w_gu, m.w_d)]


@pytest.mark.parametrize("T,d,E,k,h,dtype", [(1, 16, 2, 1, 8, torch.bfloat16), (50, 64, 4, 2, 72, torch.float32),
                                             (300, 128, 5, 3, 264, torch.bfloat16)])
def test_layer(T, d, E, k, h, dtype):
    """Gradients against the formulas at the kept values, in 64 bits.  Each tensor passes at most five roundings to bf16 on its
    way (rms 2^-8 / sqrt(3) each at most, independent): 2-norm of the error at most 2 sqrt(5 / 3) 2^-8 of the gradient's; a
    quarter of that again for values of [g | u] that the products' order moves across a border of the 8 bits."""
    from trenowanie_generatora_obrazkow_amd import MoESwiGLU, ops as o
    m, x, dy = layer(T, d, E, k, h, dtype, checkpoint="fp8")
    y, dx, dwr, dwgu, dwd = step(m, x, dy)
    with torch.no_grad():
        wr, wgu, wd = (p.to(torch.bfloat16) for p in (m.router_weight, m.w_gu, m.w_d))
        logits, ids, tw = o.route_topk(x, wr, k, bias=m.logit_bias)
    X, W1, W2, D = (t.detach().double().cpu() for t in (x, wgu, wd, dy))
    wr64, ids = wr.detach().double().cpu(), ids.long().cpu()
    z = (X @ wr64.t()).requires_grad_(True)
    p = torch.softmax(z, 1).gather(1, ids)
    w = p / p.sum(1, keepdim=True)
    dX, dW1, dW2, dw, Y = torch.zeros_like(X), torch.zeros_like(W1), torch.zeros_like(W2), torch.zeros(T, k).double(), torch.zeros_like(X)
    for e in range(E):
        t, slot = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        gu = (X[t] @ W1[e]).to(torch.bfloat16)
        we = w.detach()[t, slot][:, None]
        g, u = gu.double().split(h, 1)
        Y.index_add_(0, t, we * ((g * torch.sigmoid(g) * u) @ W2[e]))
        g, u = kept_values(gu).split(h, 1)
        s = torch.sigmoid(g)
        act, dh = g * s * u, D[t] @ W2[e].t()
        dw[t, slot] = (dh * act).sum(1)
        dgu = we * torch.cat([dh * u * (s + g * s * (1 - s)), dh * g * s], 1)
        dX.index_add_(0, t, dgu @ W1[e].t())
        dW1[e], dW2[e] = X[t].t() @ dgu, act.t() @ (we * D[t])
    z.grad = None
    w.backward(dw)
    dX += z.grad @ wr64
    lim = 1.25 * 2 * (5 / 3) ** 0.5 * 2.0 ** -8
    for name, a, b in (("y", y, Y), ("dx", dx, dX), ("dwgu", dwgu, dW1), ("dwd", dwd, dW2)):
        err = float((a.double().cpu() - b).norm() / b.norm().clamp(min=1e-300))
        assert err <= lim, (name, err, lim)
    if k > 1:
        b = z.grad.t() @ X
        assert float((dwr.double().cpu() - b).norm() / b.norm()) <= lim
    assert dwgu.dtype == dtype and dwd.dtype == dtype


def test_layer_keeps_less():
    def kept(ck):
        m, x, dy = layer(2048, 256, 8, 2, 512, checkpoint=ck)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = m(x)
        torch.cuda.synchronize()
        n = torch.cuda.memory_allocated() - before
        y.backward(dy)
        return n
    M, d, h = 4096, 256, 512
    assert kept("fp8") < 0.55 * kept(None)
    assert kept(None) - kept("fp8") > 0.9 * (2 * M * (d + 3 * h) - M * 2 * h * 33 // 32)


def test_same_routing_and_options():
    from trenowanie_generatora_obrazkow_amd import Gate
    for gate in (None, Gate(score="sigmoid", scaling=2.0)):
        m, x, dy = layer(120, 64, 6, 2, 64, gate=gate, balance=gate is not None)
        a = step(m, x, dy)
        ids = m.last_topk_ids
        m.checkpoint = "fp8"
        b = step(m, x, dy)
        assert torch.equal(ids, m.last_topk_ids)
        for u, v in zip(a, b):  # an e4m3 rounding is at most 2^-4 of its value
            assert float((u.double() - v.double()).norm() / u.double().norm()) < 2.0 ** -3
        with torch.no_grad():
            y1 = m(x)
            m.checkpoint = None
            assert torch.equal(y1, m(x))


def test_residual_block():
    from trenowanie_generatora_obrazkow_amd import MoEResidual
    torch.manual_seed(0)
    r = MoEResidual(64, 72, 4, 2, post_norm=True, device=DEV, checkpoint="fp8")
    x = rand(2, 40, 64).requires_grad_(True)
    sc, sh, ga = (rand(2, 64, seed=i, std=0.1).requires_grad_(True) for i in range(3))
    dy = rand(2, 40, 64, seed=9)
    grads = []
    for ck in ("fp8", None):
        r.mlp.checkpoint = ck
        r.zero_grad(set_to_none=True)
        for t in (x, sc, sh, ga):
            t.grad = None
        r(x, sc, sh, ga).backward(dy)
        grads.append([t.grad.double() for t in (x, sc, sh, ga, *r.parameters())])
    for a, b in zip(*grads):
        assert float((a - b).norm() / b.norm()) < 2.0 ** -3


def test_step_graph():
    from trenowanie_generatora_obrazkow_amd.graphs import StepGraph
    m, x, dy = layer(256, 64, 4, 2, 96, checkpoint="fp8")
    g = StepGraph(lambda: step(m, x, dy))
    for i in range(4):
        with torch.no_grad():
            x.copy_(rand(256, 64, seed=20 + i))
        want = [t.clone() for t in step(m, x, dy)]
        torch.cuda.synchronize()
        got = g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_frozen_parts():
    m, x, dy = layer(64, 32, 3, 2, 40, checkpoint="fp8")
    full = step(m, x, dy)
    m.w_d.requires_grad_(False)
    part = step(m, x, dy)
    assert part[4] is None and all(torch.equal(a, b) for a, b in zip(full[:4], part[:4]))
    m.w_gu.requires_grad_(False)
    x2 = x.detach().requires_grad_(True)
    part = step(m, x2, dy)
    assert part[3] is None and torch.equal(part[1], full[1])


def test_backward_twice():
    m, x, dy = layer(32, 32, 3, 2, 40, checkpoint="fp8")
    y = m(x)
    y.backward(dy, retain_graph=True)
    first = x.grad.clone()
    x.grad = None
    y.backward(dy)
    assert torch.equal(first, x.grad)  # twice over one forward: what was kept is read, not consumed
    with pytest.raises(RuntimeError):
        y.backward(dy)
