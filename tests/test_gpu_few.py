"""A routed layer for a few tokens in two kernels against the formula in 64 bits.

Bound, by the steps: [g | u] sums d products in fp32 (2^-23 of the magnitudes per addition); silu within 2^-20; the activation
enters its product with 16 bits (2^-16), fp16 weights with 16 (2^-16); h products in fp32; the slots' sum 2^-21; one rounding to
the output's type.  8-bit experts: x is quantised exactly, and the activation moves by what its own error moves it across borders
of the 8 bits (`moved`)."""
import pytest
import torch

import f8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ops():
    from trenowanie_generatora_obrazkow_amd import ops
    return ops


def rand(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


def weights(kind, E, d, h, dtype, seed=0):
    """(what the call takes, the values in 64 bits) of both stacks."""
    from trenowanie_generatora_obrazkow_amd.hf_compat import _quant_int8
    o = ops()
    wt = dtype if kind in ("bf16", "fp16") else torch.bfloat16
    w1, w2 = rand(E, d, 2 * h, seed=seed + 1, dtype=wt, std=d ** -0.5), rand(E, h, d, seed=seed + 2, dtype=wt, std=h ** -0.5)
    if kind == "int8":
        (q1, s1), (q2, s2) = _quant_int8(w1), _quant_int8(w2)
        return dict(wgu=q1, wd=q2, wgu_s=s1, wd_s=s2.float()), (q1.double() * s1.double()[:, None], q2.double() * s2.double()[:, None])
    if kind == "fp8":
        f1, f2 = o.F8Stack.from_weights(w1, halves=2), o.F8Stack.from_weights(w2)
        return dict(wgu=f1, wd=f2), (f1.dequant().double(), f2.dequant().double())
    return dict(wgu=w1, wd=w2), (w1.double(), w2.double())


def reference(x, ids, tw, w1, w2, fp8, add=None):
    """(out, bound of its error before the last rounding) in 64 bits."""
    T, k = ids.shape
    E, d, h2 = w1.shape
    h = h2 // 2
    X = x.double().cpu()
    if fp8:
        X = R.quant(X)[0]
    out, err = torch.zeros(T, d, dtype=torch.float64), torch.zeros(T, d, dtype=torch.float64)
    w1, w2, tw = w1.cpu(), w2.cpu(), tw.double().cpu()
    for t in range(T):
        for s in range(k):
            e = int(ids[t, s])
            if not 0 <= e < E:
                continue
            gu, mag = X[t] @ w1[e], (d + 16) * 2.0 ** -23 * (X[t].abs() @ w1[e].abs())
            g, u = gu.split(h)
            eg, eu = mag.split(h)
            silu = g * torch.sigmoid(g)
            act = silu * u
            ea = 1.1 * eg * (u.abs() + eu) + eu * silu.abs() + 2.0 ** -20 * act.abs()
            if fp8:
                q = lambda a: R.quant(a[None])[0][0]
                far = torch.where(act < 0, -ea, ea)
                a8 = q(act)
                ea = torch.maximum((q(act + far) - a8).abs(), (q(act - far) - a8).abs())
                act = a8
            else:
                ea = ea + 2.0 ** -16 * act.abs()
            y, m = act @ w2[e], act.abs() @ w2[e].abs()
            out[t] += tw[t, s] * y
            err[t] += tw[t, s].abs() * (ea @ w2[e].abs() + ((h + 16) * 2.0 ** -23 + 2.0 ** -16 + 2.0 ** -21) * m)
    if add is not None:
        out = out + add.double().cpu()
        err = err + 2.0 ** -22 * add.double().cpu().abs()
    return out, err


def check(y, ref, err, dtype):
    y = y.double().cpu()
    tol = err + HALF[dtype] * (ref.abs() + err) + (2.0 ** -25 if dtype is torch.float16 else 0)
    assert ((y - ref).abs() <= tol).all(), float(((y - ref).abs() / tol.clamp(min=1e-300)).max())


def routing(T, E, k, seed=0, same=False, drop=False):
    g = torch.Generator().manual_seed(seed)
    if same:
        ids = torch.randint(0, E, (T, k), generator=g)
    else:
        ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    if drop:
        ids[0, 0], ids[T // 2, k - 1] = -1, E + 7
    return ids.int().to(DEV), torch.rand(T, k, generator=g).to(DEV)


CASES = [  # T, E, k, d, h, same ids within a token, dropped ids
    (1, 1, 1, 16, 16, False, False),
    (1, 8, 2, 64, 48, False, False),
    (2, 5, 3, 208, 144, False, True),
    (5, 3, 2, 272, 336, False, False),
    (16, 3, 2, 144, 272, True, True),
    (16, 1, 2, 128, 64, True, False),     # every row one expert's: 32 rows
    (7, 40, 8, 400, 96, False, True),
    (16, 200, 16, 48, 32, False, False),  # 256 rows
    (3, 4, 2, 2064, 528, False, False),
]


@pytest.mark.parametrize("kind,dtype", [("bf16", torch.bfloat16), ("fp16", torch.float16), ("int8", torch.bfloat16),
                                        ("int8", torch.float16), ("fp8", torch.bfloat16), ("fp8", torch.float16)])
@pytest.mark.parametrize("T,E,k,d,h,same,drop", CASES)
def test_experts(T, E, k, d, h, same, drop, kind, dtype):
    o = ops()
    w, (w1, w2) = weights(kind, E, d, h, dtype)
    x = rand(T, d, seed=3, dtype=dtype)
    ids, tw = routing(T, E, k, T + d, same, drop)
    add = rand(T, d, seed=4, dtype=dtype) if k > 1 else None
    y = o.few_experts(x, ids, tw, add=add, **w)
    check(y, *reference(x, ids, tw, w1, w2, kind == "fp8", add), dtype)
    assert torch.equal(y, o.few_experts(x, ids, tw, add=add, **w))  # the same bits whichever workgroup comes last
    assert torch.equal(y, o.few_experts(x, ids.long(), tw, add=add, **w))


@pytest.mark.parametrize("d,h", [(8, 8), (24, 8), (72, 200), (1000, 712)])
def test_odd_widths(d, h):
    o = ops()
    for kind, dtype in (("bf16", torch.bfloat16), ("fp16", torch.float16)):
        w, (w1, w2) = weights(kind, 6, d, h, dtype)
        x = rand(4, d, seed=3, dtype=dtype)
        ids, tw = routing(4, 6, 2, d)
        check(o.few_experts(x, ids, tw, **w), *reference(x, ids, tw, w1, w2, False), dtype)


def test_large_activations_in_fp16():
    """Activations past fp16's largest number: the sums stay finite where the output does."""
    o = ops()
    E, d, h = 2, 64, 64
    w = dict(wgu=rand(E, d, 2 * h, seed=1, dtype=torch.float16, std=20.0), wd=rand(E, h, d, seed=2, dtype=torch.float16, std=2e-4))
    x = rand(2, d, seed=3, dtype=torch.float16, std=4.0)
    ids, tw = routing(2, E, 1)
    y = o.few_experts(x, ids, tw, **w)
    ref, err = reference(x, ids, tw, w["wgu"].double(), w["wd"].double(), False)
    assert torch.isfinite(y).all()
    check(y, ref, err, torch.float16)


def test_no_expert_at_all():
    o = ops()
    w, _ = weights("bf16", 4, 64, 48, torch.bfloat16)
    x, add = rand(3, 64), rand(3, 64, seed=8)
    ids = torch.full((3, 2), -1, dtype=torch.int32, device=DEV)
    tw = torch.ones(3, 2, device=DEV)
    assert torch.equal(o.few_experts(x, ids, tw, **w), torch.zeros_like(x))
    assert torch.equal(o.few_experts(x, ids, tw, add=add, **w), add)


def test_types_strides_and_nan():
    o = ops()
    w, (w1, w2) = weights("bf16", 5, 64, 48, torch.bfloat16)
    big = rand(6, 160, seed=2)
    x = big[:, 32:96]
    ids, tw = routing(6, 5, 2, 1)
    y = o.few_experts(x, ids, tw, **w)
    assert torch.equal(y, o.few_experts(x.contiguous(), ids, tw, **w))
    for t in (torch.bfloat16, torch.float16):
        assert torch.equal(o.few_experts(x, ids, tw.to(t), **w), o.few_experts(x, ids, tw.to(t).float(), **w))
    x2 = x.clone()
    x2[3, 7] = float("nan")
    y2 = o.few_experts(x2, ids, tw, **w)
    assert torch.isnan(y2[3]).all()
    keep = [0, 1, 2, 4, 5]
    assert torch.equal(y2[keep], y[keep])
    tw2 = tw.clone()
    ids2 = ids.clone()
    ids2[0, 1], tw2[0, 1] = -5, float("nan")  # a slot that names no expert, whatever its weight
    assert torch.isfinite(o.few_experts(x, ids2, tw2, **w)).all()


def test_empty():
    o = ops()
    w, _ = weights("bf16", 4, 64, 48, torch.bfloat16)
    y = o.few_experts(rand(0, 64), torch.empty(0, 2, dtype=torch.int32, device=DEV), torch.empty(0, 2, device=DEV), **w)
    assert y.shape == (0, 64)


@pytest.mark.parametrize("T", [1, 3, 16])
@pytest.mark.parametrize("E,k,d,h,renorm,biased", [(1, 1, 64, 48, True, False), (16, 2, 256, 64, True, True), (8, 8, 72, 64, False, False),
                                                   (13, 3, 1000, 40, True, True), (40, 4, 128, 64, True, True), (256, 16, 64, 16, True, False)])
def test_with_router(T, E, k, d, h, renorm, biased):
    """The router's ids and weights to the last bit, and the output of few_experts on them."""
    o = ops()
    w, _ = weights("bf16", E, d, h, torch.bfloat16)
    x, wr = rand(T, d, seed=T), rand(E, d, seed=5, std=d ** -0.5)
    bias = rand(E, seed=6, dtype=torch.float32) if biased else None
    if biased and E > k:
        bias[E // 2] = -float("inf")
    y, ids, tw = o.few_forward(x, wr, w["wgu"], w["wd"], k, bias=bias, renorm=renorm, scaling=1.5)
    _, ids2, tw2 = o.route_topk(x, wr, k, bias=bias, renorm=renorm, scaling=1.5)
    assert torch.equal(ids, ids2) and torch.equal(tw, tw2)
    assert torch.equal(y, o.few_experts(x, ids2, tw2, **w))


def test_against_the_layers_other_forms():
    """Within the roundings that those make on the way (bf16 activations, weights and outputs of the slots: six of 2^-8)."""
    o = ops()
    T, E, k, d, h = 16, 8, 2, 256, 192
    w, _ = weights("bf16", E, d, h, torch.bfloat16)
    x, wr = rand(T, d), rand(E, d, seed=5, std=d ** -0.5)
    y, _, _ = o.few_forward(x, wr, w["wgu"], w["wd"], k)
    z, _, _, _ = o.moe_forward(x, wr, w["wgu"], w["wd"], k)
    assert float((y.double() - z.double()).norm() / z.double().norm()) < 6 * 2.0 ** -8 / 3 ** 0.5


def test_graph_two_streams():
    """Replays with other inputs and routing, beside an eager call on another stream with its own workspace."""
    o = ops()
    T, E, k, d, h = 4, 16, 2, 256, 320
    w, _ = weights("bf16", E, d, h, torch.bfloat16)
    x, wr = rand(T, d), rand(E, d, seed=5, std=d ** -0.5)
    run = lambda: o.few_forward(x, wr, w["wgu"], w["wd"], k)
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    side = torch.cuda.Stream()
    for i in range(5):
        x.copy_(rand(T, d, seed=30 + i))
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(side):
            other = run()
        torch.cuda.synchronize()
        for a, b, c in zip(out, want, other):
            assert torch.equal(a, b) and torch.equal(c, b)
