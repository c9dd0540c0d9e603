"""Quantisation to 8 bits with block scales, and the grouped products over quantised rows and stacks, against the definitions
in 64 bits (tests/f8_ref.py).

Bounds: the quantised values are exact.  The 8-bit matrix instructions add the products of eight consecutive k at the exponent
of the largest of them and drop what lies below 2^-13 of it (two products 2^p and 1 give their sum up to p = 13 and 2^p above,
where they stand in one group of eight; in different groups up to fp32's 24 bits), so seven products of a group lose less than
7 * 2^-13 of its largest one, itself at most max|a| max|w| over the group (`lost`).  The groups' sums are added in fp32, each
addition off by at most 2^-23 of the sum of the magnitudes, and y is rounded once:
|y - ref| <= 7 * 2^-13 sum over groups of max|a| max|w| + (K + 8) 2^-23 sum|a w| + half a step of y's type."""
import pytest
import torch

import f8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def ops():
    from trenowanie_generatora_obrazkow_amd import ops
    return ops


def rand(*shape, seed=0, dtype=torch.bfloat16, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=g))
    return x.to(dtype).to(DEV)


def lost(a, b, wide=False):
    """Bound of what the products a (M, K) @ b (K, N) lose in their groups of eight."""
    if wide:  # products of bf16 numbers: none
        return 0.0
    ga, gb = (t.abs().unflatten(dim, (-1, 8)).amax(-1 if dim else 1) for t, dim in ((a, 1), (b, 0)))
    return 7 * 2.0 ** -13 * (ga @ gb)


def products(a, b, e, wide=False):
    """a[r] @ b[e[r]] in 64 bits, and the bound of the 8-bit products' own error, sorted rows."""
    M, K = a.shape
    ref = torch.empty(M, b.shape[2], dtype=torch.float64, device=a.device)
    err = torch.empty_like(ref)
    for i in e.unique().tolist():
        r = e == i
        ref[r] = a[r] @ b[i]
        err[r] = lost(a[r], b[i], wide) + (K + 8) * 2.0 ** -23 * (a[r].abs() @ b[i].abs())
    return ref, err


def check(y, ref, err, dtype):
    y, ref, err = y.double().cpu(), ref.cpu(), err.cpu()
    tol = err + HALF[dtype] * (ref.abs() + err)
    if dtype is torch.float16:
        tol = tol + 2.0 ** -25  # half its smallest step
        # its largest number is 65504, with a step of 32: from 65520 on a sum rounds to infinity
        over = ref.abs() + err >= 65520
        assert ((y == ref.sign() * float("inf")) | (ref.abs() - err < 65520))[over].all()
        y, ref, tol = y[~over], ref[~over], tol[~over]
    bad = (y - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((y - ref).abs() / tol.clamp(min=1e-300)).max():.3g} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 16), (3, 128), (5, 144), (70, 2064), (257, 336)])
def test_quant_rows(M, K, dtype):
    o = ops()
    x = rand(M, K, seed=M + K, dtype=dtype)
    q, s = o.quant_rows(x)
    want, e = R.quant(x)
    assert torch.equal(s.view(torch.uint8).cpu().long() - 127, e)
    assert torch.equal(o.dequant_rows(q, s).double().cpu(), want)
    back = o.dequant_rows(q, s, dtype)
    assert torch.equal(back.cpu(), want.to(dtype))


def test_quant_rows_borders():
    """Largest values at 448 2^e, just past it, halfway between steps, tiny, zero, infinite and NaN."""
    o = ops()
    x = torch.zeros(8, 128)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = 448.0, 17.0, 19.0, 21.0     # steps of 2 from 16 on: ties to even
    x[1, 0], x[1, 1] = 448.5, -1.0
    x[2, :3] = torch.tensor([float("inf"), 1.0, -2.0])
    x[3, :3] = torch.tensor([float("nan"), 3.0, -448.0])
    x[4, :2] = torch.tensor([2.0 ** -140, 2.0 ** -135])
    x[6] = 3.4028234663852886e38
    x[7, 5] = 2.0 ** -9 * 1.5
    x[7, 6] = 448.0
    q, s = o.quant_rows(x.to(DEV))
    want, e = R.quant(x)
    got = o.dequant_rows(q, s).double().cpu()
    assert torch.equal(s.view(torch.uint8).cpu().long() - 127, e)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fin = ~torch.isnan(want)
    # (fp32's largest number, 255.99.. * 2^120, rounds to 256 * 2^120 = 2^128: infinite as an fp32 number)
    assert torch.equal(got[fin], want.float().double()[fin])
    assert torch.isnan(got[2, 0]) and torch.isnan(got[3, 0]) and got[2, 1] == 1.0


def test_quant_rows_strided():
    o = ops()
    x = rand(33, 400, seed=2)[:, 16:16 + 272]
    q, s = o.quant_rows(x)
    want, _ = R.quant(x)
    assert torch.equal(o.dequant_rows(q, s).double().cpu(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("E,K,N,halves", [(1, 16, 16, 1), (2, 144, 336, 1), (3, 272, 352, 2), (1, 2064, 160, 2)])
def test_quant_stack(E, K, N, halves, dtype):
    o = ops()
    w = rand(E, K, N, seed=K, dtype=dtype)
    st = o.F8Stack.from_weights(w, halves=halves, grad=True)
    assert tuple(st.shape) == (E, K, N)
    assert torch.equal(st.dequant().double().cpu(), R.quant_stack(w, halves))
    # the gradient's layout: blocks over all of N
    want = R.quant_stack(w, 1)
    s = st.grad_s.to(torch.float32)[:, :, : -(-N // 128)].repeat_interleave(128, 1)[:, :K].repeat_interleave(128, 2)[:, :, :N]
    assert torch.equal((st.grad_q.float() * s).double().cpu(), want)


SHAPES = [  # E, M, K, N, halves, counts
    (1, 1, 16, 16, 1, "even"),
    (3, 5, 144, 48, 1, "skew"),
    (4, 40, 272, 336, 1, "skew"),
    (2, 61, 2064, 352, 2, "even"),
    (5, 700, 208, 528, 1, "skew"),
    (2, 523, 400, 800, 2, "one"),
    (70, 400, 128, 272, 1, "skew"),
    (300, 700, 64, 32, 1, "skew"),
    (1, 1030, 384, 256, 1, "even"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("E,M,K,N,halves,kind", SHAPES)
def test_grouped_mm(E, M, K, N, halves, kind, dtype):
    o = ops()
    x, w = rand(M, K, seed=M, dtype=dtype), rand(E, K, N, seed=N, dtype=torch.bfloat16)
    q, s = o.quant_rows(x)
    st = o.F8Stack.from_weights(w, halves=halves)
    counts = R.counts_of(M, E, kind)
    y = o.grouped_mm_f8(q, s, st, counts.to(DEV), dtype=dtype)
    a, b = o.dequant_rows(q, s).double(), st.dequant().double()
    e = torch.repeat_interleave(torch.arange(E), counts.long()).to(DEV)
    check(y, *products(a, b, e), dtype)


@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,T,k,K,N", [(4, 30, 2, 272, 336), (6, 400, 3, 144, 528)])
def test_gather_scatter_scale(E, T, k, K, N, scale_dtype):
    o = ops()
    M = T * k
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(0, E, (M,), generator=g)
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids, minlength=E).to(torch.int64)
    x, w = rand(T, K, seed=1), rand(E, K, N, seed=2)
    scale = torch.rand(M, generator=g).to(scale_dtype)
    q, s = o.quant_rows(x)
    st = o.F8Stack.from_weights(w)
    y = o.grouped_mm_f8(q, s, st, counts.to(DEV), M, a_idx=(order // k).int().to(DEV), y_idx=order.int().to(DEV),
                        scale=scale.to(DEV))
    a, b = o.dequant_rows(q, s).double().cpu(), st.dequant().double().cpu()
    rows, err = products(a[order // k], b, ids[order])
    ref, sc = torch.empty_like(rows), scale.double()[:, None]
    ref[order], err[order] = sc * rows, sc * err
    check(y, ref, err + 2.0 ** -23 * ref.abs(), torch.bfloat16)


def test_rows_no_expert_counts_are_zeros():
    o = ops()
    q, s = o.quant_rows(rand(90, 144))
    st = o.F8Stack.from_weights(rand(3, 144, 48, seed=4))
    for counts in ([10, 0, 25], [0, 0, 0], [90, 0, 0], [40, 50, 60]):
        c = torch.tensor(counts, dtype=torch.int32, device=DEV)
        y = o.grouped_mm_f8(q, s, st, c)
        n = min(sum(counts), 90)
        assert torch.equal(y[n:], torch.zeros_like(y[n:]))
        full = o.grouped_mm_f8(q[:n], s[:n], st, c) if n else y[:0]
        assert torch.equal(y[:n], full)


def test_nan_rows_stay_in_their_rows():
    o = ops()
    x = rand(70, 272, spread=False)
    x[3, 200] = float("inf")
    x[66, 1] = float("nan")
    st = o.F8Stack.from_weights(rand(2, 272, 64, seed=4))
    c = torch.tensor([35, 35], device=DEV)
    y = o.grouped_mm_f8(*o.quant_rows(x), st, c)
    bad = torch.isnan(y).any(1)
    assert torch.isnan(y[[3, 66]]).all() and int(bad.sum()) == 2


@pytest.mark.parametrize("form", ["store", "gate_up", "wide"])
@pytest.mark.parametrize("E,M,K,N", [(3, 2600, 400, 4096), (1, 9700, 400, 4096), (3, 5000, 272, 2016), (2, 9000, 272, 2400),
                                     (2, 700, 272, 992), (3, 5000, 1168, 736)])
def test_large_tiles(E, M, K, N, form):
    """Large products (tiles of 128 and 256 rows, whole last rounds and halved ones) are bit for bit the same rows in calls of
    50 rows: every sum is added in the order of k, whatever the tile."""
    o = ops()
    x, w = rand(M, K, seed=M, spread=False), rand(E, K, N, seed=N, spread=False) * K ** -0.5
    q, s = o.quant_rows(x)
    st = o.F8Stack.from_weights(w, halves=1 if form == "store" else 2)
    counts = R.counts_of(M, E, "skew")

    def product(r, c):
        c = torch.tensor(c, dtype=torch.int32, device=DEV)
        if form == "store":
            return (o.grouped_mm_f8(q[r], s[r], st, c),)
        act, act_s = o.gate_up_swiglu_f8(q[r], s[r], st, c, wide=form == "wide")
        return act.view(torch.uint8), act_s.view(torch.uint8)

    whole = product(slice(0, M), counts.tolist())
    r0 = 0
    for e, n in enumerate(counts.tolist()):
        for i in range(r0, r0 + n, 50):
            r = slice(i, min(i + 50, r0 + n))
            part = product(r, [(r.stop - r.start) * (j == e) for j in range(E)])
            assert all(torch.equal(a[r], b) for a, b in zip(whole, part)), (e, i)
        r0 += n


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("E,M,d,h,kind", [(1, 1, 16, 16, "even"), (3, 50, 272, 336, "skew"), (4, 600, 400, 144, "skew"),
                                          (2, 600, 128, 272, "one"), (40, 300, 2064, 64, "skew")])
def test_gate_up(E, M, d, h, kind, wide):
    """act within half an e4m3 step of silu(g) u in 64 bits, plus the step that act's own error may move it by."""
    o = ops()
    x, w = rand(M, d, seed=M, spread=False), rand(E, d, 2 * h, seed=h, spread=False) * d ** -0.5
    q, s = o.quant_rows(x)
    st = o.F8Stack.from_weights(w, halves=2)
    counts = R.counts_of(M, E, kind)
    act, act_s = o.gate_up_swiglu_f8(q, s, st, counts.to(DEV), wide=wide)
    a, b = o.dequant_rows(q, s).double(), st.dequant().double()
    e = torch.repeat_interleave(torch.arange(E), counts.long()).to(DEV)
    gu, mag = products(a, b, e, wide)
    g, u = gu.split(h, 1)
    ref = g * torch.sigmoid(g) * u
    # |silu'| <= 1.1; silu in fp32 with an approximate exp and reciprocal: 8 steps of 2^-24
    err = (1.1 * mag[:, :h] * (u.abs() + mag[:, h:]) + mag[:, h:] * (g * torch.sigmoid(g)).abs()) + 2.0 ** -20 * ref.abs()
    top = torch.zeros(M, -(-h // 128), dtype=torch.float64, device=DEV)
    for j in range(top.shape[1]):
        top[:, j] = ref[:, 128 * j:128 * j + 128].abs().amax(1)
    exps = act_s.view(torch.uint8).double() - 127
    off = torch.stack([err[:, 128 * j:128 * j + 128].amax(1) for j in range(top.shape[1])], 1)
    assert ((top - off <= 448 * torch.exp2(exps)) & (top + off > 224 * torch.exp2(exps)) | (top == 0)).all()
    sc = torch.exp2(exps).repeat_interleave(128, 1)[:, :h]
    val = o.dequant_rows(act, act_s).double()
    half = torch.maximum(2.0 ** -4 * ref.abs(), 2.0 ** -10 * sc)
    assert ((val - ref).abs() <= half + (1 + 2.0 ** -4) * err).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,d,h", [(1, 3, 2, 64, 48), (37, 8, 2, 272, 336), (700, 5, 3, 144, 160)])
def test_moe_experts(T, E, k, d, h, dtype):
    """One call gives the bits of its steps, also for ids that name no expert."""
    o = ops()
    g = torch.Generator().manual_seed(T)
    x = rand(T, d, seed=3, dtype=dtype, spread=False)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).int()
    if T > 1:
        ids[T // 2, 0], ids[T // 3, k - 1] = -1, E
    ids = ids.to(DEV)
    tw = torch.rand(T, k, generator=g).to(DEV)
    gu, dn = o.F8Stack.from_weights(rand(E, d, 2 * h, seed=5, spread=False) * d ** -0.5, halves=2), o.F8Stack.from_weights(
        rand(E, h, d, seed=6, spread=False) * h ** -0.5)
    y, inv, bad = o.moe_experts(x, ids, tw, gu, dn)
    disp = o.dispatch(ids, E, want_xs=False)
    M = T * k
    act, act_s = o.gate_up_swiglu_f8(*o.quant_rows(x), gu, disp.counts, M, a_idx=disp.a_idx, wide=dtype is torch.float16)
    n = int(disp.counts.sum())
    flat = disp.order[:n].long()
    # (positions past the counted rows carry no index: a permutation stands in for them)
    y2 = o.grouped_mm_f8(act, act_s, dn, disp.counts, M, scale=torch.cat([tw.reshape(-1)[flat], tw.new_zeros(M - n)]), dtype=dtype)
    assert torch.equal(y[flat], y2[:n])
    assert torch.equal(inv, disp.inv_pos) and int(bad) == M - n
    out = o.combine(y, T, k, inv_pos=inv)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,M,K,N,kind", [(1, 1, 16, 16, "even"), (4, 300, 272, 400, "skew"), (3, 700, 144, 2064, "one")])
def test_gradient(E, M, K, N, kind, dtype):
    from trenowanie_generatora_obrazkow_amd.moe_triton import grouped_mm
    o = ops()
    a = rand(M, K, seed=M, dtype=dtype, spread=False).requires_grad_(True)
    st = o.F8Stack.from_weights(rand(E, K, N, seed=N, spread=False) * K ** -0.5, grad=True)
    counts = R.counts_of(M, E, kind).to(DEV)
    dy = rand(M, N, seed=9, dtype=dtype, spread=False)
    y = grouped_mm(a, st, counts)
    y.backward(dy)
    assert torch.equal(y.detach(), o.grouped_mm_f8(*o.quant_rows(a.detach()), st, counts, dtype=dtype))
    d, _ = R.quant(dy)
    e = torch.repeat_interleave(torch.arange(E), counts.long().cpu())
    check(a.grad, *products(d, st.dequant().double().cpu().transpose(1, 2).contiguous(), e), dtype)


def test_gradient_against_differences():
    """Along a direction, the gradient of <y, dy> is what differences of the quantised product give, to the steps of both
    quantisations: |<da, v> - diff| is a sum over elements of independent roundings, each at most 2^-4 of its factor."""
    from trenowanie_generatora_obrazkow_amd.moe_triton import grouped_mm
    o = ops()
    M, K, N = 64, 256, 256
    a = rand(M, K, seed=1, dtype=torch.float32, spread=False).requires_grad_(True)
    st = o.F8Stack.from_weights(rand(1, K, N, seed=2, spread=False) * K ** -0.5, grad=True)
    counts = torch.tensor([M], device=DEV)
    dy, v = rand(M, N, seed=3, dtype=torch.float32, spread=False), rand(M, K, seed=4, dtype=torch.float32, spread=False)
    grouped_mm(a, st, counts).backward(dy)
    y = lambda t: (grouped_mm(t, st, counts).double() * dy.double()).sum()
    with torch.no_grad():
        diff = float(y(a + v) - y(a - v)) / 2
    w = st.dequant().double()[0]
    full = (dy.double() @ w.t())
    got = float((a.grad.double() * v.double()).sum())
    # rms of the roundings: 2^-4 / sqrt(3) of each factor at most; six of them
    noise = 2.0 ** -4 * (float((full * v.double()).norm()) + float((full * (a.detach().double().abs() + v.double().abs())).norm())
                         + float((dy.double().abs() * (v.double() @ w).abs()).norm()))
    assert abs(got - diff) < 6 / 3 ** 0.5 * noise


def test_tail_gradient_is_zero():
    from trenowanie_generatora_obrazkow_amd.moe_triton import grouped_mm
    o = ops()
    a = rand(50, 64).requires_grad_(True)
    st = o.F8Stack.from_weights(rand(2, 64, 32, seed=4), grad=True)
    y = grouped_mm(a, st, torch.tensor([10, 7], device=DEV))
    y.sum().backward()
    assert torch.equal(a.grad[17:], torch.zeros_like(a.grad[17:])) and torch.equal(y[17:], torch.zeros_like(y[17:]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_one_call(dtype):
    """The product with its rows quantised on the way has the bits of the two calls."""
    o = ops()
    x = rand(60, 400, seed=2, dtype=dtype)[:, 16:16 + 272]
    st = o.F8Stack.from_weights(rand(3, 272, 96, seed=4), halves=2)
    c = torch.tensor([20, 0, 25], device=DEV)
    a = torch.randint(0, 60, (45,), generator=torch.Generator().manual_seed(0)).int().to(DEV)
    y_idx, sc = torch.randperm(45).int().to(DEV), torch.rand(45, device=DEV)
    q, s = o.quant_rows(x)
    assert torch.equal(o.quant_mm_f8(x, st, c, a_idx=a, y_idx=y_idx, scale=sc), o.grouped_mm_f8(q, s, st, c, 45, a, y_idx, sc, dtype))
    assert torch.equal(o.quant_mm_f8(x, st, c, dtype=torch.float32), o.grouped_mm_f8(q, s, st, c, dtype=torch.float32))


def test_empty():
    o = ops()
    st = o.F8Stack.from_weights(rand(2, 64, 32, seed=4))
    q, s = o.quant_rows(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16))
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert o.grouped_mm_f8(q, s, st, zero).shape == (0, 32)
    assert o.quant_mm_f8(torch.empty(0, 64, device=DEV), st, zero).shape == (0, 32)


def test_graph_and_stream():
    """Captured once on a side stream and replayed with other inputs, eager work between the replays."""
    o = ops()
    T, E, k, d, h = 40, 4, 2, 144, 160
    gu, dn = (o.F8Stack.from_weights(rand(E, d, 2 * h, seed=5, spread=False) * d ** -0.5, halves=2),
              o.F8Stack.from_weights(rand(E, h, d, seed=6, spread=False) * h ** -0.5))
    x = rand(T, d, seed=1, spread=False)
    ids = torch.stack([torch.randperm(E)[:k] for _ in range(T)]).int().to(DEV)
    tw = torch.rand(T, k, device=DEV)
    run = lambda: o.combine(*(lambda y, inv, _: (y, T, k))(*o.moe_experts(x, ids, tw, gu, dn)))
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for i in range(4):
        x.copy_(rand(T, d, seed=10 + i, spread=False))
        ids.copy_(ids.roll(1, 0))
        want = run().clone()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
