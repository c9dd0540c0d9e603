"""The 8-bit, checkpoint and few-token operators where sizes end: arrays past 2^31 elements, layers of no tokens, rows that
nothing routes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from trenowanie_generatora_obrazkow_amd import ops
    return ops


def rand(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def long_rows(M, K, seed):
    """M rows that repeat 1000 random ones, built in pieces (M K past 2^31)."""
    return rand(1000, K, seed=seed).repeat(-(-M // 1000), 1)[:M]


def test_experts_past_2_gib():
    """T k rows of 2048 columns are more than 2^31 values; the sampled tokens' rows are those of a call of their own."""
    o = ops()
    T, E, k, d, h = 70000, 16, 16, 2048, 16
    x = long_rows(T, d, 1)
    ids = torch.rand(T, E, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).argsort(1).int()
    tw = torch.rand(T, k, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    st = (o.F8Stack.from_weights(rand(E, d, 2 * h, seed=4) * d ** -0.5, halves=2), o.F8Stack.from_weights(rand(E, h, d, seed=5) * h ** -0.5))
    y, inv, bad = o.moe_experts(x, ids, tw, *st)
    assert int(bad) == 0 and y.shape == (T * k, d)
    for t in (0, 33333, 65530, T - 40):
        r = slice(t, t + 40)
        part, _, _ = o.moe_experts(x[r], ids[r].contiguous(), tw[r].contiguous(), *st)
        assert torch.equal(y.view(T, k, d)[r].reshape(-1, d), part), t


def test_rows_past_2_gib():
    """Quantisation, the product of sorted rows, and the way back."""
    o = ops()
    M, K, N = 300000, 8192, 32
    x = long_rows(M, K, 6)
    q, s = o.quant_rows(x)
    st = o.F8Stack.from_weights(rand(1, K, N, seed=7) * K ** -0.5)
    c = torch.tensor([M], device=DEV)
    y = o.grouped_mm_f8(q, s, st, c)
    r = slice(M - 300, M)
    q2, s2 = o.quant_rows(x[r].contiguous())
    assert torch.equal(q[r].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[r].view(torch.uint8), s2.view(torch.uint8))
    assert torch.equal(y[r], o.grouped_mm_f8(q2, s2, st, torch.tensor([300], device=DEV)))
    assert torch.equal(o.dequant_rows(q, s, dtype=torch.bfloat16)[r], o.dequant_rows(q2, s2, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="2 GiB"):
        o.grouped_mm_f8(q, s, st, c, a_idx=torch.arange(M, device=DEV, dtype=torch.int32))


def test_checkpoint_past_2_gib():
    o = ops()
    M, h = 300000, 4096
    gu, dh = long_rows(M, 2 * h, 8), long_rows(M, h, 9)
    act, kept = o.swiglu_pack(gu)
    dgu, a, dw = o.swiglu_pack_bwd(dh, kept)
    r = slice(M - 100, M)
    act2, kept2 = o.swiglu_pack(gu[r])
    dgu2, a2, dw2 = o.swiglu_pack_bwd(dh[r], kept2)
    for u, v in ((act[r], act2), (kept.q[r].view(torch.uint8), kept2.q.view(torch.uint8)), (dgu[r], dgu2), (a[r], a2), (dw[r], dw2)):
        assert torch.equal(u, v)


@pytest.mark.parametrize("kw", [dict(checkpoint="fp8"), dict(few_tokens=16)])
def test_layers_of_no_tokens(kw):
    from trenowanie_generatora_obrazkow_amd import MoESwiGLU
    m = MoESwiGLU(64, 96, 4, top_k=2, **kw).to(DEV, torch.bfloat16)
    x = torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = m(x)
    y.backward(torch.zeros_like(y))
    assert y.shape == (0, 64) and x.grad.shape == (0, 64) and not m.w_gu.grad.any() and not m.w_d.grad.any()
    with torch.no_grad():
        assert m(x).shape == (0, 64)


def test_product_of_no_rows_with_a_gradient():
    from trenowanie_generatora_obrazkow_amd.moe_triton import grouped_mm
    o = ops()
    st = o.F8Stack.from_weights(rand(3, 64, 32), grad=True)
    a = torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = grouped_mm(a, st, torch.zeros(3, device=DEV, dtype=torch.int64))
    y.backward(torch.zeros_like(y))
    assert y.shape == (0, 32) and a.grad.shape == (0, 64)


def test_strided_and_shared_gradients():
    """a as a view of wider rows, dy as an expanded row: the same bits as of contiguous copies."""
    from trenowanie_generatora_obrazkow_amd.moe_triton import grouped_mm
    o = ops()
    st = o.F8Stack.from_weights(rand(2, 64, 48, seed=1), grad=True)
    wide = rand(30, 160, seed=2).requires_grad_(True)
    c = torch.tensor([11, 19], device=DEV)
    dy = rand(1, 48, seed=3).expand(30, 48)
    y = grouped_mm(wide[:, 32:96], st, c)
    y.backward(dy)
    a = wide.detach()[:, 32:96].contiguous().requires_grad_(True)
    y2 = grouped_mm(a, st, c)
    y2.backward(dy.contiguous())
    assert torch.equal(y, y2) and torch.equal(wide.grad[:, 32:96], a.grad)
    assert not wide.grad[:, :32].any() and not wide.grad[:, 96:].any()


@pytest.mark.parametrize("form", ["store", "gate_up", "wide"])
@pytest.mark.parametrize("E,M,K,N", [(8, 100, 256, 288), (40, 90, 2048, 96), (1, 1, 128, 32), (3, 70, 640, 544)])
def test_few_rows_per_expert(E, M, K, N, form):
    """Few rows per expert (weights copied past the caches), one expert with more than a tile's: the bits of a product of twelve
    times the rows of each."""
    o = ops()
    st = o.F8Stack.from_weights(rand(E, K, N, seed=N) * K ** -0.5, halves=1 if form == "store" else 2)
    g = torch.Generator().manual_seed(M)
    counts = torch.bincount(torch.randint(0, E, (M // 2,), generator=g), minlength=E)
    counts[E // 2] += M - M // 2
    x = rand(M, K, seed=M)

    def product(x, c):
        q, s = o.quant_rows(x)
        if form == "store":
            return (o.grouped_mm_f8(q, s, st, c.to(DEV)),)
        act, act_s = o.gate_up_swiglu_f8(q, s, st, c.to(DEV), wide=form == "wide")
        return act.view(torch.uint8), act_s.view(torch.uint8)

    few = product(x, counts)
    many = product(torch.cat([t.repeat(12, 1) for t in x.split(counts.tolist())]), counts * 12)
    r0 = 0
    for n in counts.tolist():
        for a, b in zip(few, many):
            assert torch.equal(a[r0:r0 + n], b[12 * r0:12 * r0 + n])
        r0 += n
