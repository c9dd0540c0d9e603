"""8-bit float experts and the form for a few tokens where a program has them: fuse_moe, MoESwiGLU, moe_triton.grouped_mm; and a
run of the operators together, as a serving program uses them."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Expert(nn.Module):
    def __init__(self, d, h, act=nn.SiLU, **f):
        super().__init__()
        self.gate_proj, self.up_proj = nn.Linear(d, h, bias=False, **f), nn.Linear(d, h, bias=False, **f)
        self.down_proj = nn.Linear(h, d, bias=False, **f)
        self.act_fn = act()


class _Block(nn.Module):
    def __init__(self, d, h, E, act=nn.SiLU, **f):
        super().__init__()
        self.experts = nn.ModuleList([_Expert(d, h, act, **f) for _ in range(E)])

    def moe_infer(self, x, ids, w):
        raise NotImplementedError


def model(d, h, E, dtype=torch.bfloat16, act=nn.SiLU, seed=0):
    torch.manual_seed(seed)
    m = nn.Sequential(_Block(d, h, E, act, device=DEV, dtype=dtype))
    g = torch.Generator(device=DEV).manual_seed(seed)
    for p in m.requires_grad_(False).parameters():
        p.data.normal_(0.0, p.shape[1] ** -0.5, generator=g)
    return m


def inputs(T, E, k, d, dtype=torch.bfloat16, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, d, generator=g, device=DEV).to(dtype)
    w, ids = torch.randn(T, E, generator=g, device=DEV).softmax(-1).topk(k, -1)
    return x, ids, w / w.sum(-1, keepdim=True)


def exact(m, x, ids, w, act=torch.nn.functional.silu):
    """The unquantised block in 64 bits."""
    out = torch.zeros_like(x, dtype=torch.float64)
    for e, ex in enumerate(m[0].experts):
        t, s = (ids == e).nonzero(as_tuple=True)
        X = x[t].double()
        a = act(X @ ex.gate_proj.weight.double().t()) * (X @ ex.up_proj.weight.double().t())
        out.index_add_(0, t, w[t, s, None].double() * (a @ ex.down_proj.weight.double().t()))
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,d,h", [(1, 4, 2, 64, 48), (16, 6, 2, 72, 100), (17, 6, 2, 72, 100), (300, 8, 3, 256, 192)])
def test_fuse_moe_fp8(T, E, k, d, h, dtype):
    """Every element of x, the weights and act is off by at most r = 2^-4 of itself, with independent signs, so that products'
    errors add in quadrature.  g and u are each off by sqrt(2) r of their rms (x and a weight); for normal g the error of silu is
    E[silu'^2] / E[silu^2] = 1.07 times g's, squared; act's own rounding and Wd's add r^2 each: together
    (2 * 1.07 + 2 + 1 + 1) r^2, and the output's 2-norm error stays under sqrt(6.14) 2^-4 = 0.155 were every rounding the largest
    (0.065 expected; one token of 64 columns spreads by a half).  Widths off 16 are padded."""
    from trenowanie_generatora_obrazkow_amd.hf_compat import fuse_moe, invalid_expert_ids
    m = model(d, h, E, dtype)
    x, ids, w = inputs(T, E, k, d, dtype)
    want = exact(m, x, ids, w)
    assert fuse_moe(m, quant="fp8") == 1
    b = m[0]
    assert b._wgu.dtype == torch.uint8 and b._wgu.numel() <= E * (-(-d // 16) * 16) * 2 * (-(-h // 16) * 16)
    y = b.moe_infer(x, ids, w)
    assert y.dtype == dtype and y.shape == x.shape
    assert float((y.double() - want).norm() / want.norm()) < 0.155
    assert invalid_expert_ids(m) == 0
    m.to(torch.float16 if dtype == torch.bfloat16 else torch.bfloat16)  # a cast leaves the 8-bit weights as they are
    assert torch.equal(y, b.moe_infer(x, ids, w))
    ids = ids.clone()
    ids[0, 0] = E + 3
    y2 = b.moe_infer(x, ids, w)
    assert torch.isfinite(y2).all() and invalid_expert_ids(m) == 1


def test_few_tokens_and_many_agree():
    """A call of 16 tokens through the two kernels and the same rows inside a larger call: the same quantised operands, so they
    differ by the slots' rounding (2^-8 of two slots), the 8-bit products' and act's borders (2e-3)."""
    from trenowanie_generatora_obrazkow_amd.hf_compat import fuse_moe
    m = model(256, 192, 8)
    x, ids, w = inputs(40, 8, 2, 256)
    fuse_moe(m, quant="fp8")
    many = m[0].moe_infer(x, ids, w)[:16].double()
    few = m[0].moe_infer(x[:16], ids[:16], w[:16]).double()
    assert float((many - few).norm() / few.norm()) < 2.0 ** -8 + 2e-3


def test_fp8_with_another_activation():
    from trenowanie_generatora_obrazkow_amd.hf_compat import fuse_moe
    m = model(64, 48, 4, act=nn.GELU)
    x, ids, w = inputs(30, 4, 2, 64)
    want = exact(m, x, ids, w, act=torch.nn.functional.gelu)
    fuse_moe(m, quant="fp8")
    y = m[0].moe_infer(x, ids, w)
    assert float((y.double() - want).norm() / want.norm()) < 0.155


@pytest.mark.parametrize("quant", ["", "int8"])
def test_fuse_moe_few_tokens(quant):
    """Off unless asked for; then within the other form's roundings (six of 2^-8 / sqrt(3))."""
    from trenowanie_generatora_obrazkow_amd.hf_compat import fuse_moe, invalid_expert_ids
    a, b = model(128, 96, 6), model(128, 96, 6)
    x, ids, w = inputs(5, 6, 2, 128)
    fuse_moe(a, quant=quant)
    fuse_moe(b, quant=quant, few_tokens=8)
    assert a[0]._few_tokens == 0
    ya, yb = a[0].moe_infer(x, ids, w).double(), b[0].moe_infer(x, ids, w).double()
    assert float((ya - yb).norm() / ya.norm()) < 6 * 2.0 ** -8 / 3 ** 0.5
    ids[2, 1] = -1
    b[0].moe_infer(x, ids, w)
    assert invalid_expert_ids(b) == 1
    x9, ids9, w9 = inputs(9, 6, 2, 128)
    assert torch.equal(a[0].moe_infer(x9, ids9, w9), b[0].moe_infer(x9, ids9, w9))


def test_layer_few_tokens():
    from trenowanie_generatora_obrazkow_amd import Gate, MoESwiGLU
    for gate in (None, Gate(score="sigmoid", n_group=2, topk_group=1, scaling=2.5)):
        torch.manual_seed(0)
        m = MoESwiGLU(128, 96, 8, 2, device=DEV, few_tokens=4, gate=gate, balance=gate is not None)
        x = torch.randn(2, 2, 128, device=DEV, dtype=torch.bfloat16)
        with torch.no_grad():
            y = m(x).double()
            ids = m.last_topk_ids
            m.few_tokens = 0
            z = m(x).double()
            assert torch.equal(ids, m.last_topk_ids) and float((y - z).norm() / z.norm()) < 6 * 2.0 ** -8 / 3 ** 0.5
            big = torch.randn(5, 128, device=DEV, dtype=torch.bfloat16)
            z = m(big)
            m.few_tokens = 4
            assert torch.equal(z, m(big))
        m.few_tokens = 4
        x.requires_grad_(True)
        m(x).sum().backward()  # with a gradient to record the ordinary form runs
        assert x.grad is not None


def test_serving_run():
    """Prompts of several lengths, then tokens one by one, through one stack of 8-bit experts with the layer's own routing; the
    token steps captured in a graph."""
    from trenowanie_generatora_obrazkow_amd import F8Stack, ops
    g = torch.Generator(device=DEV).manual_seed(0)
    E, k, d, h = 12, 3, 256, 208
    wr = (torch.randn(E, d, generator=g, device=DEV) * d ** -0.5).bfloat16()
    gu = F8Stack.from_weights((torch.randn(E, d, 2 * h, generator=g, device=DEV) * d ** -0.5).bfloat16(), halves=2)
    dn = F8Stack.from_weights((torch.randn(E, h, d, generator=g, device=DEV) * h ** -0.5).bfloat16())

    def step(x):
        _, ids, w = ops.route_topk(x, wr, k)
        if x.shape[0] <= ops.FEW_TOKENS:
            return x + ops.few_experts(x, ids, w, gu, dn)
        y, inv, _ = ops.moe_experts(x, ids, w, gu, dn)
        return x + ops.combine(y, x.shape[0], k, inv_pos=inv)

    for T in (1, 16, 17, 250, 3):
        x = torch.randn(T, d, generator=g, device=DEV).bfloat16()
        y = step(step(x))
        rows = [step(step(x[i:i + 1])) for i in range(min(T, 4))]
        for i, r in enumerate(rows):
            assert float((r.double() - y[i:i + 1].double()).norm() / r.double().norm()) < 0.02
    x = torch.randn(2, d, generator=g, device=DEV).bfloat16()
    step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(step(x))
    for i in range(4):
        x.copy_(torch.randn(2, d, generator=g, device=DEV).bfloat16())
        want = step(step(x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
