"""The residual block on a few tokens: few_tokens of its layer reaches the two kernels, between the norms as they are."""
import pytest
import torch

from test_gpu_few import rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


def counted(monkeypatch):
    from trenowanie_generatora_obrazkow_amd import ops
    calls = []
    for name in ("few_forward", "few_experts"):
        f = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, f=f, name=name, **k: (calls.append(name), f(*a, **k))[1])
    return ops, calls


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gated", [False, True])
def test_block_on_few_tokens(monkeypatch, dtype, gated):
    from trenowanie_generatora_obrazkow_amd import Gate, MoEResidual
    ops, calls = counted(monkeypatch)
    torch.manual_seed(0)
    d = 64
    mlp = dict(gate=Gate("sigmoid"), balance=True) if gated else {}
    few = MoEResidual(d, 48, 6, 2, post_norm=True, alpha=0.5, device=DEV, few_tokens=8, **mlp)
    torch.manual_seed(0)
    plain = MoEResidual(d, 48, 6, 2, post_norm=True, alpha=0.5, device=DEV, **mlp)
    scale, shift, gate = (rand(2, d, seed=s) for s in (1, 2, 3))
    x = rand(2, 4, d, seed=4, dtype=dtype)
    with torch.no_grad():
        y = few(x, scale, shift, gate)
        assert calls == ["few_experts" if gated else "few_forward"]
        # the same steps one by one
        m, rows = few.mlp, x.view(8, d)
        h = ops.norm_modulate(rows, few.norm_weight, scale, shift, None, few.eps, torch.bfloat16)
        want = ops.norm_residual(m(h), rows, gate, few.post_weight, True, None, few.eps, 0.5)
        assert torch.equal(y.view(8, d), want)
        calls.clear()
        z = plain(x, scale, shift, gate)
        assert not calls and torch.equal(few.mlp.last_topk_ids, plain.mlp.last_topk_ids)
        # x and gate * n in its type, each a rounding apart by what the layer's own roundings (six of bf16) leave in n
        assert float((y.double() - z.double()).norm() / z.double().norm()) < 6 * 2.0 ** -8
        more = rand(2, 5, d, seed=5, dtype=dtype)  # ten tokens
        assert torch.equal(few(more, scale, shift, gate), plain(more, scale, shift, gate)) and not calls
    few(x, scale, shift, gate)  # with a gradient to record
    assert not calls


def test_packed_rows_with_padding(monkeypatch):
    from trenowanie_generatora_obrazkow_amd import MoEResidual
    _, calls = counted(monkeypatch)
    m = MoEResidual(64, 48, 6, 2, device=DEV, few_tokens=16)
    x = rand(9, 64)
    starts = torch.tensor([1, 4, 7], dtype=torch.int32, device=DEV)
    gate = rand(2, 64, seed=2)
    with torch.no_grad():
        y = m(x, gate=gate, starts=starts)
    assert calls and torch.equal(y[[0, 7, 8]], x[[0, 7, 8]])  # rows outside the samples pass through


def test_refusal():
    from trenowanie_generatora_obrazkow_amd import MoEResidual
    m = MoEResidual(64, 48, 6, 2, device=DEV, few_tokens=17)
    with pytest.raises(ValueError, match="few_tokens"):
        m(rand(1, 4, 64))
