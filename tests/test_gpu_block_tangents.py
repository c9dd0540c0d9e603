"""Forward-mode differentiation of the routed layer and the residual block is refused like that of their norms, also where no
input requires a gradient: a tangent is never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def _inputs():
    g = torch.Generator().manual_seed(5)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).bfloat16().cuda()
    return [r(50, 64), r(8, 64, std=0.2), r(8, 64, 128, std=0.1), r(8, 64, 64, std=0.1)]


@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("name", ["moe_swiglu", "moe_residual", "gated"])
def test_tangents_are_refused(name, which):
    from trenowanie_generatora_obrazkow_amd import Gate, moe_residual, moe_swiglu
    f = dict(moe_swiglu=moe_swiglu, moe_residual=moe_residual, gated=lambda *a: moe_swiglu(*a, gate=Gate("sigmoid")))[name]
    lv = _inputs()
    want = f(*lv, 2)
    with fwd.dual_level():
        assert all(torch.equal(a, b) for a, b in zip(f(*lv, 2), want))  # (without a tangent all is as ever)
        lv[which] = fwd.make_dual(lv[which], torch.ones_like(lv[which]))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            f(*lv, 2)
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            f(*lv, 2)


def test_tangents_of_norm_parameters():
    from trenowanie_generatora_obrazkow_amd import MoEResidual, norm_modulate
    m = MoEResidual(64, 64, 8, 2, device="cuda")
    x, sc = torch.randn(2, 6, 64, device="cuda"), torch.randn(2, 64, device="cuda")
    with fwd.dual_level():
        d = fwd.make_dual(sc, torch.ones_like(sc))
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            m(x, d)
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            norm_modulate(x, None, d)
