"""What autograd lets a program do with the routed layer's and the residual block's results: change the returned routing weights
in place before the backward."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _leaves(seed, T=150, d=64, E=8, h=64):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).bfloat16().cuda().requires_grad_(True)
    return r(T, d), r(E, d, std=0.2), r(E, d, 2 * h, std=0.1), r(E, h, d, std=0.1)


@pytest.mark.parametrize("block", [False, True])
def test_weights_changed_in_place(block):
    from trenowanie_generatora_obrazkow_amd import moe_residual, moe_swiglu
    lv = _leaves(5)
    f = moe_residual if block else moe_swiglu
    dout = torch.randn(lv[0].shape, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    out, _, _ = f(*lv, 2)
    want = torch.autograd.grad(out, lv, dout)
    out, _, tw = f(*lv, 2)
    tw.mul_(0.5)
    got = torch.autograd.grad(out, lv, dout)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
