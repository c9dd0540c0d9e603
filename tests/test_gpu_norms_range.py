"""The norms' backward over fp32's range: rows from 1e-10 to 1e17 and a tiny eps with rows of zeros, where the reciprocal
root of the mean square lies far from one and its cube outside fp32.

Tolerances: those of a row's sums, row = (d / 64 + 40) 2^-24 relative to the sum of the absolute terms.  dv = r (g - n mean(g n))
takes r, n = v r and the mean to that accuracy each: at most four of them in a term.  Then one rounding to the output's type."""
import pytest
import torch

from tests import block_ref as R

pytestmark = pytest.mark.gpu
D = 320
TOL = (D / 64 + 40) * R.EPS24


def _close(name, got, ref, mag):
    got = got.cpu().double()
    bound = (4 * TOL + R.half_step(torch.float32)) * mag + R.tiny(torch.float32)
    assert torch.isfinite(got).all(), name
    assert ((got - ref).abs() <= bound).all(), (name, float(((got - ref).abs() / bound).max()))


def _ref(v, g, eps):
    """(dv, its terms' absolute size) of u -> sum(g n) in float64."""
    r = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    n = v * r
    return r * (g - n * (g * n).mean(1, keepdim=True)), r * (g.abs() + n.abs() * (g * n).abs().mean(1, keepdim=True))


def _rows(sizes, seed):
    g = torch.Generator().manual_seed(seed)
    size = torch.tensor(sizes).repeat_interleave(5).unsqueeze(1)
    v = (torch.randn(len(size), D, generator=g) + 0.5) * size
    u, w = torch.randn(len(size), D, generator=g) * 0.1, torch.randn(D, generator=g) * 0.1 + 1
    # (an upstream gradient along the row: the projection is as large as the rest)
    u += 0.2 * torch.nan_to_num(v / size)
    return v, u, w


@pytest.mark.parametrize("sizes,eps", [((1e-10, 1.0, 1e10, 1e15, 1e17), 1e-6), ((0.0, 1e-16, 1e-13, 1.0), 1e-30)],
                         ids=["large", "tiny_eps"])
def test_backward_of_rows_of_any_size(sizes, eps):
    from trenowanie_generatora_obrazkow_amd import ops
    v, u, w = _rows(sizes, 3)
    eps32 = float(torch.tensor(eps, dtype=torch.float32))
    ref, mag = _ref(v.double(), (u * w).double(), eps32)
    dx, dw, _, _ = ops.norm_modulate_bwd(u.cuda(), v.cuda(), weight=w.cuda(), eps=eps)
    _close("norm_modulate", dx, ref, mag)
    dy, _, dw2 = ops.norm_residual_bwd(u.cuda(), v.cuda(), weight=w.cuda(), eps=eps)
    _close("norm_residual", dy, ref, mag)
    assert torch.isfinite(dw).all() and torch.isfinite(dw2).all()
    # every row by itself (samples of one row are walked by another form of the kernel)
    one = torch.ones(len(v), D, device="cuda")
    dx, _, _, _ = ops.norm_modulate_bwd(u.cuda(), v.cuda(), weight=w.cuda(), scale=one - 1, eps=eps)
    _close("norm_modulate, a sample a row", dx, ref, mag)
    dy, _, _ = ops.norm_residual_bwd(u.cuda(), v.cuda(), weight=w.cuda(), gate=one, eps=eps)
    _close("norm_residual, a sample a row", dy, ref, mag)
