"""Calls that the block's functions and gradient clipping have to answer or refuse and that no size or mask brings up: a single
row whose elements are strided, clipping outputs given twice or laid over another gradient, parameters for another number of
samples than the input holds."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_one_row_with_strided_elements():
    from trenowanie_generatora_obrazkow_amd import MoEResidual, norm_modulate, norm_residual
    g = torch.Generator().manual_seed(61)
    x = torch.randn(1, 256, generator=g).cuda()[:, ::2]
    y = torch.randn(1, 256, generator=g).cuda()[:, 1::2]
    assert torch.equal(norm_modulate(x), norm_modulate(x.contiguous()))
    assert torch.equal(norm_residual(x, y), norm_residual(x.contiguous(), y.contiguous()))
    m = MoEResidual(128, 192, 16, 2, device="cuda")
    for grad in (True, False):
        with torch.set_grad_enabled(grad):
            assert torch.equal(m(x), m(x.contiguous()))


def test_outputs_beside_a_list_that_has_its_own():
    from trenowanie_generatora_obrazkow_amd import ops
    a, o = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    gl = ops.GradList([a])
    with pytest.raises(ValueError, match="GradList"):
        ops.grad_clip(gl, ops.grad_sq_norm(gl), 1.0, out=[o])
    assert (a == 1).all() and (o == 0).all()
    gl = ops.GradList([a], [o])
    ops.grad_clip(gl, ops.grad_sq_norm(gl), 1.0)
    # norm 8, factor 1 / (8 + 1e-6): 1.25e-7 below 1 / 8, and two fp32 roundings of 6e-8
    assert (a == 1).all() and (o - 0.125).abs().max() <= 0.125 * 2.5e-7


def test_an_output_laid_over_another_gradient():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    a, b, c = (torch.full((64,), v, device="cuda") for v in (1.0, 2.0, 3.0))
    for out in ([b, c], [c, a], [b, a]):
        with pytest.raises(ValueError, match="another gradient"):
            clip_grad_norm([a, b], 1.0, out=out)
    assert (a == 1).all() and (b == 2).all() and (c == 3).all()
    e = torch.empty(0, device="cuda")  # (no element, no overlap)
    clip_grad_norm([a, e, e], 1e9, out=[c, e, e])
    assert (c == 1).all()
    clip_grad_norm([a, b], 1.0, out=[a, c])  # its own is in place
    assert (a < 1).all() and (b == 2).all() and (c < 2).all()


def test_parameters_of_other_samples():
    from trenowanie_generatora_obrazkow_amd import MoEResidual, norm_modulate, norm_residual
    r = lambda *s: torch.randn(*s, device="cuda")
    x, m = r(2, 6, 128), MoEResidual(128, 192, 16, 2, device="cuda")
    for n in (3, 4, 6):  # they divide the 12 rows, but not along the samples
        for f in (lambda: norm_modulate(x, None, r(n, 128)), lambda: norm_modulate(x, None, None, r(n, 128)),
                  lambda: norm_residual(x, x, r(n, 128)), lambda: m(x, r(n, 128)), lambda: m(x, None, None, r(n, 128))):
            with pytest.raises(ValueError, match="leading dimensions"):
                f()
    for n in (1, 2, 12):  # one set, a set per sample, a set per row
        s = r(n, 128)
        want = norm_modulate(x.view(12, 128), None, s.repeat_interleave(12 // n, 0).contiguous()).view(2, 6, 128)
        assert torch.equal(norm_modulate(x, None, s), want)
    frames = r(2, 3, 2, 128)
    for n in (1, 2, 6, 12):
        assert norm_residual(frames, frames, r(n, 128)).shape == frames.shape
    with pytest.raises(ValueError, match="leading dimensions"):
        norm_residual(frames, frames, r(3, 128))
