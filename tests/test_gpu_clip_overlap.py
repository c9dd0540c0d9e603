"""Clipping with outputs beside, on and over the gradients: what overlaps is refused and leaves every tensor as it was, what only
touches is answered."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


def test_overlapping_outputs():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    flat = torch.arange(1, 4001, dtype=FP, device="cuda")
    keep = flat.clone()
    half = flat.view(BF)  # (two 16-bit elements in each of flat's)
    other = torch.zeros(100, device="cuda")
    for grads, out in (([half[:1000]], [flat[:1000]]),                             # the same start, another type
                       ([flat[:100]], [flat[50:150]]), ([flat[50:150]], [flat[:100]]),
                       ([flat[:100], flat[200:300]], [other, flat[99:199]]),       # the last element of another gradient
                       ([flat[:100], flat[200:300]], [flat[400:500], flat[499:599]]),
                       ([flat[:101], flat[100:200]], None)):
        with pytest.raises(ValueError, match="another gradient or output"):
            clip_grad_norm(grads, 1e-3, out=out)
        assert torch.equal(flat, keep)


def test_neighbours_and_shared_gradients():
    """Views that touch, in any order; a gradient that two entries read (it counts twice)."""
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    flat = torch.ones(4000, device="cuda")
    grads = [flat[1000:2000], flat[:1000], flat[2000:2001]]
    out = [flat[3000:4000], torch.empty(1000, device="cuda"), flat[2001:2002]]
    assert abs(float(clip_grad_norm(grads, 1.0, out=out)) - 2001 ** 0.5) < 1e-4
    want = 1 / (2001 ** 0.5 + 1e-6)
    assert all(((o - want).abs() < 1e-8).all() for o in out)
    assert (flat[:2001] == 1).all() and (flat[2002:3000] == 1).all()
    a, o = torch.ones(50, device="cuda"), [torch.empty(50, device="cuda") for _ in range(2)]
    assert abs(float(clip_grad_norm([a, a], 5.0, out=o)) - 10) < 1e-5
    assert all(((t - 0.5).abs() < 1e-6).all() for t in o) and (a == 1).all()
