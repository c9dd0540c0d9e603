"""The bound of a clipping call is a 64-bit number: the factor max_norm / (norm + 1e-6) is formed from it unrounded and rounded
once to fp32."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_factor_is_rounded_once():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    one = torch.ones(4, device="cuda")  # norm 2, exactly
    out = torch.empty(4, device="cuda")
    for i in range(1, 60):
        bound = 2 * i / 61
        clip_grad_norm([one], bound, out=[out])
        want = torch.tensor(bound / (2 + 1e-6), dtype=torch.float64).float()
        assert (out.cpu() == want).all(), (bound, float(out[0]), float(want))


def test_bounds_outside_fp32():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    a = torch.full((4,), 1e30, device="cuda")
    assert clip_grad_norm([a], 1e39) and (a == 1e30).all()
    a[0] = math.inf  # an infinite norm: zeros, and NaN in the infinite place
    clip_grad_norm([a], 1e39)
    assert torch.isnan(a[0]) and not a[1:].any()
    # no bound at all: the factor is one, whatever the norm
    a = torch.tensor([1.0, math.inf], device="cuda")
    assert clip_grad_norm([a], math.inf) == math.inf and a[0] == 1 and a[1] == math.inf
