"""The gated residual without its norm is linear in the slots' sum: the gradient dy = dout w gate does not depend on it, also
where it holds infinities or NaN."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [1, 2])
def test_gradient_is_that_of_a_linear_map(k):
    from trenowanie_generatora_obrazkow_amd import ops
    g = torch.Generator().manual_seed(7)
    T, d = 40, 136
    y = torch.randn(T * k, d, generator=g)
    y[3, 5], y[9, 7], y[20] = math.inf, -math.inf, math.nan
    dout, gate = torch.randn(T, d, generator=g), torch.randn(4, d, generator=g)
    for gt, per in ((None, 1.0), (gate, gate.repeat_interleave(T // 4, 0))):
        dy, _, _ = ops.norm_residual_bwd(dout.cuda(), y.cuda(), gate=None if gt is None else gt.cuda(), norm=False, k=k)
        assert torch.equal(dy.cpu(), dout * per)  # (one fp32 product)
