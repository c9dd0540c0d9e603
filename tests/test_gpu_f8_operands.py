"""grouped_mm over an F8Stack on operands as programs have them: rows that lie in any stride, output gradients that begin anywhere."""
import pytest
import torch

from test_gpu_few import ops, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


def setup(grad=False):
    from trenowanie_generatora_obrazkow_amd.moe_triton import grouped_mm
    w = ops().F8Stack.from_weights(rand(3, 64, 48, seed=1), grad=grad)
    return grouped_mm, w, torch.tensor([5, 0, 9], device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_in_any_stride(dtype):
    mm, w, counts = setup()
    a = rand(14, 64, seed=2, dtype=dtype)
    y = mm(a, w, counts)
    wide = torch.zeros(14, 77, device=DEV, dtype=dtype)  # an odd stride, then one of a row too many
    wide[:, 5:69] = a
    off = torch.zeros(14 * 64 + 1, device=DEV, dtype=dtype)
    off[1:] = a.flatten()
    for view in (wide[:, 5:69], a.t().contiguous().t(), off[1:].view(14, 64), a.repeat_interleave(2, 0)[::2]):
        assert torch.equal(mm(view, w, counts), y)
    one = rand(1, 64, seed=3, dtype=dtype)
    row = one.expand(14, 64)  # one row for all
    assert torch.equal(mm(row, w, counts), mm(row.contiguous(), w, counts))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_that_begin_anywhere(dtype):
    mm, w, counts = setup(grad=True)
    a = rand(14, 64, seed=2, dtype=dtype).requires_grad_()
    dy = rand(14, 48, seed=4, dtype=dtype)
    (want,) = torch.autograd.grad(mm(a, w, counts), a, dy)
    off = torch.zeros(14 * 48 + 3, device=DEV, dtype=dtype)
    off[3:] = dy.flatten()
    wide = torch.zeros(14, 51, device=DEV, dtype=dtype)
    wide[:, 1:49] = dy
    for g in (off[3:].view(14, 48), wide[:, 1:49], dy.t().contiguous().t()):
        (got,) = torch.autograd.grad(mm(a, w, counts), a, g)
        assert torch.equal(got, want)
    (got,) = torch.autograd.grad(mm(a, w, counts).sum(), a)  # one number for all
    (want,) = torch.autograd.grad(mm(a, w, counts), a, torch.ones(14, 48, device=DEV, dtype=dtype))
    assert torch.equal(got, want)
