"""The gradient of the 8-bit product's rows against differences, where nothing is rounded on the way to 8 bits.

Rows a, the direction v and the output's gradient dy hold whole numbers of at most 15 in magnitude, a +- v as well.  A block's scale
is the least 2^e with its largest value at most 448 * 2^e, so 2^-4 at most here, and such numbers times 16 have four significant
bits: they are e4m3 values.  The product is then linear in a, and

    (<y(a + v), dy> - <y(a - v), dy>) / 2 = <da, v>

but for the products' own errors (test_gpu_f8.py: what the 8-bit matrix instructions drop, the fp32 sums, the fp32 outputs).  v has
the gradient's signs, so that <da, v> is the sum of its magnitudes: a factor on da, or a block's scale missing, shows."""
import pytest
import torch

import f8_ref as R
from test_gpu_f8 import DEV, HALF, ops, products, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,M,K,N,kind", [(1, 64, 256, 256, "even"), (3, 200, 144, 400, "skew"), (4, 90, 400, 144, "one")])
def test_gradient_against_exact_differences(E, M, K, N, kind):
    from trenowanie_generatora_obrazkow_amd.moe_triton import grouped_mm
    g = torch.Generator().manual_seed(M)
    whole = lambda *s: torch.randint(-7, 8, s, generator=g).float().to(DEV)
    a, dy = whole(M, K).requires_grad_(True), whole(M, N)
    # stacks whose blocks have scales of their own
    w = rand(E, K, N, seed=N, spread=False) * K ** -0.5 * torch.exp2(torch.arange(N, device=DEV) // 128 - torch.arange(K, device=DEV)[:, None] // 128)
    st = ops().F8Stack.from_weights(w, grad=True)
    counts = R.counts_of(M, E, kind).to(DEV)
    e = torch.repeat_interleave(torch.arange(E), counts.long().cpu())
    wd = st.dequant().double().cpu()
    full, err_da = products(dy.double().cpu(), wd.transpose(1, 2).contiguous(), e)
    v = 2 * full.sign()
    err_da = err_da + HALF[torch.float32] * (full.abs() + err_da)
    diff, bound = 0.0, float((err_da * v.abs()).sum())
    grouped_mm(a, st, counts).backward(dy)
    got = float((a.grad.double().cpu() * v).sum())
    for s in (1, -1):
        t = a.detach() + s * v.float().to(DEV)
        ref, err = products(t.double().cpu(), wd, e)
        diff += s * float((grouped_mm(t, st, counts).double() * dy.double()).sum()) / 2
        bound += float(((err + HALF[torch.float32] * (ref.abs() + err)) * dy.double().cpu().abs()).sum()) / 2
    assert bound < 0.1 * diff
    assert abs(got - diff) <= bound
