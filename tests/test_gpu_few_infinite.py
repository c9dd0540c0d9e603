"""A layer for a few tokens whose activations leave bf16's range: they enter the down projection as infinities, as in a larger
call, and other tokens keep their bits."""
import pytest
import torch

from test_gpu_few import ops, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_activations_past_the_range(kind):
    o = ops()
    E, d, h, k = 2, 64, 48, 1
    wgu = torch.zeros(E, d, 2 * h, device=DEV)
    wgu[:, 0, :h] = 1.0             # g = x[0]
    wgu[:, 1, h:], wgu[:, 2, h:] = 1.0, 1.0  # u = x[1] + x[2]
    wd = torch.arange(1, h + 1, device=DEV)[None, :, None].expand(E, h, d) / 64.0
    if kind == "int8":
        w = dict(wgu=wgu.to(torch.int8), wd=(wd * 64).to(torch.int8).contiguous(), wgu_s=torch.ones(E, 2 * h, device=DEV),
                 wd_s=torch.full((E, d), 1 / 64.0, device=DEV))
    else:
        w = dict(wgu=wgu.bfloat16(), wd=wd.bfloat16().contiguous())
    x = torch.zeros(5, d, device=DEV)
    x[0, :2] = torch.tensor([1e25, 1e25])                    # act overflows fp32
    x[1, :3] = torch.tensor([2.0 ** 64, 2.0 ** 64, -2.0 ** 54])  # finite, and rounds to an infinite bf16
    x[2, :2] = torch.tensor([1e25, -1e25])
    x[3] = rand(d, seed=1).float()
    x[4, :2] = torch.tensor([float("inf"), 2.0])             # (inf * 0 in the sums)
    x = x.bfloat16()
    ids = torch.zeros(5, k, dtype=torch.int32, device=DEV)
    tw = torch.ones(5, k, device=DEV)
    y = o.few_experts(x, ids, tw, **w).float()
    assert (y[0] == float("inf")).all() and (y[1] == float("inf")).all() and (y[2] == -float("inf")).all()
    z, inv, _ = o.moe_experts(x, ids, tw, **w)
    z = o.combine(z, 5, k, inv_pos=inv).float()
    assert torch.equal(z[[0, 1, 2]], y[[0, 1, 2]]) and torch.equal(torch.isnan(z), torch.isnan(y))
    assert torch.isfinite(y[3]).all() and torch.equal(o.few_experts(x[3:4], ids[3:4], tw[3:4], **w)[0].float(), y[3])
