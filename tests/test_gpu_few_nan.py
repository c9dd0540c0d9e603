"""A layer for a few tokens with its router inside the first kernel, on tokens whose logits are NaN: the later slots of such a token
name no expert and read nothing, its output is NaN, and the other tokens keep their bits."""
import pytest
import torch

from test_gpu_few import ops, rand, weights

pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("E,k", [(16, 2), (10, 3), (3, 3), (16, 16), (1, 1), (40, 2)])
@pytest.mark.parametrize("T,bad", [(1, (0,)), (6, (3,)), (16, (0, 7, 15))])
def test_nan_tokens(E, k, T, bad):
    o = ops()
    d, h = 136, 48
    w, _ = weights("bf16", E, d, h, torch.bfloat16)
    x, wr = rand(T, d, seed=T), rand(E, d, seed=5, std=d ** -0.5)
    y, ids, tw = o.few_forward(x, wr, w["wgu"], w["wd"], k)
    for value in (float("nan"), float("inf")):
        x2 = x.clone()
        for t in bad:
            x2[t, 9 * t % d] = value
        y2, ids2, tw2 = o.few_forward(x2, wr, w["wgu"], w["wd"], k)
        _, ids3, tw3 = o.route_topk(x2, wr, k)
        assert torch.equal(ids2, ids3) and same(tw2, tw3)
        keep = [t for t in range(T) if t not in bad]
        assert torch.equal(y2[keep], y[keep]) and torch.equal(ids2[keep], ids[keep]) and torch.equal(tw2[keep], tw[keep])
        assert not torch.isfinite(y2[list(bad)]).any()


def test_nan_router_weights():
    """A router that is NaN throughout, or for one expert: every token's weights are NaN, and so is its output."""
    o = ops()
    T, E, k, d, h = 5, 12, 3, 64, 48
    w, _ = weights("bf16", E, d, h, torch.bfloat16)
    x, wr = rand(T, d), rand(E, d, seed=5, std=d ** -0.5)
    for rows in (slice(None), slice(4, 5)):
        wr2 = wr.clone()
        wr2[rows, 2] = float("nan")
        y, ids, tw = o.few_forward(x, wr2, w["wgu"], w["wd"], k)
        _, ids3, tw3 = o.route_topk(x, wr2, k)
        assert torch.equal(ids, ids3) and same(tw, tw3)
        assert torch.isnan(y).all()


def test_nan_token_through_the_module():
    from trenowanie_generatora_obrazkow_amd import MoESwiGLU
    m = MoESwiGLU(64, 48, 8, top_k=2, device="cuda", few_tokens=16).eval()
    x = rand(5, 64)
    with torch.no_grad():
        y = m(x)
        x2 = x.clone()
        x2[2, 1] = float("nan")
        y2 = m(x2)
    assert torch.isnan(y2[2]).all()
    keep = [0, 1, 3, 4]
    assert torch.equal(y2[keep], y[keep])
