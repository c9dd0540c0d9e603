"""Padding tokens in the backward of the routing: their logits may hold anything, their gradient is zero and the other tokens'
that of clean logits, bit for bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_garbage_logits_of_padding_tokens(score, renorm, dtype):
    from trenowanie_generatora_obrazkow_amd import ops
    g = torch.Generator().manual_seed(17)
    for T, E, k in ((37, 16, 2), (50, 100, 5)):
        lg = (torch.randn(T, E, generator=g) * 1.5).to(dtype)
        live = torch.rand(T, generator=g) < 0.6
        bad = lg.clone()
        off = (~live).nonzero().squeeze(1)
        bad[off[0::4], 3] = math.nan
        bad[off[1::4], 0] = math.inf
        bad[off[2::4]] = math.nan
        bad[off[3::4]] = -math.inf
        dtw = torch.randn(T, k, generator=g)
        dtw_bad = dtw.clone()
        dtw_bad[off[::2]] = math.nan
        got = []
        for l, dw in ((lg, dtw), (bad, dtw_bad)):
            ids, w = ops.route_scores(l.cuda(), k, score, renorm=renorm, live=live.cuda())
            got.append((ids, w, ops.route_scores_bwd(dw.cuda(), w, l.cuda(), ids, score, renorm)))
        assert all(torch.equal(a, b) for a, b in zip(*got))
        dl = got[1][2].cpu()
        assert not dl[off].any() and dl[live].abs().amax(1).min() > 0
