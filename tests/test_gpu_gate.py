"""Routing from logits (route_scores) and its backward against 64-bit arithmetic: both scores, selection bias, groups of any
size, ties, disabled experts, rows without a finite logit, NaN, padding tokens, types and row strides.

Tolerances.  Ids are equal.  A score is exp (1 ulp), a sum of E terms over 16 lanes (E / 16 + 4 steps) and a division: relative
error (E / 16 + 8) 2^-24; a weight adds the sum over k slots, a division and a product: (E / 16 + 32) 2^-24 in all.  dlogits
is a sum of terms of the size p (|ds| + sum p |ds|), each with that error, and one rounding to the logits' type."""
import math

import pytest
import torch

from tests import block_ref as R

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32

CASES = [
    # T, E, k, score, bias, n_group, topk_group, group_top, renorm, dtype, padded
    (1, 1, 1, "softmax", False, 1, 1, 2, True, FP, False),
    (5, 4, 4, "sigmoid", True, 1, 1, 2, False, FP, False),
    (33, 16, 2, "softmax", True, 1, 1, 2, True, FP, True),
    (257, 17, 3, "softmax", False, 1, 1, 2, False, BF, True),
    (100, 40, 5, "sigmoid", False, 8, 3, 2, True, FP, False),      # five experts per group
    (64, 128, 8, "sigmoid", True, 8, 2, 2, True, FP, False),
    (70, 160, 6, "softmax", False, 8, 3, 1, False, FP, True),      # groups by their best expert
    (50, 150, 12, "softmax", True, 6, 2, 2, True, HF, False),
    (40, 256, 8, "sigmoid", True, 8, 4, 2, True, BF, True),
    (31, 300, 16, "softmax", True, 1, 1, 2, True, FP, False),
    (20, 512, 10, "sigmoid", True, 64, 7, 2, True, FP, True),
    (21, 512, 16, "softmax", False, 2, 1, 2, True, FP, False),
    (19, 384, 7, "sigmoid", False, 48, 48, 2, True, FP, False),    # every group kept
    (12, 66, 9, "sigmoid", True, 33, 9, 1, False, FP, False),
]
names = [f"{c[0]}x{c[1]}k{c[2]}{c[3][:2]}g{c[5]}" for c in CASES]


def _inputs(T, E, k, dtype, bias, padded, seed):
    g = torch.Generator().manual_seed(seed)
    lg = (torch.randn(T, E, generator=g) * 1.5).to(dtype)
    b = torch.randn(E, generator=g) * 0.1 if bias else None
    live = torch.rand(T, generator=g) < 0.8 if padded else None
    return lg, b, live, torch.randn(T, k, generator=g)


def _dev(t):
    return None if t is None else t.cuda()


def _check(got, ref, rel, extra=0.0):
    got64 = got.cpu().double()
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got64), nan)
    bound = rel * ref.abs() + extra + R.half_step(got.dtype) * ref.abs() + R.tiny(got.dtype)
    assert ((got64 - ref).abs() <= bound)[~nan].all(), float(((got64 - ref).abs() / (bound + 1e-300))[~nan].max())


def _check_bwd(dl, lg, ids, w, dtw, score, renorm, scaling):
    E = lg.shape[1]
    rel = (E / 16 + 64) * R.EPS24
    leaf = lg.double().requires_grad_(True)
    out = R.route_weights(leaf, ids, w, score, renorm, scaling)
    ref, = torch.autograd.grad((out * dtw.double()).sum(), leaf)
    with torch.no_grad():
        s = torch.softmax(leaf, 1) if score == "softmax" else torch.sigmoid(leaf)
        on = (ids >= 0) & (w != 0)
        sel = torch.where(on, s.gather(1, ids.long().clamp(min=0)), 0.0)
        den = sel.sum(1, keepdim=True) + 1e-20 if renorm else 1.0
        u = (scaling * dtw.double()).abs()
        ds = (u + ((u * sel).sum(1, keepdim=True) / den if renorm else 0.0)) / den
        ds = torch.where(on, ds, 0.0)
        mag = torch.zeros_like(s).scatter_add_(1, ids.long().clamp(min=0), ds * (sel if score == "sigmoid" else 1.0))
        if score == "softmax":
            mag = s * (mag + (sel * ds).sum(1, keepdim=True))
    _check(dl, ref, 0.0, rel * mag)


@pytest.mark.parametrize("case", CASES, ids=names)
def test_route_scores(case):
    from trenowanie_generatora_obrazkow_amd import ops
    T, E, k, score, bias, ng, tg, gt, renorm, dtype, padded = case
    print("route_scores", case, flush=True)
    lg, b, live, dtw = _inputs(T, E, k, dtype, bias, padded, T + E)
    ids, w = ops.route_scores(lg.cuda(), k, score, _dev(b), ng, tg, gt, renorm, 2.5, _dev(live))
    rid, rw = R.route(lg, k, score, b, ng, tg, gt, renorm, 2.5, live)
    assert torch.equal(ids.cpu(), rid)
    _check(w, rw, (E / 16 + 32) * R.EPS24)
    dl = ops.route_scores_bwd(dtw.cuda(), w, lg.cuda(), ids, score, renorm, 2.5)
    assert dl.dtype == dtype
    _check_bwd(dl, lg, rid, rw, dtw, score, renorm, 2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [False, True])
def test_ties_and_disabled_experts(score, groups):
    """Equal values go to the lower expert; experts off by logit or bias come last, lowest first, with the weight 0; a row
    with nothing left keeps defined ids, zero weights and zero gradients; the type's lowest value is not -inf."""
    from trenowanie_generatora_obrazkow_amd import ops
    inf = math.inf
    E, k = 32, 4
    ng, tg = (8, 2) if groups else (1, 1)
    lg = torch.zeros(8, E)
    lg[1, ::3] = 1.0
    lg[2] = -inf
    lg[3] = -inf
    lg[3, [5, 9]] = 0.25
    lg[4] = torch.finfo(FP).min
    lg[5, 7:] = -inf
    lg[6] = torch.arange(E) % 4 * 0.5
    lg[7] = 60.0
    bias = torch.zeros(E)
    bias[2] = -inf
    for b in (None, bias):
        ids, w = ops.route_scores(lg.cuda(), k, score, _dev(b), ng, tg)
        rid, rw = R.route(lg, k, score, b, ng, tg, 2, True, 1.0, None)
        assert torch.equal(ids.cpu(), rid), (b is None, ids, rid)
        _check(w, rw, 64 * R.EPS24)
        assert not w[2].any()
        dl = ops.route_scores_bwd(torch.ones(8, k, device="cuda"), w, lg.cuda(), ids, score).cpu()
        assert torch.isfinite(dl).all() and not dl[2].any()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_nan_and_infinite_logits(score):
    from trenowanie_generatora_obrazkow_amd import ops
    lg = torch.randn(4, 20, generator=torch.Generator().manual_seed(2))
    lg[0, 3] = math.nan
    lg[1, 4] = math.inf
    lg[2] = math.nan
    for b in (None, torch.zeros(20)):
        ids, w = ops.route_scores(lg.cuda(), 3, score, _dev(b))
        ids, w = ids.cpu(), w.cpu()
        assert ((ids >= 0) & (ids < 20)).all() and all(len(set(r)) == 3 for r in ids.tolist())
        assert 3 not in ids[0].tolist() or b is not None and score == "softmax"
        assert torch.isfinite(w[3]).all()
        if score == "softmax":
            assert torch.isnan(w[:3]).all()
        else:
            assert ids[1, 0] == 4 and torch.isfinite(w).all() and not w[2].any()


def test_close_selection_values():
    """Scores that fp32 cannot tell apart: sigmoid of logits near 12 differ by less than an fp32 step of the score, and the
    bias moves them by that much."""
    from trenowanie_generatora_obrazkow_amd import ops
    g = torch.Generator().manual_seed(4)
    lg = 12 + torch.rand(200, 64, generator=g)
    bias = torch.rand(64, generator=g) * 1e-6
    for b in (None, bias):
        ids, _ = ops.route_scores(lg.cuda(), 8, "sigmoid", _dev(b))
        assert torch.equal(ids.cpu(), R.route(lg, 8, "sigmoid", b, 1, 1, 2, True, 1.0, None)[0])


def test_row_stride_and_no_tokens():
    from trenowanie_generatora_obrazkow_amd import ops
    wide = torch.randn(30, 77, generator=torch.Generator().manual_seed(8)).cuda()
    lg = wide[:, 3:3 + 40]
    a, b = ops.route_scores(lg, 4), ops.route_scores(lg.contiguous(), 4)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    dtw = torch.ones(30, 4, device="cuda")
    assert torch.equal(ops.route_scores_bwd(dtw, a[1], lg, a[0], renorm=False),
                       ops.route_scores_bwd(dtw, a[1], lg.contiguous(), a[0], renorm=False))
    ids, w = ops.route_scores(lg[:0], 4)
    assert ids.shape == (0, 4) and ops.route_scores_bwd(w, w, lg[:0], ids).shape == (0, 40)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_repeated_and_foreign_ids(score):
    """An expert named by two slots gets the sum of both gradients; ids outside [0, E) and zero weights have none."""
    from trenowanie_generatora_obrazkow_amd import ops
    g = torch.Generator().manual_seed(6)
    lg = torch.randn(3, 24, generator=g)
    ids = torch.tensor([[3, 3, 5], [-1, 7, 24], [1, 2, 2 ** 31 - 1]], dtype=torch.int32)
    w = torch.tensor([[1.0, 1.0, 1.0], [1.0, 1.0, 1.0], [0.0, 1.0, 1.0]])
    dtw = torch.randn(3, 3, generator=g)
    dl = ops.route_scores_bwd(dtw.cuda(), w.cuda(), lg.cuda(), ids.cuda(), score, False, 1.0)
    on = torch.where(ids >= 24, -1, ids)
    _check_bwd(dl, lg, on, w, dtw, score, False, 1.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_against_differences(score):
    """Central differences of the kernel's own fp32 weights: truncation t^2 / 6 and rounding 2^-22 / t of unit-sized terms,
    below 1e-3 at t = 2^-6, while the ids stay."""
    from trenowanie_generatora_obrazkow_amd import ops
    g = torch.Generator().manual_seed(12)
    T, E, k, t = 64, 24, 4, 2.0 ** -6
    lg = torch.stack([torch.randperm(E, generator=g) for _ in range(T)]).float().cuda() * 0.25
    dtw = torch.randn(T, k, generator=g).cuda()
    e = torch.sign(torch.randn(T, E, generator=g)).cuda()
    ids, w = ops.route_scores(lg, k, score)
    dl = ops.route_scores_bwd(dtw, w, lg, ids, score)
    hi, lo = ops.route_scores(lg + t * e, k, score), ops.route_scores(lg - t * e, k, score)
    assert torch.equal(hi[0], ids) and torch.equal(lo[0], ids)
    diff = ((hi[1] - lo[1]).double() * dtw.double()).sum(1) / (2 * t)
    want = (dl.double() * e.double()).sum(1)
    assert ((diff - want).abs() <= 1e-3 * dtw.double().abs().sum(1)).all()


def test_padding_tokens_route_nowhere():
    """A padded batch through routing, experts and combine: the live tokens' rows are those of the batch without padding."""
    from trenowanie_generatora_obrazkow_amd import ops
    g = torch.Generator().manual_seed(15)
    T, d, E, k, h = 90, 64, 16, 2, 64
    x = torch.randn(T, d, generator=g).bfloat16().cuda()
    wgu = (torch.randn(E, d, 2 * h, generator=g) * 0.1).bfloat16().cuda()
    wd = (torch.randn(E, h, d, generator=g) * 0.1).bfloat16().cuda()
    lg = torch.randn(T, E, generator=g).cuda()
    live = (torch.rand(T, generator=g) < 0.7).cuda()
    x[~live] = math.nan

    def out(lg, x, live):
        ids, w = ops.route_scores(lg, k, "sigmoid", n_group=4, topk_group=2, live=live)
        y, inv, _ = ops.moe_experts(x, ids, w, wgu, wd)
        return ops.combine(y, x.shape[0], k, inv_pos=inv)

    a, b = out(lg, x, live), out(lg[live].contiguous(), x[live].contiguous(), None)
    assert torch.equal(a[live], b) and not a[~live].any()


def test_replays():
    from trenowanie_generatora_obrazkow_amd import ops
    from trenowanie_generatora_obrazkow_amd.graphs import StepGraph
    g = torch.Generator().manual_seed(1)
    lg = torch.randn(500, 64, generator=g).cuda()
    bias = torch.zeros(64, device="cuda")
    dtw = torch.randn(500, 6, generator=g).cuda()

    def step():
        ids, w = ops.route_scores(lg, 6, "sigmoid", bias, 8, 4)
        return ids, w, ops.route_scores_bwd(dtw, w, lg, ids, "sigmoid")

    graph = StepGraph(step)
    for rep in range(3):
        if rep:
            lg.copy_(torch.randn(500, 64, generator=g))
            bias.copy_(torch.randn(64, generator=g) * 0.1)
        want = [t.clone() for t in step()]
        got = graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep
