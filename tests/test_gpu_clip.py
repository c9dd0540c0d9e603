"""Gradient clipping by the global norm (clip_grad_norm, grad_sq_norm, grad_clip) against 64-bit arithmetic: types, sizes around
the vector and chunk sizes, views that start at any element, more tensors than one launch takes, outputs in fp32, NaN and
infinities, a factor of one.

Tolerances.  The squares and their sum are fp64 (n 2^-53 at most), the norm is rounded once to fp32; the factor is rounded once
to fp32, the product once in fp32 and once to the output's type: 2 2^-24 plus the type's half step."""
import math

import pytest
import torch

from tests import block_ref as R

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _norm64(grads):
    return math.sqrt(sum(float(g.double().cpu().square().sum()) for g in grads))


def _check(got, src, factor):
    ref = src.double().cpu() * factor
    tol = (2 * R.EPS24 + R.half_step(got.dtype)) * ref.abs() * 1.001 + 2 * R.tiny(got.dtype)
    assert ((got.double().cpu() - ref).abs() <= tol).all()


def _lists():
    g = torch.Generator().manual_seed(3)
    r = lambda n, dt, std: (torch.randn(n, generator=g) * std).to(dt).cuda()
    mixed = [r(n, dt, s) for n in (1, 7, 8, 9, 2047, 2048, 16383, 16384, 16385, 100003)
             for dt, s in ((BF, 0.1), (HF, 0.03), (FP, 1.0))]
    bucket = r(20000, BF, 0.5)
    views = list(bucket.split([1 + 13 * i for i in range(50)] + [20000 - 50 - 13 * 1225]))
    fbucket = r(5001, FP, 0.5)
    many = [r(i % 5, FP, 0.2) for i in range(300)]
    return {"mixed": mixed, "views": views, "fviews": [fbucket[1:], fbucket[:1]], "many": many,
            "shapes": [r(24, BF, 1.0).view(2, 3, 4), r(60, FP, 1.0).view(6, 10).t(), r(1, HF, 1.0).view(())]}


@pytest.mark.parametrize("name", ["mixed", "views", "fviews", "many", "shapes"])
@pytest.mark.parametrize("mode", ["inplace", "same", "fp32"])
def test_clip(name, mode):
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    grads = _lists()[name]
    print("clip", name, mode, flush=True)
    src = [t.clone() for t in grads]
    norm = _norm64(src)
    out = None if mode == "inplace" else [torch.full_like(t, math.nan, dtype=t.dtype if mode == "same" else FP) for t in grads]
    got = clip_grad_norm(grads, 0.5 * norm, out=out)
    assert got.shape == () and got.dtype == FP and abs(float(got) - norm) <= 1.01 * R.EPS24 * norm
    factor = 0.5 * norm / (norm + 1e-6)
    for a, b in zip(grads if out is None else out, src):
        _check(a, b, factor)
    if out is not None:
        assert all(torch.equal(a, b) for a, b in zip(grads, src))


def test_below_the_bound_nothing_changes():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    grads = _lists()["mixed"]
    src = [t.clone() for t in grads]
    norm = _norm64(src)
    for bound in (2 * norm, math.inf):
        got = clip_grad_norm(grads, bound)
        assert abs(float(got) - norm) <= 1.01 * R.EPS24 * norm
        assert all(torch.equal(a, b) for a, b in zip(grads, src))
    out = [torch.empty_like(t, dtype=FP) for t in grads]
    clip_grad_norm(grads, 2 * norm, out=out)
    assert all(torch.equal(a, b.float()) for a, b in zip(out, src))


def test_neighbours_are_left_alone():
    """Views of a bucket, clipped in place, change no element beside them."""
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    for dt in (BF, FP):
        bucket = torch.ones(40000, dtype=dt, device="cuda")
        clip_grad_norm([bucket[3:3 + 17000], bucket[20001:20001 + 9], bucket[30000:30000]], 0.0)
        b = bucket.cpu()
        assert not b[3:17003].any() and not b[20001:20010].any()
        assert (b[:3] == 1).all() and (b[17003:20001] == 1).all() and (b[20010:] == 1).all()


def test_extreme_values():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm, ops
    big = torch.full((1000,), 1e30, device="cuda")
    small = torch.full((3000,), 1e-30, device="cuda")
    assert abs(float(ops.grad_sq_norm([big])) / 1e63 - 1) < 1e-6
    assert abs(float(ops.grad_sq_norm([small])) / 3e-57 - 1) < 1e-6
    n = clip_grad_norm([big], 1.0)
    assert abs(float(n) / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    assert torch.allclose(big, torch.full_like(big, 1000 ** -0.5), rtol=1e-6)
    # NaN anywhere makes all gradients NaN; an infinite norm zeros, and NaN where a gradient is infinite
    a, b = torch.ones(5, device="cuda"), torch.ones(9, device="cuda", dtype=BF)
    a[2] = math.nan
    assert torch.isnan(clip_grad_norm([a, b], 1.0)) and torch.isnan(a).all() and torch.isnan(b).all()
    a, b = torch.ones(5, device="cuda"), torch.ones(9, device="cuda", dtype=BF)
    a[2] = math.inf
    assert torch.isinf(clip_grad_norm([a, b], 1.0)) and torch.isnan(a[2]) and not b.any() and not a[[0, 1, 3, 4]].any()


def test_empty_lists_and_none():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    assert float(clip_grad_norm([], 1.0)) == 0
    assert float(clip_grad_norm([None, torch.empty(0, device="cuda")], 1.0)) == 0
    g = torch.full((4,), 3.0, device="cuda")
    out = [None, torch.empty(4, device="cuda")]
    assert float(clip_grad_norm([None, g], 1.0, out=out)) == 6.0 and abs(float(out[1][0]) - 0.5) < 1e-6


def test_two_halves():
    """The squared norms of two lists, added on the device, clip each by the norm of both."""
    from trenowanie_generatora_obrazkow_amd import ops
    g = torch.Generator().manual_seed(1)
    a, b = [torch.randn(500, generator=g).cuda()], [torch.randn(700, generator=g).cuda()]
    sa, sb = a[0].clone(), b[0].clone()
    sq = ops.grad_sq_norm(a) + ops.grad_sq_norm(b)
    norm = _norm64([sa, sb])
    ops.grad_clip(a, sq, 1.0)
    ops.grad_clip(b, sq, 1.0)
    _check(a[0], sa, 1.0 / (norm + 1e-6))
    _check(b[0], sb, 1.0 / (norm + 1e-6))


def test_same_bits_every_time_and_replays():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    from trenowanie_generatora_obrazkow_amd.graphs import StepGraph
    g = torch.Generator().manual_seed(2)
    grads = [torch.randn(n, generator=g).to(dt).cuda() for n, dt in ((300001, BF), (7, FP), (50000, HF))] \
        + [torch.randn(11, generator=g).cuda() for _ in range(150)]
    out = [torch.empty_like(t) for t in grads]
    step = lambda: (clip_grad_norm(grads, 3.0, out=out), *out)
    graph = StepGraph(step)
    for rep in range(3):
        if rep:
            grads[0].mul_(1.5)
        want = [t.clone() for t in step()]
        again = [t.clone() for t in step()]
        got = graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, again))
        assert all(torch.equal(a, b) for a, b in zip(want, got)), rep
