"""Rows and elements past 32-bit offsets: the norms, routing and clipping on tensors of more than 4 GiB, against the same rows
or elements taken alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _far(T, d, ld, dt, seed):
    """(T, d) rows that lie ld elements apart, and their contiguous copy."""
    buf = torch.empty((T - 1) * ld + d, dtype=dt, device="cuda")
    x = buf.as_strided((T, d), (ld, 1))
    v = torch.randn(T, d, generator=torch.Generator().manual_seed(seed)).to(dt).cuda()
    x.copy_(v)
    return x, v


def test_far_rows():
    from trenowanie_generatora_obrazkow_amd import ops
    x, v = _far(5, 520, (1 << 29) + 8, BF, 1)           # 4.3 GB between the first row and the last
    w, u = torch.randn(520, device="cuda"), torch.randn(5, 520, device="cuda").to(BF)
    assert torch.equal(ops.norm_modulate(x, w), ops.norm_modulate(v, w))
    assert torch.equal(ops.norm_residual(u, x, weight=w), ops.norm_residual(u, v, weight=w))
    for a, b in zip(ops.norm_modulate_bwd(u, x, w), ops.norm_modulate_bwd(u, v, w)):
        assert a is None and b is None or torch.equal(a, b)
    lg, lv = _far(5, 48, (1 << 28) + 3, torch.float32, 2)
    ids, tw = ops.route_scores(lg, 4, "sigmoid", None, 8, 4)
    i2, t2 = ops.route_scores(lv, 4, "sigmoid", None, 8, 4)
    assert torch.equal(ids, i2) and torch.equal(tw, t2)
    for score in ("sigmoid", "softmax"):
        assert torch.equal(ops.route_scores_bwd(tw, tw, lg, ids, score), ops.route_scores_bwd(tw, tw, lv, ids, score))


def test_many_rows():
    from trenowanie_generatora_obrazkow_amd import ops
    T, d, k, n = 1_100_000, 1024, 2, 300                 # 2.25 GB of x, 4.5 GB of y
    y = torch.zeros(T * k, d, dtype=BF, device="cuda")
    x = torch.zeros(T, d, dtype=BF, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    x[-n:] = torch.randn(n, d, generator=g, device="cuda")
    y[-n * k:] = torch.randn(n * k, d, generator=g, device="cuda")
    gate = torch.randn(d, generator=g, device="cuda")
    assert torch.equal(ops.norm_residual(y, x, gate, k=k)[-n:], ops.norm_residual(y[-n * k:], x[-n:], gate, k=k))
    dy, dg, _ = ops.norm_residual_bwd(x, y, gate, k=k)
    dy2, dg2, _ = ops.norm_residual_bwd(x[-n:], y[-n * k:], gate, k=k)
    assert torch.equal(dy[-n:], dy2)
    # the same terms in another order: n of them, each off by a few 2^-24 of the sum of their absolute values
    assert (dg - dg2).abs().max() <= 64 * 2.0 ** -24 * n * 16


def test_many_elements():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm
    n = (1 << 31) + 12345                                # 4.3 GB in bf16, 8.6 GB of fp32 output
    g = torch.zeros(n, dtype=BF, device="cuda")
    g[:3] = 3.0
    g[-3:] = 4.0
    out = torch.empty(n, device="cuda")
    norm = clip_grad_norm([g], 1.0, out=[out])
    want = 75.0 ** 0.5
    assert abs(float(norm) - want) <= 2e-7 * want
    c = 1.0 / (want + 1e-6)
    assert (out[:3] - 3 * c).abs().max() <= 1e-6 and (out[-3:] - 4 * c).abs().max() <= 1e-6
    assert out[3:-3].abs().max() == 0
