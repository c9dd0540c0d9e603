"""Refusals of the tensor-level wrappers of the norms, routing from logits and gradient clipping: wrong shapes, types, layouts
and mixtures stop on the host."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_refusals():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm, ops
    dev = "cuda"
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device=dev, dtype=dt)
    f32 = torch.float32
    x = z(6, 64)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    bad = [
        # norms: width, layout, parameter shapes and types, samples, starts, types of stream and block
        lambda: ops.norm_modulate(z(6, 60)), lambda: ops.norm_modulate(z(2, 3, 64)), lambda: ops.norm_modulate(z(64, 6).t()),
        lambda: ops.norm_modulate(z(6, 68)[:, :64]), lambda: ops.norm_modulate(z(1, 64).expand(6, 64)),
        lambda: ops.norm_modulate(x, weight=z(63)), lambda: ops.norm_modulate(x, weight=z(64, dt=torch.int32)),
        lambda: ops.norm_modulate(x, weight=torch.zeros(64)), lambda: ops.norm_modulate(x, scale=z(4, 64)),
        lambda: ops.norm_modulate(x, scale=z(2, 64), shift=z(3, 64)),
        lambda: ops.norm_modulate(x, scale=z(2, 64), shift=z(2, 64, dt=f32)),
        lambda: ops.norm_modulate(x, scale=z(64, 2).t()),
        lambda: ops.norm_modulate(x, scale=z(2, 64), starts=i32(0, 2, 4, 6)), lambda: ops.norm_modulate(x, starts=i32(0)),
        lambda: ops.norm_modulate(x, starts=i32(0, 6).long()), lambda: ops.norm_modulate(x, dtype=f32),
        lambda: ops.norm_modulate(x, dtype=torch.float16), lambda: ops.norm_modulate(z(6, 64, dt=torch.float64)),
        lambda: ops.norm_modulate_bwd(z(5, 64), x), lambda: ops.norm_modulate_bwd(z(6, 64, dt=f32), x),
        lambda: ops.norm_modulate_bwd(x, x, dres=z(6, 64, dt=f32)), lambda: ops.norm_modulate_bwd(z(64, 6).t(), x),
        lambda: ops.norm_residual(z(11, 64), x, k=2), lambda: ops.norm_residual(x, x, k=0),
        lambda: ops.norm_residual(z(6, 64, dt=f32), x), lambda: ops.norm_residual(x, x, inv_pos=i32(0, 1)),
        lambda: ops.norm_residual(x, x, add=z(6, 64, dt=f32)), lambda: ops.norm_residual(x, x, gate=z(5, 64)),
        lambda: ops.norm_residual_bwd(x, z(6, 64, dt=torch.float16)), lambda: ops.norm_residual_bwd(z(6, 128)[:, :64], x),
        # routing
        lambda: ops.route_scores(z(6, 64), 0), lambda: ops.route_scores(z(6, 64), 17), lambda: ops.route_scores(z(6, 4), 5),
        lambda: ops.route_scores(z(6, 600), 2), lambda: ops.route_scores(z(6, 64, dt=torch.int32), 2),
        lambda: ops.route_scores(z(64), 2), lambda: ops.route_scores(z(6, 64), 2, score="relu"),
        lambda: ops.route_scores(z(6, 64), 2, bias=z(64)), lambda: ops.route_scores(z(6, 64), 2, bias=z(63, dt=f32)),
        lambda: ops.route_scores(z(6, 64), 2, live=i32(1, 1, 1, 1, 1, 1)), lambda: ops.route_scores(z(64, 6).t(), 2),
        lambda: ops.route_scores(z(6, 64), 2, n_group=7, topk_group=2), lambda: ops.route_scores(z(6, 64), 9, n_group=8, topk_group=1),
        lambda: ops.route_scores(z(6, 64), 2, n_group=64, topk_group=8), lambda: ops.route_scores(z(6, 64), 2, n_group=8, topk_group=9),
        lambda: ops.route_scores(z(6, 64), 2, group_top=3, n_group=8, topk_group=2),
        lambda: ops.route_scores_bwd(z(6, 2), z(6, 2, dt=f32), x, i32(0, 0)[None].repeat(6, 1)),
        lambda: ops.route_scores_bwd(z(6, 2, dt=f32), z(6, 2, dt=f32), x, z(6, 2, dt=torch.int64)),
        lambda: ops.route_scores_bwd(z(5, 2, dt=f32), z(5, 2, dt=f32), x, z(5, 2, dt=torch.int32)),
        # clipping: types, layouts, outputs, bounds, a tensor twice
        lambda: clip_grad_norm([z(4, dt=torch.int32)], 1.0), lambda: clip_grad_norm([z(8)[::2]], 1.0),
        lambda: clip_grad_norm([z(4), torch.zeros(4)], 1.0), lambda: clip_grad_norm([x, x], 1.0),
        lambda: clip_grad_norm([z(4)], 1.0, out=[z(4), z(4)]), lambda: clip_grad_norm([z(4)], 1.0, out=[z(5)]),
        lambda: clip_grad_norm([z(4)], 1.0, out=[z(4, dt=torch.float16)]),
        lambda: clip_grad_norm([z(4, 6)], 1.0, out=[z(6, 4).t()]), lambda: clip_grad_norm([z(4)], -1.0),
        lambda: clip_grad_norm([z(4)], float("nan")), lambda: ops.grad_clip([z(4)], z(1, dt=f32), 1.0),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            f()
            print("accepted:", i)
