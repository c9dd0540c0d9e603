"""The operators around the block launch under the device of their tensors where another one is current, and refuse operands on
different devices (one GPU: which device is current is made up, and the CPU is the other one)."""
import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_launched_under_the_device_of_the_tensors(monkeypatch):
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm, ops
    x = torch.randn(16, 64, device="cuda").bfloat16()
    lg, ids = torch.randn(16, 8, device="cuda"), torch.zeros(16, 2, device="cuda", dtype=torch.int32)
    w = torch.ones(16, 2, device="cuda")
    calls = [lambda: ops.norm_modulate(x), lambda: ops.norm_modulate_bwd(x, x), lambda: ops.norm_residual(x, x),
             lambda: ops.norm_residual_bwd(x, x), lambda: ops.route_scores(lg, 2),
             lambda: ops.route_scores_bwd(w, w, lg, ids), lambda: ops.router_wgrad(lg, x), lambda: clip_grad_norm([w], 1e9)]
    entered = []

    @contextlib.contextmanager
    def device(d):
        entered.append(d)
        yield

    monkeypatch.setattr(ops, "_current_device", lambda: 7)
    monkeypatch.setattr(torch.cuda, "device", device)
    for i, f in enumerate(calls):
        entered.clear()
        f()
        assert entered and all(d == x.device for d in entered), i


def test_router_wgrad_refuses_other_devices():
    from trenowanie_generatora_obrazkow_amd import ops
    x, dl = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(4, 8, device="cuda")
    for f in (lambda: ops.router_wgrad(dl.cpu(), x), lambda: ops.router_wgrad(dl, x.cpu()), lambda: ops.router_wgrad(dl[:3], x),
              lambda: ops.router_wgrad(dl.bfloat16(), x), lambda: ops.router_wgrad(dl.t().contiguous().t(), x)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            f()
    assert not ops.router_wgrad(dl, x).any()
