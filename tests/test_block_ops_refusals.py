"""Refusals of the norms, routing from logits and gradient clipping: the C entry points' argument codes (no kernel is launched
on these paths) and the Python wrappers on CPU tensors.  CPU only."""
import ctypes
import math

import pytest
import torch

P = 4096  # a non-null stand-in address: never dereferenced
BF, HF, FP, I32 = 0, 1, 2, 3
ARG, SHAPE, DTYPE, WORKSPACE = -1, -2, -3, -5


@pytest.fixture(scope="module")
def L():
    from trenowanie_generatora_obrazkow_amd import _lib
    return _lib.lib()


def test_norm_modulate_codes(L):
    def f(x=P, ldx=64, xdt=BF, w=P, wdt=BF, sc=P, sh=P, mdt=FP, starts=None, B=2, T=4, d=64, h=P, hdt=BF):
        return L.hmoe_norm_modulate(x, ldx, xdt, w, wdt, sc, sh, mdt, starts, B, T, d, 1e-6, h, hdt, None)
    assert f(T=0) == 0
    assert f(T=-1) == ARG and f(d=0) == ARG and f(B=0) == ARG
    assert f(x=None) == ARG and f(h=None) == ARG
    assert f(d=60) == SHAPE and f(d=16392, ldx=16392) == SHAPE and f(T=1 << 31) == SHAPE
    assert f(T=5) == SHAPE                      # rows that do not divide into the samples
    assert f(T=5, starts=P, x=P + 8) == ARG     # (with starts they need not: the next check is reached)
    assert f(ldx=56) == ARG and f(ldx=68) == ARG
    assert f(x=P + 2) == ARG and f(h=P + 8) == ARG and f(w=P + 4) == ARG and f(sc=P + 8) == ARG and f(sh=P + 8) == ARG
    assert f(xdt=BF, hdt=FP) == DTYPE and f(xdt=BF, hdt=HF) == DTYPE and f(xdt=I32) == DTYPE
    assert f(wdt=I32) == DTYPE and f(mdt=5) == DTYPE


def test_norm_modulate_bwd_codes(L):
    T, d, B = 4, 64, 2
    n = L.hmoe_norm_modulate_bwd_workspace_size(T, d, B)
    assert n > 0 and L.hmoe_norm_modulate_bwd_workspace_size(-1, d, B) == 0

    def f(dh=P, hdt=BF, x=P, ldx=64, xdt=BF, w=P, sc=P, sh=P, T=T, d=d, B=B, dres=None, dx=P, dw=P, dsc=P, dsh=P, ws=P, n=n):
        return L.hmoe_norm_modulate_bwd(dh, hdt, x, ldx, xdt, w, BF, sc, sh, FP, None, B, T, d, 1e-6, dres, 1.0, dx, dw, dsc,
                                        dsh, ws, n, None)
    assert f(ws=None) == WORKSPACE and f(n=16) == WORKSPACE and f(ws=P + 8) == ARG
    assert f(dh=None) == ARG and f(x=None) == ARG and f(dx=None) == ARG and f(dres=P + 2) == ARG
    assert f(w=None) == ARG and f(sc=None) == ARG and f(sh=None) == ARG  # a gradient of a parameter that is not there
    assert f(dw=P + 2) == ARG and f(dsc=P + 2) == ARG and f(dsh=P + 2) == ARG
    assert f(d=68) == SHAPE and f(T=3) == SHAPE and f(xdt=HF) == DTYPE


def test_norm_residual_codes(L):
    def f(y=P, k=2, add=None, ydt=BF, x=P, ldx=64, xdt=BF, w=P, gate=P, gdt=BF, B=2, T=4, d=64, out=P):
        return L.hmoe_norm_residual(y, None, k, add, ydt, x, ldx, xdt, w, BF, gate, gdt, None, B, T, d, 1, 1e-6, 1.0, out,
                                    None)
    assert f(T=0) == 0 and f(T=0, k=0) == ARG
    assert f(k=0) == ARG and f(y=None) == ARG and f(x=None) == ARG and f(out=None) == ARG
    assert f(y=P + 8) == ARG and f(add=P + 8) == ARG and f(out=P + 4) == ARG and f(gate=P + 2) == ARG and f(ldx=60) == ARG
    assert f(ydt=HF) == DTYPE and f(ydt=FP) == DTYPE and f(gdt=4) == DTYPE
    assert f(d=12) == SHAPE and f(T=3) == SHAPE
    n = L.hmoe_norm_residual_bwd_workspace_size(4, 64, 2)

    def b(dout=P, odt=BF, y=P, k=2, w=P, gate=P, dy=P, dw=P, dg=P, ws=P, n=n):
        return L.hmoe_norm_residual_bwd(dout, odt, y, None, k, None, BF, w, BF, gate, BF, None, 2, 4, 64, 1, 1e-6, dy, dw, dg,
                                        ws, n, None)
    assert b(ws=None) == WORKSPACE and b(n=8) == WORKSPACE
    assert b(dout=None) == ARG and b(y=None) == ARG and b(dy=None) == ARG and b(k=0) == ARG
    assert b(w=None) == ARG and b(gate=None) == ARG and b(dy=P + 2) == ARG and b(odt=HF) == DTYPE


def test_route_scores_codes(L):
    def f(lg=P, ld=64, dt=FP, T=4, E=64, k=4, score=1, ng=8, tg=2, gt=2, ids=P, w=P):
        return L.hmoe_route_scores(lg, ld, dt, None, None, T, E, k, score, ng, tg, gt, 1, 1.0, ids, w, None)
    assert f(T=0) == 0 and f(T=0, ids=None, w=None) == 0
    assert f(lg=None) == ARG and f(ids=None) == ARG and f(w=None) == ARG and f(ld=63) == ARG and f(T=-1) == ARG
    assert f(score=2) == ARG and f(k=0) == ARG
    assert f(dt=I32) == DTYPE
    assert f(E=513, ld=513, ng=1, tg=1) == SHAPE and f(k=17) == SHAPE and f(E=3, k=4, ng=1, tg=1) == SHAPE
    assert f(ng=7) == SHAPE and f(tg=9) == SHAPE and f(tg=0) == SHAPE and f(gt=3) == SHAPE
    assert f(ng=64, tg=8, gt=2) == SHAPE          # one expert per group, its two best asked for
    assert f(ng=32, tg=1, k=3) == SHAPE           # two experts in the kept group
    assert f(E=512, ld=512, ng=128, tg=8, gt=1) == SHAPE

    def b(dw=P, w=P, lg=P, ids=P, dl=P, T=4, E=64, k=4):
        return L.hmoe_route_scores_bwd(dw, w, lg, 64, FP, ids, T, E, k, 0, 1, 1.0, dl, None)
    assert b(T=0) == 0
    assert b(dw=None) == ARG and b(w=None) == ARG and b(lg=None) == ARG and b(ids=None) == ARG and b(dl=None) == ARG
    assert b(E=65) == ARG and b(k=17) == SHAPE


def test_router_wgrad_codes(L):
    n = L.hmoe_router_bwd_workspace_size(4, 8, 64)

    def f(dl=P, x=P, ldx=64, E=8, d=64, dwr=P, dt=FP, ws=P, n=n):
        return L.hmoe_router_wgrad(dl, x, ldx, 4, E, d, dwr, dt, ws, n, None)
    assert f(ws=None) == WORKSPACE and f(n=n - 1) == WORKSPACE
    assert f(dl=None) == ARG and f(x=None) == ARG and f(dwr=None) == ARG and f(x=P + 2) == ARG and f(ldx=60) == ARG
    assert f(E=257) == SHAPE and f(dt=HF) == DTYPE


def test_clip_codes(L):
    ptr, num, dts = (ctypes.c_void_p * 2)(P, P), (ctypes.c_int64 * 2)(8, 8), (ctypes.c_int * 2)(BF, FP)
    n = L.hmoe_grad_sq_norm_workspace_size(2)
    assert L.hmoe_grad_sq_norm_workspace_size(-1) == 0
    norm = lambda p=ptr, m=num, d=dts, c=2, sq=P, ws=P, n=n: L.hmoe_grad_sq_norm(p, m, d, c, sq, ws, n, None)
    assert norm(p=None) == ARG and norm(m=None) == ARG and norm(d=None) == ARG and norm(c=-1) == ARG and norm(sq=None) == ARG
    assert norm(ws=None) == WORKSPACE and norm(n=n - 1) == WORKSPACE and norm(ws=P + 4) == ARG
    assert norm(d=(ctypes.c_int * 2)(BF, I32)) == DTYPE
    assert norm(m=(ctypes.c_int64 * 2)(8, -1)) == ARG
    assert norm(p=(ctypes.c_void_p * 2)(P, None)) == ARG
    assert norm(p=(ctypes.c_void_p * 2)(P, P + 2)) == ARG       # an fp32 tensor off its element
    assert norm(m=(ctypes.c_int64 * 2)(8, 1 << 60)) == SHAPE
    clip = lambda o=ptr, od=dts, c=2, sq=P, mx=1.0: L.hmoe_grad_clip(ptr, o, num, dts, od, c, sq, mx, P, None)
    assert clip(o=None) == ARG and clip(od=None) == ARG and clip(sq=None) == ARG
    assert clip(mx=-1.0) == ARG and clip(mx=math.nan) == ARG
    assert clip(od=(ctypes.c_int * 2)(HF, FP)) == DTYPE and clip(od=(ctypes.c_int * 2)(BF, BF)) == DTYPE


def test_cpu_tensors_are_refused():
    from trenowanie_generatora_obrazkow_amd import clip_grad_norm, ops
    x = torch.zeros(4, 64)
    for f in (lambda: ops.norm_modulate(x), lambda: ops.norm_modulate_bwd(x, x), lambda: ops.norm_residual(x, x),
              lambda: ops.norm_residual_bwd(x, x), lambda: ops.route_scores(x, 2),
              lambda: ops.route_scores_bwd(x[:, :2], x[:, :2], x, x[:, :2].int()), lambda: clip_grad_norm([x], 1.0)):
        with pytest.raises(RuntimeError, match="GPU"):
            f()
