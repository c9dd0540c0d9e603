"""Refusals of the 8-bit experts: the C entry points' argument codes (no kernel is launched on these paths), the Python
wrappers on CPU tensors, and the definition's reference against torch's own conversion.  CPU only."""
import pytest
import torch

import f8_ref as R

P = 4096  # a non-null stand-in address: never dereferenced
BF, HF, FP, I32, I64, I8 = 0, 1, 2, 3, 4, 5
ARG, SHAPE, DTYPE, WORKSPACE = -1, -2, -3, -5


@pytest.fixture(scope="module")
def L():
    from trenowanie_generatora_obrazkow_amd import _lib
    return _lib.lib()


def test_scale_ld(L):
    from trenowanie_generatora_obrazkow_amd import ops
    for K in (16, 128, 2048, 2064, 4096, 10000):
        assert L.hmoe_f8_scale_ld(K) == ops._f8_ld(K) and L.hmoe_f8_scale_ld(K) % 16 == 0
        assert L.hmoe_f8_scale_ld(K) >= -(-K // 128)
    assert L.hmoe_f8_scale_ld(0) == 0


def test_quant_rows_codes(L):
    def f(x=P, ldx=64, dt=BF, M=4, K=64, q=P, ldq=64, s=P, lds=16):
        return L.hmoe_f8_quant_rows(x, ldx, dt, M, K, q, ldq, s, lds, None)
    assert f(M=0) == 0 and f(M=-1) == ARG and f(K=0) == ARG and f(dt=I8) == DTYPE
    assert f(x=None) == ARG and f(q=None) == ARG and f(s=None) == ARG
    assert f(K=72, ldx=80, ldq=80) == SHAPE
    assert f(ldx=56) == ARG and f(ldx=68) == ARG and f(ldq=48) == ARG and f(ldq=72) == ARG and f(lds=8) == ARG and f(lds=24) == ARG
    assert f(x=P + 8) == ARG and f(q=P + 8) == ARG and f(s=P + 8) == ARG


def test_dequant_rows_codes(L):
    def f(q=P, ldq=64, s=P, lds=16, M=4, K=64, block=128, x=P, ldx=64, dt=BF):
        return L.hmoe_f8_dequant_rows(q, ldq, s, lds, M, K, block, x, ldx, dt, None)
    assert f(M=0) == 0 and f(M=-1) == ARG and f(dt=I32) == DTYPE and f(block=64) == SHAPE and f(K=60) == SHAPE
    assert f(block=32, lds=1) == ARG and f(ldx=56) == ARG and f(x=None) == ARG and f(x=P + 8) == ARG and f(q=P + 4) == ARG


def test_quant_stack_codes(L):
    def f(w=P, dt=BF, E=2, K=64, N=96, se=64 * 96, sk=96, halves=1, tr=1, q=P, s=P):
        return L.hmoe_f8_quant_stack(w, dt, E, K, N, se, sk, halves, tr, q, s, None)
    assert f(E=0) == ARG and f(K=0) == ARG and f(halves=3) == ARG and f(halves=2, N=96 + 1) == ARG and f(dt=I8) == DTYPE
    assert f(K=72) == SHAPE and f(N=88) == SHAPE and f(halves=2, N=80) == SHAPE and f(E=2000) == SHAPE
    assert f(halves=2, tr=0) == SHAPE
    assert f(w=None) == ARG and f(sk=88) == ARG and f(sk=100) == ARG and f(se=100) == ARG and f(w=P + 8) == ARG and f(q=P + 8) == ARG


def test_grouped_mm_codes(L):
    def f(a=P, lda=64, a_s=P, ld_s=16, w=P, w_s=P, E=2, K=64, N=96, halves=1, c=P, cdt=I32, M=4, ai=None, sc=None, sdt=FP, y=P,
          ldy=96, ydt=BF, rows=None):
        return L.hmoe_f8_grouped_mm(a, lda, a_s, ld_s, M if rows is None else rows, w, w_s, E, K, N, halves, c, cdt, M, ai, None, sc, sdt, 0, y, ldy, ydt,
                                    None)
    assert f(M=0) == 0 and f(M=-1) == ARG and f(E=0) == ARG and f(c=None) == ARG and f(cdt=FP) == DTYPE
    assert f(E=1025) == SHAPE and f(M=2 ** 31) == SHAPE and f(ydt=I8) == DTYPE and f(sc=P, sdt=I32) == DTYPE
    assert f(a=None) == ARG and f(a_s=None) == ARG and f(w=None) == ARG and f(w_s=None) == ARG and f(y=None) == ARG
    assert f(K=72, lda=80) == SHAPE and f(N=104, ldy=104) == SHAPE and f(N=80, halves=2) == SHAPE and f(halves=3) == ARG
    assert f(lda=48) == ARG and f(lda=72) == ARG and f(ld_s=8) == ARG and f(ldy=88) == ARG and f(ldy=100) == ARG
    assert f(a=P + 8) == ARG and f(a_s=P + 4) == ARG and f(w=P + 8) == ARG and f(w_s=P + 8) == ARG and f(y=P + 8) == ARG
    assert f(K=1 << 16, lda=1 << 16, ld_s=512, N=1 << 15, ldy=1 << 15) == SHAPE  # one expert's weights past 2 GiB
    assert f(rows=1 << 26, ai=P) == SHAPE                                        # gathered rows past 2 GiB
    assert f(rows=3) == ARG and f(rows=0, ai=P) == ARG


def test_quant_mm_codes(L):
    n = L.hmoe_f8_quant_mm_workspace_size(4, 64)
    assert n >= 4 * (64 + 16) and L.hmoe_f8_quant_mm_workspace_size(-1, 64) == 0

    def f(x=P, ldx=64, dt=BF, rows=4, w=P, K=64, N=96, halves=1, cdt=I32, M=4, sc=None, sdt=FP, y=P, ldy=96, ydt=BF, ws=P, n=n):
        return L.hmoe_f8_quant_mm(x, ldx, dt, rows, w, P, 2, K, N, halves, P, cdt, M, None, None, sc, sdt, 0, y, ldy, ydt, ws, n, None)
    assert f(M=0) == 0 and f(rows=-1) == ARG and f(M=-1) == ARG and f(rows=3) == ARG and f(x=None) == ARG and f(w=None) == ARG
    assert f(ws=None) == WORKSPACE and f(n=n - 1) == WORKSPACE and f(ws=P + 8) == WORKSPACE
    assert f(dt=I8) == DTYPE and f(ydt=I8) == DTYPE and f(sc=P, sdt=I32) == DTYPE and f(cdt=FP) == DTYPE
    assert f(K=72, n=1 << 20) == SHAPE and f(N=104, ldy=104) == SHAPE and f(ldy=88) == ARG and f(y=P + 8) == ARG and f(ldx=68) == ARG


def test_gate_up_codes(L):
    def f(x=P, M=4, d=64, h=48, act=P, act_s=P, E=2):
        return L.hmoe_f8_gate_up_swiglu(x, d, P, 16, M, None, P, P, E, d, h, P, I32, M, 0, act, act_s, None)
    assert f(M=0) == 0 and f(h=0) == ARG and f(h=40) == SHAPE and f(act=None) == ARG and f(act_s=None) == ARG and f(act=P + 8) == ARG


def test_moe_experts_codes(L):
    n = L.hmoe_f8_moe_experts_workspace_size(4, 64, 3, 2, 48)
    assert n > 0 and L.hmoe_f8_moe_experts_workspace_size(-1, 64, 3, 2, 48) == 0

    def f(x=P, ldx=64, dt=BF, ids=P, wdt=FP, T=4, d=64, E=3, k=2, h=48, y=P, ws=P, n=n):
        return L.hmoe_f8_moe_experts(x, ldx, dt, ids, I32, P, wdt, P, P, P, P, T, d, E, k, h, y, P, P, ws, n, None)
    assert f(dt=FP) == DTYPE and f(wdt=I32) == DTYPE and f(ws=None) == WORKSPACE and f(n=n - 1) == WORKSPACE
    assert f(ws=P + 8) == WORKSPACE and f(x=None) == ARG and f(ids=None) == ARG and f(y=None) == ARG and f(ldx=56) == ARG
    assert f(ldx=68) == ARG and f(x=P + 8) == ARG and f(k=0) == ARG
    big = L.hmoe_f8_moe_experts_workspace_size(4, 72, 3, 2, 48)
    assert f(d=72, ldx=72, n=big) == SHAPE
    big = L.hmoe_f8_moe_experts_workspace_size(4, 64, 3, 2, 40)
    assert f(h=40, n=big) == SHAPE


def test_cpu_tensors_are_refused():
    from trenowanie_generatora_obrazkow_amd import F8Stack, ops
    from trenowanie_generatora_obrazkow_amd.moe_triton import grouped_mm
    w, x = torch.zeros(2, 32, 32, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        F8Stack.from_weights(w)
    with pytest.raises(RuntimeError):
        ops.quant_rows(x)
    st = F8Stack(torch.zeros(2, 32, 32).to(torch.float8_e4m3fn), torch.zeros(2, 1, 16, dtype=torch.uint8).view(torch.float8_e8m0fnu))
    with pytest.raises((RuntimeError, ValueError)):
        grouped_mm(x, st, torch.tensor([2, 2]))
    with pytest.raises(ValueError, match="own scales"):
        grouped_mm(x, st, torch.tensor([2, 2]), w_scale=torch.ones(2, 32))
    with pytest.raises(ValueError, match="grad=True"):
        grouped_mm(x.requires_grad_(True), st, torch.tensor([2, 2]))
    with pytest.raises(ValueError, match="sorted rows"):
        grouped_mm(x, st, torch.tensor([2, 2]), a_idx=torch.arange(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="own scales"):
        ops.moe_experts(x, torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, 1), st, st, wgu_s=torch.ones(2, 32))


def test_reference_against_torch():
    """The definition's rounding is torch's conversion of the scaled values; its scale is the least one that holds them."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 300, generator=g) * torch.exp(3 * torch.randn(40, 300, generator=g))
    q, e = R.quant(x)
    for j in range(3):
        b, s = x[:, 128 * j:128 * j + 128], torch.exp2(e[:, j].float())[:, None]
        assert torch.equal((b / s).to(torch.float8_e4m3fn).double() * s, q[:, 128 * j:128 * j + 128])
        top = b.abs().amax(1, keepdim=True)
        assert (top <= 448 * s).all() and (top > 224 * s).all()


def test_pack_codes(L):
    def f(gu=P, ld=128, M=4, h=64, act=P, q=P, s=P, dt=BF):
        return L.hmoe_swiglu_pack(gu, ld, M, h, act, q, s, dt, None)
    assert f(M=0) == 0 and f(M=-1) == ARG and f(h=0) == ARG and f(h=60) == SHAPE and f(dt=FP) == DTYPE
    assert f(gu=None) == ARG and f(act=None) == ARG and f(q=None) == ARG and f(s=None) == ARG
    assert f(ld=120) == ARG and f(ld=132) == ARG and f(gu=P + 8) == ARG and f(act=P + 8) == ARG and f(q=P + 4) == ARG

    def b(dh=P, q=P, s=P, w=P, wdt=FP, M=4, h=64, dgu=P, act=P, dt=BF):
        return L.hmoe_swiglu_pack_bwd(dh, q, s, w, wdt, M, h, dgu, act, None, P, dt, None)
    assert b(M=0) == 0 and b(h=60) == SHAPE and b(dt=FP) == DTYPE and b(wdt=I32) == DTYPE
    assert b(dh=None) == ARG and b(q=None) == ARG and b(s=None) == ARG and b(dgu=None) == ARG
    assert b(dh=P + 8) == ARG and b(dgu=P + 8) == ARG and b(act=P + 8) == ARG and b(q=P + 4) == ARG


def test_down_dgrad_codes(L):
    def f(dy=P, wd=P, E=2, h=64, d=32, c=P, cdt=I32, M=4, dh=P):
        return L.hmoe_down_dgrad(dy, None, wd, E, h, d, c, cdt, M, dh, None)
    assert f(M=0) == 0 and f(dy=None) == ARG and f(wd=None) == ARG and f(dh=None) == ARG and f(c=None) == ARG
    assert f(h=60) == SHAPE and f(d=36) == SHAPE and f(cdt=FP) == DTYPE and f(dh=P + 8) == ARG


def test_pack_wrappers():
    from trenowanie_generatora_obrazkow_amd import MoESwiGLU, moe_swiglu, ops
    with pytest.raises((RuntimeError, ValueError)):
        ops.swiglu_pack(torch.zeros(2, 16, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="checkpoint"):
        MoESwiGLU(16, 16, 2, checkpoint="int8")
    with pytest.raises(ValueError, match="checkpoint"):
        moe_swiglu(torch.zeros(2, 16, dtype=torch.bfloat16), None, None, None, 1, checkpoint="bf16")


def test_few_codes(L):
    n = L.hmoe_few_workspace_size(4, 64, 3, 2, 48, BF, BF)
    assert n > 0 and L.hmoe_few_workspace_size(17, 64, 3, 2, 48, BF, BF) == 0 and L.hmoe_few_workspace_size(4, 64, 3, 2, 48, HF, BF) == 0
    P2 = 1 << 16  # 256-byte aligned

    def f(x=P, ldx=64, dt=BF, ids=P, idt=I32, tw=P, twdt=FP, w1=P, s1=None, sdt=BF, w2=P, s2=None, wdt=BF, T=4, d=64, E=3, k=2,
          h=48, add=None, out=P, ws=P2, n=1 << 24):
        return L.hmoe_few_experts(x, ldx, dt, ids, idt, tw, twdt, w1, s1, sdt, w2, s2, sdt, wdt, T, d, E, k, h, add, out, None, ws, n, None)
    assert f(T=0) == 0 and f(T=-1) == ARG and f(d=0) == ARG and f(k=0) == ARG
    assert f(dt=FP) == DTYPE and f(wdt=HF) == DTYPE and f(dt=HF, wdt=BF) == DTYPE and f(idt=FP) == DTYPE and f(twdt=I32) == DTYPE
    assert f(wdt=I8) == ARG and f(s1=P) == ARG and f(wdt=I8, s1=P, s2=P, sdt=HF) == DTYPE and f(wdt=6) == ARG
    assert f(T=17) == SHAPE and f(k=17) == SHAPE and f(E=1025) == SHAPE and f(d=60, ldx=64) == SHAPE and f(h=44) == SHAPE
    assert f(wdt=I8, s1=P, s2=P, h=40) == SHAPE
    assert f(x=None) == ARG and f(ids=None) == ARG and f(tw=None) == ARG and f(w1=None) == ARG and f(w2=None) == ARG and f(out=None) == ARG
    assert f(ldx=56) == ARG and f(ldx=68) == ARG and f(x=P + 8) == ARG and f(out=P + 8) == ARG and f(add=P + 8) == ARG and f(w1=P + 8) == ARG
    assert f(ws=None) == WORKSPACE and f(n=n - 1) == WORKSPACE and f(ws=P2 + 64) == WORKSPACE

    def g(wr=P, ids=P, tw=P, k=2, E=3, n=1 << 24):
        return L.hmoe_few_forward(P, 64, wr, None, P, P, 4, 64, E, k, 48, 1, 1.0, None, P, ids, tw, P2, n, None)
    assert g(wr=None) == ARG and g(ids=None) == ARG and g(tw=None) == ARG and g(k=4) == SHAPE and g(E=300, n=1 << 28) == SHAPE
    assert g(n=16) == WORKSPACE


def test_few_wrappers():
    from trenowanie_generatora_obrazkow_amd import ops
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.few_experts(x, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1), torch.zeros(1, 64, 32, dtype=torch.bfloat16),
                        torch.zeros(1, 16, 64, dtype=torch.bfloat16))


def test_pack_launch_limit(L):
    """A workgroup per row: 2^25 rows would be 2^33 threads, more than a launch takes."""
    assert L.hmoe_swiglu_pack(P, 8192, 1 << 25, 4096, P, P, P, BF, None) == SHAPE
    assert L.hmoe_swiglu_pack_bwd(P, P, P, P, FP, 1 << 25, 4096, P, P, None, P, BF, None) == SHAPE
