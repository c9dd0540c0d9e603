"""Refusals of the clipping entry with an fp64 bound.  CPU only: nothing is launched on these paths."""
import ctypes
import math


def test_bounds_and_lists():
    from trenowanie_generatora_obrazkow_amd import _lib
    P = 1 << 20
    one = lambda t, v: (t * 1)(v)
    p, o = one(ctypes.c_void_p, P), one(ctypes.c_void_p, P + 4096)
    num, bf, fp = one(ctypes.c_int64, 8), one(ctypes.c_int, 0), one(ctypes.c_int, 2)
    f = lambda mx=1.0, sq=P + 64, out=o, odt=fp, n=1: _lib.lib().hmoe_grad_clip_f64(p, out, num, bf, odt, n, sq, mx, None, None)
    assert f(mx=-1e-300) == -1 and f(mx=math.nan) == -1 and f(mx=-math.inf) == -1  # (rounded to fp32 the first is -0)
    assert f(sq=None) == -1 and f(out=None) == -1 and f(odt=None) == -1 and f(n=-1) == -1
    assert f(odt=one(ctypes.c_int, 1)) == -3 and f(out=p) == -8
