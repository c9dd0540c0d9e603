"""Clipping refuses lists in which a tensor to be written lies over another one, before anything is launched (the GPU's workgroups
would race).  CPU only: the C entry with stand-in addresses, which are compared and never dereferenced."""
import ctypes

import pytest

BF, HF, FP = 0, 1, 2
OVERLAP = -8
SQ, A = 1 << 20, 1 << 30


@pytest.fixture(scope="module")
def clip():
    from trenowanie_generatora_obrazkow_amd import _lib

    def f(grads, outs=None):
        """grads, outs: (address, elements, type)"""
        n = len(grads)
        outs = grads if outs is None else outs
        arr = lambda t, v: (t * n)(*v)
        return _lib.lib().hmoe_grad_clip(arr(ctypes.c_void_p, [g[0] for g in grads]), arr(ctypes.c_void_p, [o[0] for o in outs]),
                                         arr(ctypes.c_int64, [g[1] for g in grads]), arr(ctypes.c_int, [g[2] for g in grads]),
                                         arr(ctypes.c_int, [o[2] for o in outs]), n, SQ, 1.0, None, None)
    return f


@pytest.mark.parametrize("grads,outs", [
    ([(A, 100, BF)], [(A, 100, FP)]),                                        # its own gradient, in another type
    ([(A, 100, FP)], [(A + 4, 100, FP)]),                                    # its own gradient, an element on
    ([(A, 100, BF)], [(A + 196, 100, FP)]),                                  # the gradient's last two elements
    ([(A + 398, 100, BF)], [(A, 100, FP)]),                                  # the output's last element
    ([(A, 100, FP), (A + 4000, 100, FP)], [(A + 8000, 100, FP), (A + 396, 100, FP)]),   # inside another gradient
    ([(A, 100, FP), (A + 4000, 100, FP)], [(A + 8000, 100, FP), (A + 8396, 100, FP)]),  # inside another output
    ([(A, 100, FP), (A + 396, 100, FP)], None),                              # gradients in place, one element shared
    ([(A, 1000, FP), (A + 400, 10, BF)], None),                              # one inside the other
    ([(A + 4000, 1000, FP), (A, 1000, HF), (A + 1996, 10, BF)], None),       # not in the order of their addresses
    ([(A, 5000, FP), (A + 100, 1, FP), (A + 15000, 1, FP)], [(A + 30000, 5000, FP), (A + 60000, 1, FP), (A + 15000, 1, FP)]),
    ([(A, 100, FP), (A, 100, FP)], None),                                    # one twice
    ([(A + 8 * i, 2, FP) for i in range(700)] + [(A + 796, 1, FP)], None),   # many
])
def test_refused(clip, grads, outs):
    assert clip(grads, outs) == OVERLAP


def test_text():
    from trenowanie_generatora_obrazkow_amd import _lib
    assert _lib.ERR_OVERLAP == OVERLAP and "over another" in _lib.lib().hmoe_error_string(OVERLAP).decode()
