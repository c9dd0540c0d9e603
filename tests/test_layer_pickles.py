"""Modules pickled whole before the layer had gates and a selection bias load as plain softmax layers; newer ones keep both.
CPU only."""
import copy
import pickle

import torch


def test_module_without_the_newer_attributes():
    from trenowanie_generatora_obrazkow_amd import MoESwiGLU
    m = MoESwiGLU(16, 16, 4, 2)
    state = {k: v for k, v in m.__dict__.items() if k not in ("gate", "select_bias")}
    old = MoESwiGLU.__new__(MoESwiGLU)
    old.__setstate__(state)
    assert old.gate is None and old.select_bias is None
    assert set(old.state_dict()) == set(m.state_dict())


def test_round_trips():
    from trenowanie_generatora_obrazkow_amd import Gate, MoESwiGLU
    m = MoESwiGLU(16, 16, 4, 2, gate=Gate("sigmoid", 2, 1), balance=True)
    m.select_bias[1] = 3.0
    for n in (pickle.loads(pickle.dumps(m)), copy.deepcopy(m)):
        assert n.gate == m.gate and torch.equal(n.select_bias, m.select_bias) and "select_bias" in n.state_dict()
    n = copy.deepcopy(MoESwiGLU(16, 16, 4, 2))
    assert n.gate is None and n.select_bias is None
