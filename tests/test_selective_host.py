"""Selective state space models on the host: their model files, plans and refusals."""
import os

import numpy as np
import pytest
import torch
from torch import nn

from rosenna_b200 import api, selective, writer


def write(d, layers=1, width=12, T=7, eight_bit=False, with_state=True, mode="last", head=True, **kw):
    torch.manual_seed(3)
    mods = [selective.SelectiveLayer(width, **kw) for _ in range(layers)]
    hd = [nn.Linear(width, 5), nn.Tanh()] if head and mode == "last" else []
    writer.write_model_files(selective.export_selective(mods, hd, 1, T, mode, with_state, eight_bit), str(d))
    return mods, hd


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("mode,with_state", [("last", True), ("last", False), ("y", True), ("y", False)])
def test_plan_runs_the_operators(tmp_path, eight_bit, mode, with_state):
    write(tmp_path, 2, eight_bit=eight_bit, mode=mode, with_state=with_state)
    desc = api.check_model(str(tmp_path))
    lines = desc.splitlines()
    assert sum(x.startswith("causal_conv") for x in lines) == 2 and sum(x.startswith("scan") for x in lines) == 2, desc
    assert sum(x.startswith("gemm8") for x in lines) == (8 if eight_bit else 0), desc
    # operands are read where they lie: the only moved rows are the last step's
    assert sum(x.startswith("gather") for x in lines) == (1 if mode == "last" else 0), desc
    assert "deinterleave" not in desc, desc


def test_unread_states_are_not_computed(tmp_path):
    write(tmp_path, with_state=False)
    desc = api.check_model(str(tmp_path))
    assert "state b-1->b-1" in desc, desc


def test_layer_step_by_step_equals_the_whole():
    torch.manual_seed(0)
    ly = selective.SelectiveLayer(6, states=5, taps=3).double()
    x = torch.randn(4, 9, 6, dtype=torch.float64)
    y, cs, hs = ly(x)
    c = h = None
    for t in range(9):
        yt, c, h = ly(x[:, t:t + 1], c, h)
        assert torch.allclose(yt[:, 0], y[:, t], atol=1e-12)
    assert torch.allclose(c, cs, atol=1e-12) and torch.allclose(h, hs, atol=1e-12)
    ly(x)[0].sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in ly.parameters())


def broken(d, old, new, file="variables.fpp"):
    p = os.path.join(str(d), file)
    with open(p) as f:
        text = f.read()
    assert old in text, (old, text)
    with open(p, "w") as f:
        f.write(text.replace(old, new, 1))
    with pytest.raises(api.RosennaError) as e:
        api.check_model(str(d))
    return e.value.code


@pytest.mark.parametrize("old,new,code", [
    ("[0, 4])", "[99, 4])", api.ERR_SHAPE),            # the convolution's features lie outside its operand
    ("[0, 4])", "[-1, 4])", api.ERR_SHAPE),
    ("[0, 4])", "[0, 2])", api.ERR_UNSUPPORTED),       # an activation it has not
    ("[0, 4])", "[0])", api.ERR_FORMAT),
    (", 24, 1, 1])", ", 24, 5, 1])", api.ERR_SHAPE),   # groups that do not divide the channels
    (", 24, 1, 1])", ", 25, 1, 1])", api.ERR_SHAPE),   # the gate's features
    (", 24, 1, 1])", ", 24, 1])", api.ERR_FORMAT),
    ("'scan_state0']", "'conv_state0']", api.ERR_SHAPE),
    ("'SelectiveScan'", "'Scan'", api.ERR_UNSUPPORTED),
])
def test_malformed_entries_are_refused(tmp_path, old, new, code):
    write(tmp_path, head=False)
    assert broken(tmp_path, old, new) == code


def test_gemm8_entries_are_refused(tmp_path):
    for k, (old, new, code) in enumerate([("('Gemm8', ['input'], ['output0'], [0, 0])", "('Gemm8', ['input'], ['output0'], [1, 0])", api.ERR_SHAPE),
                                          ("('Gemm8', ['input'], ['output0'], [0, 0])", "('Gemm8', ['input'], ['output0'], [0, 9])", api.ERR_FORMAT)]):
        d = tmp_path / str(k)
        write(d, head=False, eight_bit=True)
        assert broken(d, old, new) == code
    d = tmp_path / "inf"
    write(d, head=False, eight_bit=True)
    with open(d / "onnxWeights.txt") as f:
        first = f.readline().split(" ")[0]
    assert broken(d, first, "inf", "onnxWeights.txt") == api.ERR_FORMAT


def test_operator_weights_are_checked_before_the_gpu():
    def code(f):
        with pytest.raises(api.RosennaError) as e:
            f()
        return e.value.code

    z = np.zeros
    assert code(lambda: api.CausalConv(z((3, 9), np.float32))) == api.ERR_UNSUPPORTED
    assert code(lambda: api.SelectiveScan(z((3, 65), np.float32))) == api.ERR_UNSUPPORTED
    assert code(lambda: api.SelectiveScan(z((3, 4), np.float32), groups=2)) == api.ERR_SHAPE
    assert code(lambda: api.Gemm8(np.full((2, 2), np.inf, np.float32))) == api.ERR_ARG
    for bad in (lambda: api.CausalConv(z((3, 4), np.float32), bias=z(2)), lambda: api.CausalConv(z((3, 4), np.float32), act="relu"),
                lambda: api.SelectiveScan(z((3, 4)), skip=z(4)), lambda: api.Gemm8(z((3, 4)), act="gelu"), lambda: api.Gemm8(z(3))):
        with pytest.raises(ValueError):
            bad()
    if not torch.cuda.is_available():
        assert code(lambda: api.CausalConv(z((3, 4), np.float32))) == api.ERR_NO_DEVICE
