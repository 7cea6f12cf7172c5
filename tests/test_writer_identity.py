"""An ONNX Identity passes its input's name through (modelParserONNX.py:519-523): no entry, no step, no copy."""
import os

import numpy as np

from rosenna_b200 import api, writer


def graph(identity, value_info=True):
    b = writer._Builder()
    f = lambda *s: np.arange(np.prod(s), dtype=np.float32).reshape(s)  # noqa: E731

    def same(v, shape):
        if not identity:
            return v
        o = b.add("Identity", [v], [shape])[0]
        if not value_info:
            del b.vi[o]
        return o

    x = same("input", [1, 5])
    h = same(b.add("Gemm", [x, b.weight(f(8, 5)), b.weight(f(8))], [[1, 8]], {"transB": 1})[0], [1, 8])
    h = same(b.add("Relu", [h], [[1, 8]])[0], [1, 8])
    y = b.add("Gemm", [h, b.weight(f(4, 8)), b.weight(f(4))], [[1, 4]], {"transB": 1})[0]
    return writer.Graph(b.nodes, [("input", [1, 5])], [(y, [1, 4])], b.inits, b.vi, b.consts, b.true_weights)


def test_identity_adds_nothing(tmp_path):
    plans, entries = [], []
    for k, (identity, info) in enumerate([(False, True), (True, True), (True, False)]):
        d = tmp_path / str(k)
        writer.write_model_files(graph(identity, info), str(d))
        with open(os.path.join(d, "variables.fpp")) as fh:
            entries.append([ln for ln in fh if "architecture" in ln or "inputs" in ln])
        plans.append(api.check_model(str(d)))
    assert plans[0].split() == ["mlp", "b0->b1", "[5x8:relu", "8x4]"]
    assert plans[1] == plans[2] == plans[0] and entries[1] == entries[0]
