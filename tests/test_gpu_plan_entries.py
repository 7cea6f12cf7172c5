"""Model entries of the operators that the selective layers' export does not write (activations, 2-D operands, features
from the middle of a value, groups, no gate, no softplus, no activation): through use_model, against 64 bits."""
import numpy as np
import pytest
import torch

from rosenna_b200 import api, writer
from tests import ops_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device():
    assert torch.cuda.is_available(), "gpu tests need a CUDA device"
    api.set_devices([0])
    yield
    api.finalize()


def load(d, build, T, F, extra=()):
    """Model of one input (1, T, F) (T = 0: (1, F)); build(b, v) -> outputs [(name, shape)] from it as a (T, 1, F) value."""
    b = writer._Builder()
    ins = [("input", [1, T, F] if T else [1, F])] + [(k, list(s)) for k, s in extra]
    for k, s in ins:
        b.vi[k] = list(s)
    v = b.add("Transpose", ["input"], [[T, 1, F]], {"perm": [1, 0, 2]})[0] if T else "input"
    outs = build(b, v)
    writer.write_model_files(writer.Graph(b.nodes, ins, outs, b.inits, b.vi, b.consts, b.true_weights), str(d))
    api.initialize(str(d))
    return api.plan_description()


def back(b, v, T, F):
    return b.add("Transpose", [v], [[1, T, F]], {"perm": [1, 0, 2]})[0], [1, T, F]


def near(got, want, tol):
    assert got.shape == want.shape
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / tol):.2f} bounds"


@pytest.mark.parametrize("n", [1, 5, 300])
@pytest.mark.parametrize("T,F,K,M,first,act", [(0, 20, 20, 30, 0, "relu"), (0, 300, 200, 17, 64, "silu"), (0, 1400, 1300, 40, 100, "none"),
                                               (7, 24, 16, 9, 8, "tanh"), (5, 300, 140, 150, 3, "sigmoid")])
def test_gemm8(tmp_path, n, T, F, K, M, first, act):
    rng = np.random.default_rng(n + F)
    w, bias = (rng.standard_normal((M, K)) / np.sqrt(K)).astype(np.float32), rng.standard_normal(M).astype(np.float32)

    def build(b, v):
        y = b.add("Gemm8", [v, b.weight(w), b.weight(bias)], [[T, 1, M] if T else [1, M]], {"params": [first, api.ACTS[act]]})[0]
        return [back(b, y, T, M)] if T else [(y, [1, M])]

    assert "gemm8" in load(tmp_path, build, T, F)
    x = rng.standard_normal((n, T, F) if T else (n, F)).astype(np.float32)
    got = api.use_model([x])[0].reshape(n * max(T, 1), M)
    want, tol = ref.gemm8(w, np.ascontiguousarray(x.reshape(-1, F)[:, first:first + K].T), bias, act)
    near(got, want.T, tol.T)


@pytest.mark.parametrize("n", [1, 5, 300])
@pytest.mark.parametrize("T,F,D,W,first,act,state", [(9, 20, 12, 4, 8, 0, True), (1, 12, 12, 3, 0, 0, True), (30, 10, 4, 8, 5, 4, True),
                                                     (6, 5, 5, 1, 0, 0, False)])
def test_causal_conv(tmp_path, n, T, F, D, W, first, act, state):
    rng = np.random.default_rng(n + F)
    w, bias = rng.standard_normal((D, W)).astype(np.float32), rng.standard_normal(D).astype(np.float32)

    def build(b, v):
        y, s = b.add("CausalConv", [v] + (["state"] if state else []) + [b.weight(w), b.weight(bias)], [[T, 1, D], [1, W - 1, D]],
                     {"params": [first, act]})
        return ([(s, [1, W - 1, D])] if state else []) + [back(b, y, T, D)]

    load(tmp_path, build, T, F, [("state", (1, W - 1, D))] if state else [])
    x = rng.standard_normal((n, T, F)).astype(np.float32)
    s0 = rng.standard_normal((n, W - 1, D)).astype(np.float32)
    *s1, y = api.use_model([x] + ([s0] if state else []))
    want, tol, sw = ref.conv(np.ascontiguousarray(x[..., first:first + D].transpose(2, 1, 0)), w, bias,
                             np.ascontiguousarray(s0.transpose(2, 1, 0)) if state else None, silu=act == 4)
    near(y, want.transpose(2, 1, 0), tol.transpose(2, 1, 0))
    if state:
        assert np.array_equal(s1[0], sw.transpose(2, 1, 0).astype(np.float32))


@pytest.mark.parametrize("n", [1, 5, 300])
@pytest.mark.parametrize("T,D,N,G,softplus,gate,state", [(9, 12, 5, 3, True, False, True), (40, 6, 16, 1, False, True, True),
                                                         (1, 8, 8, 2, False, False, True), (70, 4, 4, 4, True, True, False)])
def test_scan(tmp_path, n, T, D, N, G, softplus, gate, state):
    """x is an 8-bit Gemm's output (its D features alone); dt, B, C and z lie at odd places of the input."""
    rng = np.random.default_rng(n + T)
    A, skip, dtb = -np.abs(rng.standard_normal((D, N))).astype(np.float32), rng.standard_normal(D).astype(np.float32), -rng.random(D).astype(np.float32)
    wx, zero = rng.standard_normal((D, D)).astype(np.float32), np.zeros(D, np.float32)
    at, F = {}, D
    for k, c in (("C", N * G), ("z", D), ("dt", D), ("B", N * G)):
        F += 1
        at[k] = F
        F += c

    def build(b, v):
        x = b.add("Gemm8", [v, b.weight(wx), b.weight(zero)], [[T, 1, D]], {"params": [0, 0]})[0]
        y, h = b.add("SelectiveScan", [x, v, v, v, v if gate else "", "state" if state else "", b.weight(A), b.weight(skip), b.weight(dtb)],
                     [[T, 1, D], [1, N, D]], {"params": [at["dt"], at["B"], at["C"], at["z"], G, int(softplus)]})
        return [back(b, x, T, D), (h, [1, N, D]), back(b, y, T, D)]

    load(tmp_path, build, T, F, [("state", (1, N, D))] if state else [])
    x = rng.standard_normal((n, T, F)).astype(np.float32)
    if not softplus:
        x[..., at["dt"]:at["dt"] + D] = 1 + 0.1 * np.abs(x[..., at["dt"]:at["dt"] + D])  # steps above 0 with the bias
    h0 = rng.standard_normal((n, N, D)).astype(np.float32)
    h, u, y = api.use_model([x] + ([h0] if state else []))  # in the order of their nodes (x and y come transposed)
    t3 = lambda a: np.ascontiguousarray(a.transpose(2, 1, 0))  # noqa: E731
    part = lambda k, c: t3(x[..., at[k]:at[k] + c])  # noqa: E731
    want, tol, hw, htol = ref.scan(t3(u), part("dt", D), part("B", N * G).reshape(G, N, T, n), part("C", N * G).reshape(G, N, T, n), A, skip,
                                   dtb, z=part("z", D) if gate else None, h0=t3(h0) if state else None, use_softplus=softplus)
    near(y, want.transpose(2, 1, 0), tol.transpose(2, 1, 0))
    near(h, hw.transpose(2, 1, 0), htol.transpose(2, 1, 0) + 1e-37)
