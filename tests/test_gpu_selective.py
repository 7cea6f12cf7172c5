"""Selective state space models through initialize() and use_model, against the
PyTorch module in 64 bits within the engine's limits (oracle/parity.py), and, with
8-bit Gemms, against the same operators run one by one, bit for bit."""
import numpy as np
import pytest
import torch
from torch import nn

from oracle import parity
from rosenna_b200 import api
from tests.test_selective_host import write

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device():
    assert torch.cuda.is_available(), "gpu tests need a CUDA device"
    api.set_devices([0])
    yield
    api.finalize()


def reference(mods, head, x, states, mode):
    """-> the model's outputs in order, 64 bits, logical shapes (N, ...)."""
    v, out = torch.from_numpy(x.astype(np.float64)), []
    for i, m in enumerate(mods):
        st = [torch.from_numpy(s.astype(np.float64)) for s in states[2 * i:2 * i + 2]] if states else [None, None]
        v, c, h = m.double()(v, *st)
        out += [c, h] if states else []
    v = nn.Sequential(*head).double()(v[:, -1]) if mode == "last" else v
    return [o.detach().numpy() for o in out + [v]]


@pytest.mark.parametrize("n", [1, 3, 129, 1000])
@pytest.mark.parametrize("layers,width,T,kw,mode,with_state", [
    (1, 12, 7, {}, "last", True), (2, 16, 1, {}, "last", True), (2, 9, 50, dict(states=7, taps=3), "y", True),
    (1, 32, 20, dict(expand=1), "last", False), (1, 8, 300, {}, "y", False)])
def test_model_matches_the_module(tmp_path, n, layers, width, T, kw, mode, with_state):
    mods, head = write(tmp_path, layers, width, T, mode=mode, with_state=with_state, **kw)
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, T, width)).astype(np.float32)
    states = []
    for m in mods if with_state else []:
        states += [0.5 * rng.standard_normal((n, m.taps - 1, m.channels)).astype(np.float32),
                   0.5 * rng.standard_normal((n, m.states, m.channels)).astype(np.float32)]
    api.initialize(str(tmp_path))
    got = api.use_model([x] + states)
    for g, w in zip(got, reference(mods, head, x, states, mode)):
        r = parity.compare(g, w)
        assert r["ok"], parity.describe(r)


def device_model(n, arrays):
    """use_model_device on the logical arrays; -> outputs."""
    ins = [torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.float32).transpose(range(a.ndim - 1, -1, -1)))).cuda() for a in arrays]
    outs, res = [], []
    for s, b in api.output_specs():
        shape = api.batched_shape(s, b, n)
        outs.append(torch.zeros(shape[::-1], device="cuda"))
    return ins, outs


def test_steps_carry_the_state(tmp_path):
    """A one-step model called step by step with the states it returned, against the module on the whole.  (Not with
    8-bit Gemms: there a last bit of an operand can move a value to its other neighbour of 8 bits.)"""
    n, T, width = 37, 11, 16
    mods, head = write(tmp_path, 2, width, 1)
    x = np.random.default_rng(1).standard_normal((n, T, width)).astype(np.float32)
    zero = []
    for m in mods:
        zero += [np.zeros((n, m.taps - 1, m.channels), np.float32), np.zeros((n, m.states, m.channels), np.float32)]
    api.initialize(str(tmp_path))
    st = zero
    for t in range(T):
        *st, y = api.use_model([x[:, t:t + 1]] + st)
    for g, w in zip(st + [y], reference(mods, head, x, zero, "last")):
        r = parity.compare(g, w)
        assert r["ok"], parity.describe(r)


def test_eight_bit_layer_equals_its_operators(tmp_path):
    n, T, width = 130, 9, 24
    (m,), _ = write(tmp_path, 1, width, T, eight_bit=True, with_state=False, mode="y")
    x = np.random.default_rng(2).standard_normal((n, T, width)).astype(np.float32)
    api.initialize(str(tmp_path))
    got = api.use_model([x])[0]
    f = lambda p: p.detach().numpy()  # noqa: E731
    D, R, S, c = m.channels, m.dt_rank, m.states, T * n
    g = [api.Gemm8(f(p)) for p in (m.in_proj.weight, m.x_proj.weight, m.dt_proj.weight, m.out_proj.weight)]
    conv = api.CausalConv(f(m.conv1d.weight)[:, 0], f(m.conv1d.bias))
    A = (-np.exp(m.A_log.detach().double().numpy())).astype(np.float32)
    scan = api.SelectiveScan(A, f(m.D), f(m.dt_proj.bias))
    ws = torch.zeros(max(16, max(k.workspace_bytes(c) for k in g), scan.workspace_bytes(n, T)), dtype=torch.uint8, device="cuda")
    w = dict(workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    e = lambda r: torch.zeros((r, c), device="cuda")  # noqa: E731
    xin = torch.from_numpy(np.ascontiguousarray(x.transpose(2, 1, 0)).reshape(width, c)).cuda()
    xz, u, dbc, dt, s, y = e(2 * D), e(D), e(R + 2 * S), e(D), e(D), e(width)
    p = lambda t, row=0: t.data_ptr() + 4 * row * c  # noqa: E731
    g[0].run(c, p(xin), p(xz), **w)
    conv.run(n, T, p(xz), p(u), stream=w["stream"])
    g[1].run(c, p(u), p(dbc), **w)
    g[2].run(c, p(dbc), p(dt), **w)
    scan.run(n, T, p(u), p(dt), p(dbc, R), p(dbc, R + S), p(s), z=p(xz, D), **w)
    g[3].run(c, p(s), p(y), **w)
    want = y.cpu().numpy().reshape(width, T, n).transpose(2, 1, 0)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("eight_bit", [False, True])
def test_every_entry_point_agrees(tmp_path, eight_bit):
    n, T, width = 1000, 6, 16
    write(tmp_path, 2, width, T, eight_bit=eight_bit, with_state=False)
    x = np.random.default_rng(3).standard_normal((n, T, width)).astype(np.float32)
    api.initialize(str(tmp_path))
    want = api.use_model([x])[0]
    assert np.array_equal(api.use_model([x.astype(np.float64)], dtype=np.float64)[0].astype(np.float32), want)
    ins, outs = device_model(n, [x])
    st = torch.cuda.current_stream().cuda_stream
    for fn in (api.use_model_device, api.use_model_device_noalloc):
        outs[0].fill_(0)
        fn(n, [t.data_ptr() for t in ins], [t.data_ptr() for t in outs], st)
        assert np.array_equal(outs[0].cpu().numpy().T, want), fn.__name__
    # fewer samples after more, whose rows then have gaps between them
    whole = api.last_launch_count()
    for k in (1, 333):
        got = api.use_model([x[:k]])[0]
        ins, outs = device_model(k, [x[:k]])
        api.use_model_device(k, [t.data_ptr() for t in ins], [t.data_ptr() for t in outs], st)
        assert api.last_launch_count() <= whole + 8  # (few columns are quantised ahead, a launch more each)
        assert np.array_equal(got, want[:k]) and np.array_equal(outs[0].cpu().numpy().T, want[:k])


def test_leading_rows_of_a_value_are_read_in_place(tmp_path):
    """A Slice of the first features is no copy: what reads it takes those rows alone, and as a model's output it is
    copied out of the wider buffer."""
    rng = np.random.default_rng(6)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    w1, b1, w2, b2 = f(8, 5), f(8), f(4, 3), f(4)
    from rosenna_b200 import writer

    for tail in ("gemm", "relu", "none"):
        b = writer._Builder()
        h = b.add("Gemm", ["input", b.weight(w1), b.weight(b1)], [[1, 8]], {"transB": 1})[0]
        r = b.add("Slice", [h], [[1, 3]], {"axes": [1], "starts": [0], "ends": [3]})[0]
        out, shape = r, [1, 3]
        if tail == "gemm":
            out, shape = b.add("Gemm", [r, b.weight(w2), b.weight(b2)], [[1, 4]], {"transB": 1})[0], [1, 4]
        elif tail == "relu":
            out = b.add("Relu", [r], [[1, 3]])[0]
        g = writer.Graph(b.nodes, [("input", [1, 5])], [(out, shape)], b.inits, b.vi, b.consts, b.true_weights)
        d = tmp_path / tail
        writer.write_model_files(g, str(d))
        api.initialize(str(d))
        assert "gather" not in api.plan_description()
        for n in (1, 500):
            x = f(n, 5)
            v = (x.astype(np.float64) @ w1.T.astype(np.float64) + b1)[:, :3]
            want = v @ w2.T.astype(np.float64) + b2 if tail == "gemm" else np.maximum(v, 0) if tail == "relu" else v
            r = parity.compare(api.use_model([x])[0], want)
            assert r["ok"], (tail, n, parity.describe(r))
