"""The causal convolution, the selective scan and the 8-bit Gemm against 64-bit
references (tests/ops_reference.py, whose bounds follow from the arithmetic)."""
import numpy as np
import pytest
import torch

from rosenna_b200 import api
from tests import ops_reference as ref

pytestmark = pytest.mark.gpu
FILL = 12345.0  # what an output holds before a run


@pytest.fixture(autouse=True)
def _device():
    assert torch.cuda.is_available(), "gpu tests need a CUDA device"


def dev(a, ld=None):
    """(..., n) host array -> device tensor of rows `ld` apart (garbage between them)."""
    if a is None:
        return None
    a = np.ascontiguousarray(a)
    n = a.shape[-1]
    ld = ld or n
    t = torch.full((int(np.prod(a.shape[:-1])), ld), float("nan") if a.dtype == np.float32 else -1, device="cuda",
                   dtype=torch.float32 if a.dtype == np.float32 else torch.int32)
    t[:, :n] = torch.from_numpy(a.reshape(-1, n)).cuda()
    return t


def host(t, shape):
    return t[:, :shape[-1]].cpu().numpy().reshape(shape).astype(np.float64)


def ptr(t):
    return 0 if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def check(got, want, tol, what):
    """Within the bound; where the reference is NaN (not written) the output still holds FILL."""
    untouched = np.isnan(want)
    assert np.all(got[untouched] == FILL), what + ": wrote where it should not"
    bad = np.abs(got - want) > tol
    bad &= ~untouched
    bad |= np.isnan(got) & ~untouched
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / tol):.2f} bounds"


def rand_lens(rng, n, T):
    lens = rng.integers(0, T + 1, size=n).astype(np.int32)
    lens[0] = T
    if n > 1:
        lens[-1] = 0
    return lens


# ---- causal convolution -------------------------------------------------------------------------------------------
CONV = [  # n, T, D, W, state, lens, ld extra
    (1, 1, 3, 4, True, False, 0), (1, 1, 128, 4, False, False, 0), (33, 1, 5, 2, True, False, 0), (1000, 1, 7, 8, True, False, 3),
    (1, 2, 4, 4, True, False, 0), (1, 17, 9, 8, True, False, 0), (1, 1000, 33, 4, False, False, 0), (2, 333, 5, 3, True, True, 0),
    (3, 16, 4, 1, False, True, 0), (7, 129, 6, 5, True, True, 0), (31, 15, 3, 6, True, True, 5), (32, 50, 8, 4, False, False, 0),
    (64, 33, 4, 7, True, True, 0), (100, 50, 3, 4, True, True, 28), (129, 5, 2, 4, True, False, 0), (256, 64, 4, 4, True, False, 0),
    (4096, 50, 4, 4, False, True, 0), (1028, 3, 2, 8, True, True, 0), (40000, 1, 20, 4, True, True, 0),
    (40000, 1, 20, 3, True, False, 4), (40001, 1, 20, 4, True, True, 0), (4096, 50, 10, 4, True, True, 4), (2048, 100, 12, 8, True, True, 0),
    (31, 300, 3, 8, True, True, 2), (1, 128, 2, 8, True, False, 0), (16, 8, 3, 4, True, True, 0), (4, 1025, 2, 2, False, False, 0), (5, 4099, 3, 3, True, True, 0),
]


@pytest.mark.parametrize("n,T,D,W,state,ragged,extra", CONV)
@pytest.mark.parametrize("act", ["silu", None])
def test_causal_conv(n, T, D, W, state, ragged, extra, act):
    rng = np.random.default_rng(n * 7 + T)
    x = rng.standard_normal((D, T, n)).astype(np.float32)
    w, b = rng.standard_normal((D, W)).astype(np.float32), rng.standard_normal(D).astype(np.float32)
    s0 = rng.standard_normal((D, W - 1, n)).astype(np.float32) if state and W > 1 else None
    lens = rand_lens(rng, n, T) if ragged else None
    if ragged:  # what lies behind a sample's last step reaches nothing
        x[:, np.arange(T)[:, None] >= lens[None]] = np.nan
    op = api.CausalConv(w, b if act else None, act=act)
    ld = n + extra
    tx, ts0, tl = dev(x, ld), dev(s0, ld), None if lens is None else dev(lens[None])
    y = torch.full((D * T, ld), FILL, device="cuda")
    s1 = torch.full((D * (W - 1), ld), FILL, device="cuda") if W > 1 else None
    op.run(n, T, ptr(tx), ptr(y), state_in=ptr(ts0), state_out=ptr(s1), lens=ptr(tl), ld_x=ld, ld_y=ld, ld_state_in=ld,
           ld_state_out=ld, stream=stream())
    xr = np.nan_to_num(x) if ragged else x
    want, tol, sw = ref.conv(xr, w, b if act else None, s0, lens, silu=act == "silu")
    check(host(y, (D, T, n)), want, tol, "y")
    assert torch.all(y[:, n:] == FILL)
    if W > 1:
        assert np.array_equal(host(s1, (D, W - 1, n)), sw)
        assert torch.all(s1[:, n:] == FILL)
        if s0 is not None:  # the same in place
            op.run(n, T, ptr(tx), ptr(y), state_in=ptr(ts0), state_out=ptr(ts0), lens=ptr(tl), ld_x=ld, ld_y=ld, ld_state_in=ld,
                   ld_state_out=ld, stream=stream())
            assert np.array_equal(host(ts0, (D, W - 1, n)), sw)


def test_causal_conv_of_no_steps_keeps_the_state():
    rng = np.random.default_rng(1)
    w, s0 = rng.standard_normal((5, 4)).astype(np.float32), rng.standard_normal((5, 3, 9)).astype(np.float32)
    a, b = dev(s0), torch.full((15, 9), FILL, device="cuda")
    api.CausalConv(w).run(9, 0, 0, 0, state_in=ptr(a), state_out=ptr(b), stream=stream())
    assert np.array_equal(host(b, s0.shape), s0.astype(np.float64))
    api.CausalConv(w).run(9, 0, 0, 0, state_out=ptr(b), stream=stream())
    assert torch.all(b == 0)


# ---- selective scan -----------------------------------------------------------------------------------------------
SCAN = [  # n, T, D, N, G, state, gate, lens, ld extra
    (1, 1, 3, 16, 1, True, True, False, 0), (1, 1, 128, 16, 1, False, False, False, 0), (33, 1, 6, 4, 2, True, True, False, 0),
    (300, 1, 4, 16, 1, True, True, False, 5), (1, 2, 5, 16, 1, True, True, False, 0), (1, 700, 40, 16, 1, True, True, False, 0),
    (1, 4096, 64, 16, 1, True, True, False, 0), (2, 333, 12, 7, 3, True, False, True, 0), (3, 64, 10, 1, 1, False, True, True, 0),
    (5, 1000, 9, 33, 1, True, True, True, 3), (7, 129, 6, 24, 2, True, True, True, 0), (16, 257, 8, 64, 1, False, True, False, 0),
    (31, 15, 4, 5, 1, True, False, True, 5), (32, 50, 8, 16, 1, False, True, False, 0), (64, 33, 16, 8, 4, True, True, True, 0),
    (100, 50, 6, 16, 2, True, True, True, 28), (129, 5, 2, 32, 1, True, True, False, 0), (256, 64, 20, 16, 1, True, True, False, 0),
    (129, 300, 16, 16, 1, True, True, False, 0), (64, 1111, 2, 16, 1, True, False, True, 0), (2048, 50, 16, 16, 1, False, True, True, 0),
    (40000, 1, 20, 16, 1, True, True, True, 0), (40001, 1, 20, 16, 2, True, False, True, 0), (40000, 1, 20, 7, 1, True, True, False, 4),
    (700, 1, 33, 24, 1, True, True, True, 0), (48, 1, 5, 64, 1, False, True, False, 0), (36000, 1, 17, 4, 1, False, True, False, 0), (1028, 3, 3, 16, 3, True, False, True, 0), (128, 40, 17, 16, 1, True, True, False, 0),
]


def scan_case(n, T, D, N, G, state, gate, ragged, seed=0):
    rng = np.random.default_rng(n * 7 + T + seed)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    c = dict(x=f(D, T, n), dt=0.7 * f(D, T, n), B=f(G, N, T, n), C=f(G, N, T, n), A=-np.abs(f(D, N)) * np.arange(1, N + 1, dtype=np.float32),
             skip=f(D), dt_bias=(-3 + f(D)).astype(np.float32), z=f(D, T, n) if gate else None, h0=f(D, N, n) if state else None,
             lens=rand_lens(rng, n, T) if ragged else None)
    if ragged:
        behind = np.arange(T)[:, None] >= c["lens"][None]
        for k in ("x", "dt", "B", "C", "z"):
            if c[k] is not None:
                c[k][..., behind] = np.nan
    return c


def scan_reference(c, **kw):
    q = {k: (np.nan_to_num(v) if isinstance(v, np.ndarray) and v.dtype == np.float32 else v) for k, v in c.items()}
    return ref.scan(**q, **kw)


def run_scan(c, ld=None, workspace=True, softplus=True, in_place=False):
    D, T, n = c["x"].shape
    G, N = c["B"].shape[:2]
    ld = ld or n
    op = api.SelectiveScan(c["A"], c["skip"], c["dt_bias"], softplus=softplus, groups=G)
    t = {k: dev(c[k], ld) for k in ("x", "dt", "B", "C", "z", "h0")}
    tl = None if c["lens"] is None else dev(c["lens"][None])
    y, hn = torch.full((D * T, ld), FILL, device="cuda"), torch.full((D * N, ld), FILL, device="cuda")
    if in_place:
        hn = t["h0"]
    need = op.workspace_bytes(n, T) if workspace else 0
    # the workspace starts as NaN: what a run reads of it, it has written
    ws = torch.full((need // 4 + 1,), float("nan"), device="cuda") if need else None
    op.run(n, T, ptr(t["x"]), ptr(t["dt"]), ptr(t["B"]), ptr(t["C"]), ptr(y), z=ptr(t["z"]), h0=ptr(t["h0"]), hn=ptr(hn), lens=ptr(tl),
           **{"ld_" + k: ld for k in ("x", "dt", "B", "C", "z", "y", "h0", "hn")}, workspace=ptr(ws), workspace_bytes=need, stream=stream())
    if ld > n and not in_place:
        assert torch.all(y[:, n:] == FILL) and torch.all(hn[:, n:] == FILL)
    return host(y, (D, T, n)), host(hn, (D, N, n)), need


@pytest.mark.parametrize("n,T,D,N,G,state,gate,ragged,extra", SCAN)
def test_scan(n, T, D, N, G, state, gate, ragged, extra):
    c = scan_case(n, T, D, N, G, state, gate, ragged)
    want, tol, hw, htol = scan_reference(c)
    y, hn, need = run_scan(c, n + extra)
    check(y, want, tol, "y")
    check(hn, hw, htol + 1e-37, "hn")
    if need:  # the unsplit form of the same
        y, hn, _ = run_scan(c, n + extra, workspace=False)
        check(y, want, tol, "y unsplit")
        check(hn, hw, htol + 1e-37, "hn unsplit")
    if state:
        _, hn, _ = run_scan(c, n + extra, in_place=True)
        check(hn, hw, htol + 1e-37, "hn in place")


def test_some_scans_split():
    """The list above holds scans of both forms."""
    ws = [api.SelectiveScan(np.zeros((c[2], c[3]), np.float32), groups=c[4]).workspace_bytes(c[0], c[1]) for c in SCAN]
    assert min(ws) == 0 < max(ws)


@pytest.mark.parametrize("n,T,D,N", [(3, 200, 5, 16), (40, 30, 4, 8)])
def test_scan_without_softplus_skip_and_bias(n, T, D, N):
    c = scan_case(n, T, D, N, 1, True, True, False)
    c["dt"] = np.abs(c["dt"]) * np.float32(0.1)
    c["skip"] = c["dt_bias"] = None
    want, tol, hw, htol = scan_reference(c, use_softplus=False)
    y, hn, _ = run_scan(c, softplus=False)
    check(y, want, tol, "y")
    check(hn, hw, htol + 1e-37, "hn")


@pytest.mark.parametrize("n,T", [(5, 40), (64, 1), (40000, 1), (70, 33), (2, 600)])
def test_lengths_outside_the_sequence(n, T):
    """A length below 0 counts as 0, one beyond T as T."""
    c = scan_case(n, T, 6, 8, 1, True, True, True)
    inside = c["lens"].copy()
    for k in ("x", "dt", "B", "C", "z"):
        c[k] = np.nan_to_num(c[k])
    c["lens"] = np.where(inside == 0, -7, np.where(inside == T, T + 1000, inside)).astype(np.int32)
    want, tol, hw, htol = scan_reference(dict(c, lens=inside))
    y, hn, _ = run_scan(c)
    check(y, want, tol, "y")
    check(hn, hw, htol + 1e-37, "hn")
    w, s0 = c["A"][:, :4].copy(), c["h0"][:, :3].copy()
    want, tol, sw = ref.conv(c["x"], w, None, s0, inside)
    tx, ts, tl, u = dev(c["x"]), dev(s0), dev(c["lens"][None]), torch.full((6 * T, n), FILL, device="cuda")
    api.CausalConv(w).run(n, T, ptr(tx), ptr(u), state_in=ptr(ts), state_out=ptr(ts), lens=ptr(tl), stream=stream())
    check(host(u, (6, T, n)), want, tol, "conv")
    assert np.array_equal(host(ts, (6, 3, n)), sw)


def test_a_very_long_record():
    c = scan_case(1, 30001, 3, 16, 1, True, True, False)
    want, tol, hw, htol = scan_reference(c)
    y, hn, need = run_scan(c)
    assert need > 0
    check(y, want, tol, "y")
    check(hn, hw, htol + 1e-37, "hn")


def test_scan_steps_of_every_size():
    """Steps from e^-40 to 40: the decay goes from 1 to 0, softplus keeps its relative accuracy."""
    n, T, D, N = 64, 40, 2, 16
    c = scan_case(n, T, D, N, 1, True, False, False)
    c["dt"] = np.broadcast_to(np.linspace(-40, 40, T, dtype=np.float32)[None, :, None], (D, T, n)).copy()
    c["dt_bias"][:] = 0
    want, tol, hw, htol = scan_reference(c)
    y, hn, _ = run_scan(c)
    check(y, want, tol, "y")
    check(hn, hw, htol + 1e-37, "hn")


@pytest.mark.parametrize("n", [1, 48])
def test_history_equals_its_single_steps(n):
    """The state carried over single steps: conv and scan as a solver calls them, step by step, in place."""
    T, D, N, W = 37, 12, 16, 4
    c = scan_case(n, T, D, N, 1, True, True, False)
    rng = np.random.default_rng(5)
    w, b, s0 = (rng.standard_normal(s).astype(np.float32) for s in ((D, W), (D,), (D, W - 1, n)))
    cw, ctol, _ = ref.conv(c["x"], w, b, s0)
    want, tol, hw, htol = scan_reference(c)
    conv, scan = api.CausalConv(w, b), api.SelectiveScan(c["A"], c["skip"], c["dt_bias"])
    ts, th = dev(s0), dev(c["h0"])
    for t in range(T):
        x, dt, B, C, z = (dev(np.ascontiguousarray(c[k][..., t, :])) for k in ("x", "dt", "B", "C", "z"))
        u, y = torch.full((D, n), FILL, device="cuda"), torch.full((D, n), FILL, device="cuda")
        conv.run(n, 1, ptr(x), ptr(u), state_in=ptr(ts), state_out=ptr(ts), stream=stream())
        scan.run(n, 1, ptr(x), ptr(dt), ptr(B), ptr(C), ptr(y), z=ptr(z), h0=ptr(th), hn=ptr(th), stream=stream())
        check(host(u, (D, n)), cw[:, t], ctol[:, t], f"conv step {t}")
        check(host(y, (D, n)), want[:, t], tol[:, t], f"scan step {t}")
    check(host(th, (D, N, n)), hw, htol + 1e-37, "hn")


@pytest.mark.parametrize("n", [5, 64])
def test_scan_of_no_steps_keeps_the_state(n):
    h = np.random.default_rng(2).standard_normal((3, 7, n)).astype(np.float32)
    op = api.SelectiveScan(-np.ones((3, 7), np.float32))
    a, b = dev(h), torch.full((21, n), FILL, device="cuda")
    op.run(n, 0, 0, 0, 0, 0, 0, h0=ptr(a), hn=ptr(b), stream=stream())
    assert np.array_equal(host(b, h.shape), h.astype(np.float64))
    op.run(n, 0, 0, 0, 0, 0, 0, hn=ptr(b), stream=stream())
    assert torch.all(b == 0)


def test_rows_beyond_32_bits():
    """Rows 2^29 values apart: the sixth starts beyond 2^31 of them."""
    ld, rng = 1 << 29, np.random.default_rng(3)
    if torch.cuda.mem_get_info()[0] < 80e9:
        pytest.skip("needs 72 GB of device memory")
    spare = [torch.empty(6 * ld, device="cuda") for _ in range(6)]

    def put(i, a):  # (6 rows, n)
        t = spare[i].view(6, ld)
        t[:, :a.shape[1]] = torch.from_numpy(a).cuda()
        return t.data_ptr()

    for n in (3, 64):
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        c = dict(x=f(2, 3, n), dt=f(2, 3, n), B=f(1, 2, 3, n), C=f(1, 2, 3, n), A=-np.ones((2, 2), np.float32), z=f(2, 3, n))
        p = {k: put(i, c[k].reshape(6, n)) for i, k in enumerate(("x", "dt", "B", "C", "z"))}
        spare[5].view(6, ld)[:, :n] = FILL
        out = spare[5].view(6, ld)
        api.SelectiveScan(c["A"]).run(n, 3, p["x"], p["dt"], p["B"], p["C"], out.data_ptr(), z=p["z"], stream=stream(),
                                      **{"ld_" + k: ld for k in ("x", "dt", "B", "C", "z", "y")})
        want, tol, _, _ = ref.scan(**c)
        check(out[:, :n].cpu().numpy().reshape(2, 3, n).astype(np.float64), want, tol, "scan")
        w = f(2, 3)
        api.CausalConv(w).run(n, 3, p["x"], out.data_ptr(), ld_x=ld, ld_y=ld, stream=stream())
        want, tol, _ = ref.conv(c["x"], w)
        check(out[:, :n].cpu().numpy().reshape(2, 3, n).astype(np.float64), want, tol, "conv")
        w = f(6, 6)
        api.Gemm8(w).run(n, p["x"], out.data_ptr(), ld_x=ld, ld_y=ld, stream=stream())
        want, tol = ref.gemm8(w, c["x"].reshape(6, n))
        check(out[:, :n].cpu().numpy().astype(np.float64), want, tol, "gemm8")
    del spare, out
    torch.cuda.empty_cache()  # not kept from the tests after this one


def test_one_operator_on_two_streams():
    """Runs of the same operators at once, each with its own arrays and workspace, equal runs alone."""
    scan = api.SelectiveScan(-np.ones((32, 16), np.float32))
    rng = np.random.default_rng(4)
    gemm = api.Gemm8(rng.standard_normal((300, 1100)).astype(np.float32))
    n, T, cols = 2, 600, 700
    sets = []
    for _ in range(2):
        q = {k: torch.randn(r * T, n, device="cuda") for k, r in (("x", 32), ("dt", 32), ("B", 16), ("C", 16))}
        q |= dict(y=torch.empty(32 * T, n, device="cuda"), gx=torch.randn(1100, cols, device="cuda"), gy=torch.empty(300, cols, device="cuda"),
                  ws=torch.empty(scan.workspace_bytes(n, T), dtype=torch.uint8, device="cuda"),
                  gws=torch.empty(max(16, gemm.workspace_bytes(cols)), dtype=torch.uint8, device="cuda"))
        sets.append(q)

    def go(q, st):
        scan.run(n, T, *(q[k].data_ptr() for k in ("x", "dt", "B", "C", "y")), workspace=q["ws"].data_ptr(), workspace_bytes=q["ws"].numel(), stream=st)
        gemm.run(cols, q["gx"].data_ptr(), q["gy"].data_ptr(), workspace=q["gws"].data_ptr(), workspace_bytes=q["gws"].numel(), stream=st)

    assert sets[0]["ws"].numel() > 0
    want = []
    for q in sets:
        go(q, stream())
        want.append((q["y"].clone(), q["gy"].clone()))
        q["y"].zero_()
        q["gy"].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        for q, st in zip(sets, streams):
            go(q, st.cuda_stream)
    torch.cuda.synchronize()
    for q, (y, gy) in zip(sets, want):
        assert torch.equal(q["y"], y) and torch.equal(q["gy"], gy)


# ---- 8-bit Gemm -----------------------------------------------------------------------------------------------------
GEMM = [  # n, K, M, bias, act, ld extra
    (1, 1, 1, True, "none", 0), (1, 16, 8, True, "relu", 0), (1, 1024, 2048, False, "none", 0), (2, 300, 77, True, "silu", 0),
    (3, 128, 128, True, "tanh", 1), (8, 513, 200, False, "sigmoid", 0), (9, 256, 130, True, "none", 0), (16, 100, 100, True, "none", 0),
    (17, 2000, 64, True, "none", 0), (33, 784, 64, True, "relu", 7), (64, 256, 256, True, "none", 0), (100, 129, 257, True, "silu", 4),
    (127, 1024, 333, True, "none", 0), (128, 128, 128, False, "none", 0), (129, 640, 16, True, "none", 0), (1000, 256, 256, True, "relu", 0),
    (1024, 1024, 1000, True, "none", 0), (4097, 200, 300, True, "tanh", 0), (5000, 16, 256, True, "relu", 0), (3001, 1100, 520, True, "none", 31),
    (40000, 256, 128, True, "none", 0),
]


@pytest.mark.parametrize("n,K,M,bias,act,extra", GEMM)
def test_gemm8(n, K, M, bias, act, extra):
    rng = np.random.default_rng(n + K)
    x = (rng.standard_normal((K, n)) * np.exp2(rng.integers(-6, 6, size=(K, 1)))).astype(np.float32)
    x[:, rng.integers(0, n)] = 0  # a column of zeros
    w = (rng.standard_normal((M, K)) / np.sqrt(K)).astype(np.float32)
    w[: M // 3, : K // 2] *= 100
    b = rng.standard_normal(M).astype(np.float32) if bias else None
    op = api.Gemm8(w, b, act=act)
    ld = n + extra
    tx, y = dev(x, ld), torch.full((M, ld), FILL, device="cuda")
    need = op.workspace_bytes(n)
    ws = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")
    op.run(n, ptr(tx), ptr(y), ld_x=ld, ld_y=ld, workspace=ptr(ws), workspace_bytes=need, stream=stream())
    assert torch.all(ws[need:] == 255) and torch.all(y[:, n:] == FILL)
    want, tol = ref.gemm8(w, x, b, act)
    check(host(y, (M, n)), want, tol, "y")


@pytest.mark.parametrize("n", [5, 300])
def test_gemm8_not_finite_and_extreme_columns(n):
    rng = np.random.default_rng(n)
    K, M = 300, 40
    x = rng.standard_normal((K, n)).astype(np.float32)
    x[7, 0], x[299, 1], x[130, 2] = np.inf, np.nan, -np.inf
    x[:, 3] *= np.float32(2.0 ** 100)
    x[:, 4] = np.float32(1e-42)  # below the smallest normal number
    w = rng.standard_normal((M, K)).astype(np.float32)
    op = api.Gemm8(w)
    tx, y = dev(x), torch.full((M, n), FILL, device="cuda")
    ws = torch.zeros(op.workspace_bytes(n) + 16, dtype=torch.uint8, device="cuda")
    op.run(n, ptr(tx), ptr(y), workspace=ptr(ws), workspace_bytes=ws.numel(), stream=stream())
    got = host(y, (M, n))
    assert np.isnan(got[:, :3]).all()
    want, tol = ref.gemm8(w, x[:, 3:])
    check(got[:, 3:], want, tol, "y")


def test_gemm8_rounds_ties_to_even_and_keeps_the_scale_rule():
    """Every e4m3 value, and the values half-way between two, through a weight of 1."""
    vals = np.array([s * m * 2.0 ** e for s in (1, -1) for e in range(-9, 9) for m in np.arange(8, 16) / 8.0], dtype=np.float32)
    vals = np.concatenate([vals, vals * np.float32(1 + 1 / 16), [448.0, 449.0, 447.999, 224.0, 0.0]]).astype(np.float32)
    n, K = len(vals), 128
    x = np.zeros((K, n), np.float32)
    x[0] = vals
    x[1] = 448.0  # fixes the block's scale at 1 for every value up to 448
    w = np.zeros((1, K), np.float32)
    w[0, 0] = 1
    op = api.Gemm8(w)
    tx, y = dev(x), torch.full((1, n), FILL, device="cuda")
    ws = torch.zeros(op.workspace_bytes(n) + 16, dtype=torch.uint8, device="cuda")
    op.run(n, ptr(tx), ptr(y), workspace=ptr(ws), workspace_bytes=ws.numel(), stream=stream())
    assert np.array_equal(host(y, (1, n)), ref.quantised_columns(x)[:1])


# ---- runs together, graphs, streams ---------------------------------------------------------------------------------
def layer(n, T, seed, D=48, N=16, I=24):
    """One layer as it is used: in-projection, conv + SiLU, projections of the step and of B and C, scan with its
    gate, out-projection.  -> run(stream, workspaces) and its buffers, and the 64-bit result's inputs."""
    rng = np.random.default_rng(seed)
    f = lambda *s: (rng.standard_normal(s) / np.sqrt(s[-1])).astype(np.float32)  # noqa: E731
    p = dict(win=f(2 * D, I), wc=f(D, 4), wdt=f(D, D), wbc=f(2 * N, D), wout=f(I, D),
             A=-np.broadcast_to(np.arange(1, N + 1, dtype=np.float32), (D, N)).copy(), dtb=np.full(D, -2.0, np.float32), skip=np.ones(D, np.float32))
    ops = dict(inp=api.Gemm8(p["win"]), conv=api.CausalConv(p["wc"]), dt=api.Gemm8(p["wdt"]), bc=api.Gemm8(p["wbc"]),
               scan=api.SelectiveScan(p["A"], p["skip"], p["dtb"]), out=api.Gemm8(p["wout"]))
    x = rng.standard_normal((I, T, n)).astype(np.float32)
    c = T * n
    e = lambda r: torch.full((r, c), FILL, device="cuda")  # noqa: E731
    bufs = dict(x=torch.from_numpy(x.reshape(I, c)).cuda(), xz=e(2 * D), u=e(D), dt=e(D), bc=e(2 * N), s=e(D), y=e(I))
    size = max(16, *(ops[k].workspace_bytes(c) for k in ("inp", "dt", "bc", "out")), ops["scan"].workspace_bytes(n, T))

    def run(st, ws):
        q = {k: v.data_ptr() for k, v in bufs.items()}
        w = dict(workspace=ws.data_ptr(), workspace_bytes=size, stream=st)
        ops["inp"].run(c, q["x"], q["xz"], **w)
        ops["conv"].run(n, T, q["xz"], q["u"], stream=st)
        ops["dt"].run(c, q["u"], q["dt"], **w)
        ops["bc"].run(c, q["u"], q["bc"], **w)
        ops["scan"].run(n, T, q["u"], q["dt"], q["bc"], q["bc"] + 4 * N * c, q["s"], z=q["xz"] + 4 * D * c, **w)
        ops["out"].run(c, q["s"], q["y"], **w)

    def want():
        """Each operator's reference on its actual inputs (8-bit rounding makes the chain itself discontinuous)."""
        b = {k: v.cpu().numpy() for k, v in bufs.items()}
        r3 = lambda a: a.reshape(a.shape[0], T, n)  # noqa: E731
        checks = [("xz", *ref.gemm8(p["win"], b["x"])), ("dt", *ref.gemm8(p["wdt"], b["u"])), ("bc", *ref.gemm8(p["wbc"], b["u"])),
                  ("y", *ref.gemm8(p["wout"], b["s"]))]
        cv, ct, _ = ref.conv(r3(b["xz"][:D]), p["wc"])
        sv, stol, _, _ = ref.scan(r3(b["u"]), r3(b["dt"]), r3(b["bc"][:N])[None], r3(b["bc"][N:])[None], p["A"], p["skip"], p["dtb"], z=r3(b["xz"][D:]))
        return checks + [("u", cv.reshape(D, c), ct.reshape(D, c)), ("s", sv.reshape(D, c), stol.reshape(D, c))]

    return run, bufs, size, want


@pytest.mark.parametrize("n,T", [(1, 1), (1, 300), (70, 9), (3, 40)])
def test_operators_together(n, T):
    run, bufs, size, want = layer(n, T, n + T)
    run(stream(), torch.full((size,), 255, dtype=torch.uint8, device="cuda"))
    for k, w, tol in want():
        check(bufs[k].cpu().numpy().astype(np.float64), w, tol, k)


def test_two_graphs_side_by_side():
    """Two captured layers with a workspace each, replayed on two streams at once, equal their eager runs bit for bit;
    new inputs are taken by the replay."""
    made, want = [], []
    for seed in (1, 2):
        run, bufs, size, _ = layer(2, 130, seed)
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        run(stream(), ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(stream(), ws)
        bufs["x"].mul_(0.5)
        run(stream(), ws)
        want.append(bufs["y"].clone())
        bufs["y"].fill_(FILL)
        made.append((g, bufs, torch.cuda.Stream(), ws))
    torch.cuda.synchronize()
    for _ in range(3):
        for g, _, s, _ in made:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, bufs, _, _), w in zip(made, want):
        assert torch.equal(bufs["y"], w)


FIRST_RUN = """
import sys
sys.path.insert(0, {root!r})
import numpy as np, torch
from rosenna_b200 import api
d = "cuda"
torch.zeros(1, device=d)
conv, scan, gemm = api.CausalConv(np.ones((6, 7), np.float32)), api.SelectiveScan(-np.ones((6, 24), np.float32)), api.Gemm8(np.ones((40, 900), np.float32))
jobs = []
for n, T in ((3, 1), (64, 1), (4, 100), (64, 9)):
    a = [torch.rand(24 * T, n, device=d) for _ in range(5)] + [torch.zeros(6 * T, n, device=d) for _ in range(2)]
    ws = torch.zeros(max(16, scan.workspace_bytes(n, T)), dtype=torch.uint8, device=d)
    jobs.append((n, T, a, ws))
g1, g2 = torch.rand(900, 700, device=d), torch.zeros(40, 700, device=d)
gws = torch.zeros(max(16, *(gemm.workspace_bytes(c) for c in (1, 5, 20, 700))), dtype=torch.uint8, device=d)
torch.cuda.synchronize()

def go():
    st = torch.cuda.current_stream().cuda_stream
    for n, T, a, ws in jobs:
        p = [t.data_ptr() for t in a]
        conv.run(n, T, p[0], p[5], stream=st)
        scan.run(n, T, p[0], p[1], p[2], p[3], p[6], workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=st)
    for c in (1, 5, 20, 700):
        gemm.run(c, g1.data_ptr(), g2.data_ptr(), ld_x=700, ld_y=700, workspace=gws.data_ptr(), workspace_bytes=gws.numel(), stream=st)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    go()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for _, _, a, _ in jobs for t in a[5:]] + [g2.clone()]
go()
torch.cuda.synchronize()
assert all(torch.equal(x, y) for x, y in zip(got, [t for _, _, a, _ in jobs for t in a[5:]] + [g2])) and g2.abs().sum() > 0
print("captured first")
"""


def test_the_first_run_of_a_process_can_be_captured():
    """Nothing is left to be loaded, allocated or set up at an operator's first run."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_RUN.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_runs_repeat_bit_for_bit():
    c = scan_case(3, 500, 16, 16, 1, True, True, True)
    a, b = run_scan(c), run_scan(c)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


# ---- refusals ---------------------------------------------------------------------------------------------------------
def test_run_refusals():
    conv = api.CausalConv(np.zeros((4, 4), np.float32))
    scan = api.SelectiveScan(np.zeros((4, 16), np.float32))
    gemm = api.Gemm8(np.zeros((8, 4), np.float32))
    buf = torch.zeros(1 << 16, device="cuda")
    p = lambda off: buf.data_ptr() + 4 * off  # noqa: E731

    def refused(code, f, *a, **k):
        with pytest.raises(api.RosennaError) as e:
            f(*a, **k)
        assert e.value.code == code, str(e.value)

    refused(api.ERR_ARG, conv.run, -1, 2, p(0), p(1000))
    refused(api.ERR_ARG, conv.run, 8, -2, p(0), p(1000))
    refused(api.ERR_ARG, conv.run, 8, 2, 0, p(1000))
    refused(api.ERR_ARG, conv.run, 8, 2, p(0), 0)
    refused(api.ERR_ARG, conv.run, 8, 2, p(0) + 2, p(1000))
    refused(api.ERR_SHAPE, conv.run, 8, 2, p(0), p(1000), ld_x=7)
    refused(api.ERR_SHAPE, conv.run, 1 << 38, 2, p(0), p(1000))
    refused(api.ERR_ARG, conv.run, 8, 2, p(0), p(0))
    refused(api.ERR_ARG, conv.run, 8, 2, p(0), p(1000), state_in=p(2000), state_out=p(2008))
    refused(api.ERR_ARG, conv.run, 8, 2, p(0), p(1000), state_out=p(1000))
    refused(api.ERR_ARG, conv.run, 8, 2, p(0), p(1000), state_in=p(1000))
    refused(api.ERR_ARG, scan.run, 8, 2, p(0), p(1000), p(2000), p(3000), p(3000))
    refused(api.ERR_ARG, scan.run, 8, 2, p(0), p(1000), p(2000), 0, p(4000))
    refused(api.ERR_ARG, scan.run, 1, 4096, p(0), p(0), p(0), p(0), p(65536 - 16384), workspace=p(0), workspace_bytes=16)
    refused(api.ERR_SHAPE, scan.run, 8, 2, p(0), p(1000), p(2000), p(3000), p(4000), ld_B=4)
    refused(api.ERR_SHAPE, gemm.run, 8, p(0), p(1000), ld_y=4)
    refused(api.ERR_ARG, gemm.run, 8, p(0), p(4))
    refused(api.ERR_ARG, conv.run, 8, 2, p(0), p(1000), lens=p(1004))
    refused(api.ERR_ARG, conv.run, 8, 2, p(0), p(1000), lens=p(5000) + 1)
    refused(api.ERR_ARG, scan.run, 1, 4096, p(0), p(0), p(0), p(0), p(65536 - 16384), workspace=p(60000), workspace_bytes=1 << 30)
    closed = api.Gemm8(np.zeros((8, 4), np.float32))
    closed.close()
    refused(api.ERR_ARG, closed.run, 8, p(0), p(1000))
    refused(api.ERR_ARG, api.CausalConv.run, scan, 8, 2, p(0), p(1000))
    with pytest.raises(api.RosennaError):
        gemm.workspace_bytes(-1)
    # nothing ran, and nothing to run is not refused
    conv.run(0, 5, 0, 0)
    scan.run(0, 5, 0, 0, 0, 0, 0)
    gemm.run(0, 0, 0)
    torch.cuda.synchronize()
    assert torch.all(buf == 0)
    # columns of one array side by side are not an overlap
    conv.run(8, 2, p(0), p(8), ld_x=16, ld_y=16, stream=stream())
    torch.cuda.synchronize()
