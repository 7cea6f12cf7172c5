"""Selective scans whose states grow (A > 0, or steps of either sign without softplus): split over time or not, a
finite state stays finite."""
import numpy as np
import pytest

from tests.test_gpu_ops import check, run_scan, scan_case, scan_reference

pytestmark = pytest.mark.gpu


def growing(n, T, D, N, state, ragged=False):
    c = scan_case(n, T, D, N, 1, state, False, ragged)
    c["dt_bias"] = c["skip"] = None
    return c


@pytest.mark.parametrize("n,T,D", [(1, 700, 40), (3, 200, 5), (64, 200, 6)])
@pytest.mark.parametrize("state", [False, True])
def test_growth_of_nothing(n, T, D, state):
    """Zero inputs until the last two steps: the state is 0 until then, while a chunk's factor is e^144 or more."""
    c = growing(n, T, D, 16, state)
    c["A"] = np.full((D, 16), 3.0, np.float32)
    c["dt"][:] = 3.0
    c["x"][:, :T - 2] = 0
    if state:
        c["h0"][:] = 0
    # (the bounds of all T steps would grow as the states may: these are of the steps that hold something)
    last = {k: np.ascontiguousarray(v[..., T - 2:, :]) if k in ("x", "dt", "B", "C") else v for k, v in c.items()}
    want, tol, hw, htol = scan_reference(last, use_softplus=False)
    assert np.isfinite(hw).all() and np.isfinite(tol).all() and np.isfinite(htol).all()
    y, hn, need = run_scan(c, softplus=False)
    assert need > 0
    assert np.all(y[:, :T - 2] == 0)
    check(y[:, T - 2:], want, tol, "y")
    check(hn, hw, htol, "hn")


@pytest.mark.parametrize("n,D", [(1, 40), (64, 6)])
def test_growth_of_a_tiny_state_and_its_decay(n, D):
    """A chunk's factor beyond fp32 (e^102, then e^-102) over states that are not: 1e-30 -> 2e14 -> 1e-30.  Steps and A
    are small multiples of powers of two, so that every sum of them is exact."""
    T = 34  # two chunks
    c = growing(n, T, D, 4, True)
    c["A"] = np.full((D, 4), 2.0, np.float32)
    c["dt"][:, :17], c["dt"][:, 17:] = 3.0, -3.0
    c["x"][:] = 0
    c["h0"] = (c["h0"] * 1e-30).astype(np.float32)
    want, tol, hw, htol = scan_reference(c, use_softplus=False)
    y, hn, need = run_scan(c, softplus=False)
    assert need > 0
    check(y, want, tol, "y")
    check(hn, hw, htol, "hn")


@pytest.mark.parametrize("n,T,D", [(3, 200, 5), (64, 200, 6)])
@pytest.mark.parametrize("ragged", [False, True])
def test_parts_that_cancel(n, T, D, ragged):
    """The first step takes the state to exactly 0 (1024 - 1024), where it stays until the last two; what the chunk makes
    of the state and of the input alone are both beyond fp32 (2^170 and -2^170)."""
    c = growing(n, T, D, 16, True)
    if ragged:
        c["lens"] = np.full(n, T, np.int32)
        c["lens"][::2] = 9
    A = np.float32(6.931472)
    assert A * np.float32(1.4426950408889634) == 10  # e^A is 2^10 as the kernels take it
    c["A"] = np.full((D, 16), A)
    c["dt"][:] = 1.0
    c["h0"][:] = 1.0
    c["x"][:, :T - 2], c["x"][:, 0], c["B"][:, :, 0] = 0, -1, 1024
    last = {k: np.ascontiguousarray(v[..., T - 2:, :]) if k in ("x", "dt", "B", "C") else v for k, v in c.items()}
    last["h0"] = None
    if ragged:
        last["lens"] = np.maximum(c["lens"] - (T - 2), 0).astype(np.int32)
    want, tol, hw, htol = scan_reference(last, use_softplus=False)
    for workspace in (True, False):
        y, hn, need = run_scan(c, softplus=False, workspace=workspace)
        assert (need > 0) == workspace
        inside = np.arange(T - 2)[:, None] < (c["lens"] if ragged else np.full(n, T))[None]
        assert np.all(y[:, :T - 2][:, inside] == 0)
        check(y[:, T - 2:], want, tol, "y")
        check(hn, hw, htol, "hn")


@pytest.mark.parametrize("n,T,D,ragged", [(1, 700, 40, False), (5, 300, 12, True), (64, 300, 8, True)])
@pytest.mark.parametrize("scale", [0.3, 1.0, 3.0])
def test_finite_unsplit_is_finite_split(n, T, D, ragged, scale):
    """Steps and A of either sign and any growth."""
    c = growing(n, T, D, 16, True, ragged)
    rng = np.random.default_rng(int(10 * scale))
    c["A"] = (scale * rng.standard_normal((D, 16))).astype(np.float32)
    y, hn, need = run_scan(c, softplus=False)
    yu, hu, _ = run_scan(c, softplus=False, workspace=False)
    assert need > 0 and np.isfinite(hu).any()
    assert not (np.isfinite(yu) & ~np.isfinite(y)).any() and not (np.isfinite(hu) & ~np.isfinite(hn)).any()
