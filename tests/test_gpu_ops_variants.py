"""Every compiled variant of the scan's kernels and every mode of the 8-bit Gemm: the sizes that tests/test_gpu_ops.py
leaves out, and the rule that tells which mode a size takes."""
import numpy as np
import pytest

from tests.test_gpu_ops import GEMM, check, run_scan, scan_case, scan_reference, test_gemm8 as run_gemm8

pytestmark = pytest.mark.gpu

SCAN = [  # n, T, D, N, G, state, gate, lens, ld extra
    # histories of many samples, with 9 to 15, 17 to 31 and more than 32 states; 16-byte rows and not; split and not
    (128, 40, 17, 12, 1, True, True, True, 0), (129, 37, 9, 12, 1, True, False, True, 3), (256, 20, 18, 9, 2, False, True, True, 4),
    (256, 40, 6, 24, 2, True, True, True, 0), (100, 33, 5, 24, 1, False, True, False, 1), (640, 30, 130, 17, 1, True, True, True, 0),
    (128, 70, 4, 33, 1, True, True, True, 4), (70, 41, 3, 33, 1, True, False, False, 5), (96, 130, 4, 64, 2, True, True, True, 0),
    (65, 90, 3, 64, 1, False, False, True, 2), (512, 30, 40, 50, 1, True, True, True, 0), (1100, 9, 70, 64, 1, False, True, True, 1),
    (300, 33, 3, 2, 3, True, True, True, 0), (300, 66, 5, 32, 1, True, True, True, 1),
    # few samples
    (5, 300, 7, 12, 1, True, True, True, 0), (1, 65, 140, 10, 7, True, False, False, 0), (47, 40, 9, 64, 3, True, True, True, 1),
    (40, 130, 5, 9, 1, False, True, True, 0), (23, 100, 13, 32, 1, True, True, True, 0), (9, 70, 31, 2, 1, True, True, False, 0),
    # single steps: four samples a thread, one, few samples
    (40000, 1, 20, 24, 1, True, True, True, 0), (40000, 1, 20, 32, 2, True, False, True, 0), (40000, 1, 20, 8, 1, True, True, True, 0),
    (40000, 1, 20, 12, 1, False, True, True, 4), (40001, 1, 18, 33, 1, True, True, True, 0), (2000, 1, 7, 48, 1, True, True, True, 2),
    (130, 1, 7, 32, 1, True, True, True, 0), (130, 1, 7, 4, 1, True, True, True, 0), (130, 1, 7, 8, 7, True, False, True, 0),
    (3, 1, 50, 12, 1, True, True, False, 0), (3, 1, 50, 24, 2, True, True, True, 0), (17, 1, 6, 32, 1, False, True, True, 1),
    (2, 1, 9, 4, 1, True, False, False, 0), (2, 1, 9, 8, 3, True, True, True, 0),
]


@pytest.mark.parametrize("n,T,D,N,G,state,gate,ragged,extra", SCAN)
def test_scan(n, T, D, N, G, state, gate, ragged, extra):
    c = scan_case(n, T, D, N, G, state, gate, ragged)
    want, tol, hw, htol = scan_reference(c)
    y, hn, need = run_scan(c, n + extra)
    check(y, want, tol, "y")
    check(hn, hw, htol + 1e-37, "hn")
    if need:
        y, hn, _ = run_scan(c, n + extra, workspace=False)
        check(y, want, tol, "y unsplit")
        check(hn, hw, htol + 1e-37, "hn unsplit")
    if state:
        _, hn, _ = run_scan(c, n + extra, in_place=True)
        check(hn, hw, htol + 1e-37, "hn in place")


MORE = [  # n, K, M, bias, act, ld extra
    # weights streamed, columns on chip: one range and several, odd and even block counts, several items a CTA
    (512, 640, 300, True, "none", 0), (600, 512, 512, False, "relu", 0), (20001, 900, 260, True, "none", 0),
    (19100, 1100, 140, True, "silu", 3), (20001, 384, 600, True, "none", 0), (300, 512, 1400, True, "none", 0),
    # weights resident, several output tiles, several items a CTA
    (20001, 130, 640, True, "none", 0), (25000, 384, 256, False, "tanh", 1),
    # columns quantised ahead, several items a CTA
    (19100, 1300, 300, True, "none", 0), (700, 1290, 2100, True, "none", 1),
]


@pytest.mark.parametrize("n,K,M,bias,act,extra", MORE)
def test_gemm8(n, K, M, bias, act, extra):
    run_gemm8(n, K, M, bias, act, extra)


def mode(n, K, M):
    """The rule of gemm8.cu on 148 SMs: (mode, whether some CTA takes several items for certain)."""
    nkb, nmt, tiles = -(-K // 128), -(-M // 128), -(-n // 128)
    if n <= 8:
        return "few", False
    if nkb > 9 or (nkb >= 6 and 2 * tiles <= 148):
        return "ahead", tiles > 148
    return "resident" if nkb * nmt + nkb <= 13 else "streamed", tiles > 148


def test_every_mode_is_run():
    modes = {mode(*c[:3]) for c in GEMM + MORE}
    assert modes == {("few", False)} | {(m, several) for m in ("ahead", "resident", "streamed") for several in (False, True)}
