"""The 8-bit Gemm on values near the ends of fp32's range: a finite column whose result is finite gives it,
through every kernel (up to 8 columns, columns kept on chip, columns quantised ahead)."""
import numpy as np
import pytest
import torch

from rosenna_b200 import api
from tests import ops_reference as ref
from tests.test_gpu_ops import FILL, check, dev, host, ptr, stream

pytestmark = pytest.mark.gpu

SIZES = [(1, 300), (2, 300), (4, 300), (8, 300), (9, 300), (300, 300), (20, 1300)]  # columns, K


def run(w, x, b=None):
    n, M = x.shape[1], w.shape[0]
    op = api.Gemm8(w, b)
    tx, y = dev(x), torch.full((M, n), FILL, device="cuda")
    ws = torch.zeros(op.workspace_bytes(n) + 16, dtype=torch.uint8, device="cuda")
    op.run(n, ptr(tx), ptr(y), workspace=ptr(ws), workspace_bytes=ws.numel(), stream=stream())
    return host(y, (M, n))


@pytest.mark.parametrize("n,K", SIZES)
@pytest.mark.parametrize("size", [1e36, 1e37])
def test_large_columns_and_small_weights(n, K, size):
    """|x| up to about 5e37: neither a value nor any partial sum of the result leaves fp32, but 448 |x| would."""
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((K, n)) * size).astype(np.float32)
    w = (0.01 * rng.standard_normal((40, K)) / np.sqrt(K)).astype(np.float32)
    want, tol = ref.gemm8(w, x)
    assert np.abs(want).max() < 1e37
    check(run(w, x), want, tol, "y")


@pytest.mark.parametrize("n,K", SIZES)
@pytest.mark.parametrize("wmax,xmax", [(2.0 ** 100, 2.0 ** 100), (57344.0, 3.4e38), (57345.0, 3.4e38)])
def test_rows_of_zeros_beside_large_weights(n, K, wmax, xmax):
    """The product of a block's two scales is beyond fp32 (2^92 by 2^92, 2^8 by 2^120; 2^7 by 2^120 is just within);
    what it multiplies is 0 in these rows."""
    rng = np.random.default_rng(n + 1)
    x = (rng.uniform(-1, 1, (K, n)) * xmax).astype(np.float32)
    x[::100] = xmax
    w = (rng.uniform(-1, 1, (40, K)) * wmax).astype(np.float32)
    w[0, ::100] = wmax
    w[3], w[17] = 0, 0
    b = rng.standard_normal(40).astype(np.float32)
    got = run(w, x, b)
    assert np.array_equal(got[3], np.full(n, b[3], np.float64)) and np.array_equal(got[17], np.full(n, b[17], np.float64))


@pytest.mark.parametrize("n,K", SIZES)
def test_large_weights_and_small_columns(n, K):
    """Weights around 1e36 by columns around 1e-3: the scales' product is ordinary."""
    rng = np.random.default_rng(n + 2)
    x = (1e-3 * rng.standard_normal((K, n))).astype(np.float32)
    w = (1e36 * rng.standard_normal((40, K)) / np.sqrt(K)).astype(np.float32)
    want, tol = ref.gemm8(w, x)
    check(run(w, x), want, tol, "y")


@pytest.mark.parametrize("n,K", [(5, 200), (300, 300), (20, 1300)])
def test_rows_of_zeros_in_a_model(tmp_path, n, K):
    """The same through a model's entry."""
    from tests.test_gpu_plan_entries import load

    rng = np.random.default_rng(n + 3)
    w = (rng.uniform(-1, 1, (12, K)) * 2.0 ** 100).astype(np.float32)
    w[3] = 0
    b = rng.standard_normal(12).astype(np.float32)
    api.set_devices([0])
    try:
        load(tmp_path, lambda g, v: [(g.add("Gemm8", [v, g.weight(w), g.weight(b)], [[1, 12]], {"params": [0, 0]})[0], [1, 12])], 0, K)
        got = api.use_model([(rng.uniform(-1, 1, (n, K)) * 2.0 ** 100).astype(np.float32)])[0]
    finally:
        api.finalize()
    assert np.array_equal(got[:, 3], np.full(n, b[3]))
