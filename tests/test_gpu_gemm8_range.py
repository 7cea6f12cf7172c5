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
