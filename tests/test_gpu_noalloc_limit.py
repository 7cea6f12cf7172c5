"""The allocation-free entry point's limit on the batch counts the 8-bit Gemm's workspace: the number in its refusal runs."""
import re

import numpy as np
import pytest
import torch

from rosenna_b200 import api
from tests.test_gpu_plan_entries import load

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers", [1, 2])
def test_the_limit_in_the_message_runs(tmp_path, layers):
    """K = 1300: columns are quantised ahead, 1.4 KB each; with one layer there is no other intermediate at all."""
    K, M = 1300, 8
    z = np.ones

    def build(b, v):
        if layers == 2:
            v = b.add("Gemm8", [v, b.weight(z((K, K), np.float32)), b.weight(z(K, np.float32))], [[1, K]], {"params": [0, 0]})[0]
        return [(b.add("Gemm8", [v, b.weight(z((M, K), np.float32)), b.weight(z(M, np.float32))], [[1, M]], {"params": [0, 0]})[0], [1, M])]

    api.set_devices([0])
    try:
        load(tmp_path, build, 0, K)
        n = 100_000
        x, y, st = torch.ones((K, n), device="cuda"), torch.zeros((M, n), device="cuda"), torch.cuda.current_stream().cuda_stream
        with pytest.raises(api.RosennaError) as e:
            api.use_model_device_noalloc(n, [x.data_ptr()], [y.data_ptr()], st)
        assert e.value.code == api.ERR_SHAPE
        fits = int(re.search(r"at most about (\d+) samples", str(e.value)).group(1))
        assert 5_000 < fits < n
        api.use_model_device_noalloc(fits, [x.data_ptr()], [y.data_ptr()], st)
        torch.cuda.synchronize()
        want = (K * K + K + 1) if layers == 2 else K + 1
        assert torch.all((y.view(-1)[:M * fits] - want).abs() <= 2.0 ** -4 * want)
        with pytest.raises(api.RosennaError):
            api.use_model_device_noalloc(fits + 1, [x.data_ptr()], [y.data_ptr()], st)
    finally:
        api.finalize()
