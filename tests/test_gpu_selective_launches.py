"""Launches of a selective model at other batch sizes than the first: its Gemms over a sequence stay one launch each."""
import numpy as np
import pytest
import torch

from rosenna_b200 import api
from tests.test_gpu_selective import device_model
from tests.test_selective_host import write

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight_bit", [False, True])
def test_launches_do_not_grow_with_fewer_samples(tmp_path, eight_bit):
    """Width 16: every K is one block of 128, so no columns are quantised ahead, and 6 steps are not split over time: the
    count is the same for every batch."""
    T, width = 6, 16
    write(tmp_path, 2, width, T, eight_bit=eight_bit, with_state=False)
    assert torch.cuda.is_available()
    api.set_devices([0])
    api.initialize(str(tmp_path))
    try:
        counts = []
        for n in (1000, 1, 333, 1000, 20):
            x = np.random.default_rng(n).standard_normal((n, T, width)).astype(np.float32)
            ins, outs = device_model(n, [x])
            st = torch.cuda.current_stream().cuda_stream
            for fn in (api.use_model_device, api.use_model_device_noalloc):
                fn(n, [t.data_ptr() for t in ins], [t.data_ptr() for t in outs], st)
                counts.append(api.last_launch_count())
        torch.cuda.synchronize()
        assert len(set(counts)) == 1, counts
    finally:
        api.finalize()


def test_steps_are_labelled_by_what_may_run_them(tmp_path):
    """Which kernel runs one of these steps depends on the batch: the label names the file, not one kernel."""
    write(tmp_path, 1, 16, 6, eight_bit=True, with_state=False)
    api.set_devices([0])
    api.initialize(str(tmp_path))
    try:
        names = [name for name, _ in api.step_info()]
    finally:
        api.finalize()
    assert sum("gemm8.cu" in x for x in names) == 4 and sum("seq_ops.cu" in x for x in names) == 2, names
    assert not any(x in ("gemm8_tc_kernel", "causal_conv_kernel") for x in names)
