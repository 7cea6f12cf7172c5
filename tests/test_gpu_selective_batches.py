"""Selective models over batches that are run in pieces, and the width that its fp32 Gemms hold."""
import numpy as np
import pytest
import torch

from oracle import parity
from rosenna_b200 import api
from tests.test_gpu_selective import device_model, reference
from tests.test_selective_host import write

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device():
    assert torch.cuda.is_available(), "gpu tests need a CUDA device"
    api.set_devices([0])
    yield
    api.finalize()
    torch.cuda.empty_cache()


def on_device(x, states=()):
    n = x.shape[0]
    ins, outs = device_model(n, [x, *states])
    api.use_model_device(n, [t.data_ptr() for t in ins], [t.data_ptr() for t in outs], torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return [o.cpu().numpy().T for o in outs]


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("n", [16385, 40001])
def test_host_pieces(tmp_path, n, eight_bit):
    """The host entry point cuts these into pieces, the last of them smaller; samples do not depend on one another."""
    T, width = 3, 8
    mods, head = write(tmp_path, 1, width, T, eight_bit=eight_bit)
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, T, width)).astype(np.float32)
    states = [rng.standard_normal((n, r, mods[0].channels)).astype(np.float32) for r in (3, 16)]
    api.initialize(str(tmp_path))
    got = api.use_model([x] + states)
    for g, d in zip(got, on_device(x, states)):
        assert np.array_equal(g, d)
    if not eight_bit:
        for g, w in zip(got, reference(mods, head, x, states, "last")):
            r = parity.compare(g, w)
            assert r["ok"], parity.describe(r)


@pytest.mark.parametrize("eight_bit", [False, True])
def test_device_pieces(tmp_path, eight_bit):
    """More intermediates than a call may allocate (16 GB at most): each piece equals a call of its own."""
    T, width, n = 2000, 64, 3000
    write(tmp_path, 1, width, T, eight_bit=eight_bit, with_state=False)
    if torch.cuda.mem_get_info()[0] < 80e9:
        pytest.skip("needs 80 GB of device memory")
    api.initialize(str(tmp_path))
    x = torch.randn((width, T, n), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    y = torch.zeros((5, n), device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    api.use_model_device(n, [x.data_ptr()], [y.data_ptr()], st)
    pieces = api.last_launch_count()
    torch.cuda.synchronize()
    # the same samples, a call for each eighth: 375 samples of 128 channels are too many for their scan to be split over
    # time, as is the first piece.  The last piece may be of a few samples and split, so the last eighth is left out
    for a in range(0, n - n // 8, n // 8):
        k = n // 8
        part, out = x[..., a:a + k].contiguous(), torch.zeros((5, k), device="cuda")
        api.use_model_device(k, [part.data_ptr()], [out.data_ptr()], st)
        torch.cuda.synchronize()
        if a == 0:
            assert pieces > api.last_launch_count()  # more than one piece
        assert torch.equal(out, y[:, a:a + k])


def test_width_that_the_fp32_gemms_hold(tmp_path):
    """An in-projection of at most 880 outputs: width 220.  Wider layers run with 8-bit Gemms only."""
    T, n = 2, 5
    for width, eight_bit, runs in ((220, False, True), (221, False, False), (221, True, True), (512, True, True)):
        d = tmp_path / f"{width}{eight_bit}"
        mods, head = write(d, 1, width, T, eight_bit=eight_bit, with_state=False)
        api.check_model(str(d))
        if not runs:
            with pytest.raises(api.RosennaError) as e:
                api.initialize(str(d))
            assert e.value.code == api.ERR_UNSUPPORTED and "too wide" in str(e.value)
            continue
        api.initialize(str(d))
        x = np.random.default_rng(1).standard_normal((n, T, width)).astype(np.float32)
        got = api.use_model([x])[0]
        want = reference(mods, head, x, [], "last")[0]
        assert np.isfinite(got).all()
        if not eight_bit:  # (those are compared with their operators one by one elsewhere)
            r = parity.compare(got, want)
            assert r["ok"], parity.describe(r)
