"""Export of selective layers at the ends of what it takes: a convolution of one tap has no state; what cannot be a
model is refused before a file is written."""
import numpy as np
import pytest
import torch

from rosenna_b200 import api, selective
from tests.test_selective_host import write


@pytest.mark.parametrize("with_state", [False, True])
@pytest.mark.parametrize("eight_bit", [False, True])
def test_one_tap(tmp_path, with_state, eight_bit):
    write(tmp_path, 2, taps=1, with_state=with_state, eight_bit=eight_bit)
    desc = api.check_model(str(tmp_path))
    assert desc.count("W=1 silu state b-1->b-1") == 2, desc
    with open(tmp_path / "variables.fpp") as f:
        text = f.read()
    assert text.count("'scan_state") == (4 if with_state else 0) and "conv_state" not in text


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 6])
def test_one_tap_on_the_gpu(tmp_path, T):
    from oracle import parity

    assert torch.cuda.is_available()
    (m,), head = write(tmp_path, 1, 12, T, taps=1)
    rng = np.random.default_rng(T)
    x, h = rng.standard_normal((33, T, 12)).astype(np.float32), rng.standard_normal((33, 16, 24)).astype(np.float32)
    api.set_devices([0])
    api.initialize(str(tmp_path))
    try:
        got = api.use_model([x, h])
    finally:
        api.finalize()
    y, c, hn = m.double()(torch.from_numpy(x).double(), scan_state=torch.from_numpy(h).double())
    assert c.shape[1] == 0 and len(got) == 2
    for g, w in zip(got, (hn, torch.nn.Sequential(*head).double()(y[:, -1]))):
        r = parity.compare(g, w.detach().numpy())
        assert r["ok"], parity.describe(r)


def test_what_cannot_be_a_model_is_refused():
    ly = selective.SelectiveLayer(12)
    for args in (([], [], 1, 5), ([ly, selective.SelectiveLayer(10)], [], 1, 5), ([ly], [], 1, 0), ([ly], [], 0, 5), ([ly], [], 1, 5, "all"),
                 ([ly], [torch.nn.Tanh()], 1, 5, "y")):
        with pytest.raises(ValueError):
            selective.export_selective(*args)
