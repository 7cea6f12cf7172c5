"""States of a model's operators come in the operators' layout, (batch, taps - 1, channels) and (batch, states, channels):
the same number of values in another shape is another order of them, and refused."""
import os

import pytest

from rosenna_b200 import api
from tests.test_selective_host import write


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("name,right,wrong", [("conv_state0", [1, 3, 24], [1, 24, 3]), ("conv_state0", [1, 3, 24], [1, 72]),
                                              ("scan_state0", [1, 16, 24], [1, 24, 16]), ("scan_state0", [1, 16, 24], [1, 2, 8, 24])])
def test_states_of_another_shape_are_refused(tmp_path, name, right, wrong, eight_bit):
    write(tmp_path, eight_bit=eight_bit)
    api.check_model(str(tmp_path))
    p = os.path.join(str(tmp_path), "variables.fpp")
    with open(p) as f:
        text = f.read()
    entry = f"['{name}', {right}]"
    assert entry in text
    with open(p, "w") as f:
        f.write(text.replace(entry, f"['{name}', {wrong}]"))
    with pytest.raises(api.RosennaError) as e:
        api.check_model(str(tmp_path))
    assert e.value.code == api.ERR_SHAPE and "state must be" in str(e.value)
