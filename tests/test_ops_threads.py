"""The operators' calls beside a call of the model in another thread: they do not wait for it, and each thread's status
and message are its own.  A model call is held up by a model file that is a pipe nobody has written to yet."""
import os
import threading

import numpy as np
import pytest

from rosenna_b200 import api
from tests.test_selective_host import write


def refused():
    """-> status of an operator's call that needs no GPU to be refused."""
    with pytest.raises(api.RosennaError) as e:
        api.CausalConv(np.zeros((3, 9), np.float32))
    assert "taps" in str(e.value)
    return e.value.code


def in_thread(f, seconds):
    """-> (whether f returned in time, what it returned)"""
    out = []
    t = threading.Thread(target=lambda: out.append(f()), daemon=True)
    t.start()
    t.join(seconds)
    return not t.is_alive(), out[0] if out else None


def test_operators_do_not_wait_for_a_model_call(tmp_path):
    write(tmp_path)
    model, pipe = tmp_path / "onnxModel.txt", str(tmp_path / "pipe")
    text = model.read_text()
    os.mkfifo(pipe)
    model.unlink()
    os.symlink(pipe, model)
    result = []
    call = threading.Thread(target=lambda: result.append(api.check_model(str(tmp_path))), daemon=True)
    call.start()
    with open(pipe, "w") as f:  # (opens when the call opens its end, which it does with its lock held)
        done, code = in_thread(refused, 20)
        f.write(text)
    call.join(60)
    assert not call.is_alive() and "causal_conv" in result[0]
    assert done and code == api.ERR_UNSUPPORTED


def test_each_thread_has_its_own_status(tmp_path):
    L = api.lib()

    def model_call():
        with pytest.raises(api.RosennaError) as e:
            api.check_model(str(tmp_path))  # no files there
        return e.value.code

    assert model_call() == api.ERR_IO
    message = L.rosenna_last_error()
    assert message and L.rosenna_last_status() == api.ERR_IO

    def other():
        code = refused()
        return code, L.rosenna_last_status(), b"taps" in L.rosenna_last_error()

    assert in_thread(other, 20) == (True, (api.ERR_UNSUPPORTED, api.ERR_UNSUPPORTED, True))
    assert L.rosenna_last_status() == api.ERR_IO and L.rosenna_last_error() == message
    # a thread that has called nothing sees the model's; so does this one after its next model call
    assert in_thread(L.rosenna_last_status, 20) == (True, api.ERR_IO)
    refused()
    assert L.rosenna_last_status() == api.ERR_UNSUPPORTED and b"taps" in L.rosenna_last_error()
    assert model_call() == api.ERR_IO and L.rosenna_last_error() == message
