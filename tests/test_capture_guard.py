"""CPU: the guard that refuses a capture beside a living eager graph of the same leaf (_lib.record), with the streams and the capture state of two devices
stood in for: device 0 is current, the tensors (on the CPU, index -1) play those of another device."""
import contextlib
import sys
import threading

import pytest
import torch
from torch.autograd import Function

from combo_avs_amd import _lib


class Twice(Function):
    @staticmethod
    def forward(ctx, x):
        return 2 * x

    @staticmethod
    def backward(ctx, dy):
        return 2 * dy


@pytest.fixture
def devices(monkeypatch):
    """-> state: the raw stream and the capture state of device 0 (current) and of device -1 (the tensors')"""
    state = {"current": 0, "stream": {0: 7, -1: 0}, "capturing": {0: False, -1: False}}

    @contextlib.contextmanager
    def device(index):
        before, state["current"] = state["current"], index
        yield
        state["current"] = before
    monkeypatch.setattr(_lib, "_current_device", lambda: state["current"])
    monkeypatch.setattr(_lib, "_raw_stream", lambda index: state["stream"][index])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"][state["current"]])
    return state


def test_streams_of_the_tensors_device_count(devices):
    x = torch.ones(3, requires_grad=True)
    alive = _lib.record(Twice, x)  # the default stream of the tensors' device, another one on the current device
    devices["capturing"][-1] = True
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        _lib.record(Twice, x)
    del alive
    _lib.record(Twice, x)
    assert devices["current"] == 0


def test_streams_of_the_current_device_do_not(devices):
    devices["stream"] = {0: 0, -1: 7}
    x = torch.ones(3, requires_grad=True)
    alive = _lib.record(Twice, x)  # recorded on a stream of its own
    devices["capturing"][-1] = True
    assert torch.equal(_lib.record(Twice, x), alive)
    devices["stream"], devices["capturing"] = {0: 7, -1: 0}, {0: True, -1: False}  # a capture on the current device, the tensors are elsewhere
    again = _lib.record(Twice, x)
    assert torch.equal(_lib.record(Twice, x), again)


def test_other_threads_may_record_meanwhile(devices, monkeypatch):
    """the guard looks through the living graphs while other threads add theirs"""
    here = threading.get_ident()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: threading.get_ident() == here)
    monkeypatch.setattr(_lib, "_current_device", lambda: -1)
    leaf, other = torch.ones(1, requires_grad=True), torch.ones(1, requires_grad=True)
    done, wrong = threading.Event(), []

    def work():
        try:
            while not done.is_set():
                alive = [_lib.record(Twice, other) for _ in range(50)]
                del alive
        except Exception as e:
            wrong.append(e)
    threads = [threading.Thread(target=work) for _ in range(2)]
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        for t in threads:
            t.start()
        for _ in range(2000):
            _lib.record(Twice, leaf)
    finally:
        done.set()
        for t in threads:
            t.join()
        sys.setswitchinterval(interval)
    assert not wrong
