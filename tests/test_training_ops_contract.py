"""What the training-step operators promise beyond their values, as far as it shows without a GPU."""
import contextlib
import types

import pytest
import torch

from opus_b200 import _lib, ops


# ============================================================================ errors recorded on the device
class Devices:
    """Two devices with an error word each, in the place of torch's and the library's."""

    def __init__(self, monkeypatch):
        self.current, self.words, self.launched = 0, {0: 0, 1: 0}, []
        monkeypatch.setattr(torch.cuda, "device", self.device)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: self.current, raising=False)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
        monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(opus_fake=self.launch))
        monkeypatch.setattr(_lib, "device_error", self.take)
        monkeypatch.setattr(ops, "_devices", set())

    @contextlib.contextmanager
    def device(self, index):
        before, self.current = self.current, index
        yield
        self.current = before

    def launch(self, code, stream):
        self.launched.append((self.current, stream))
        self.words[self.current] = code
        return 0

    def take(self, tokens=True):
        code, self.words[self.current] = self.words[self.current], 0
        return code


def test_errors_of_another_device_are_reported(monkeypatch):
    d = Devices(monkeypatch)
    ops._call("opus_fake", 1, 0x202)
    assert d.launched == [(1, 101)] and d.current == 0
    with pytest.raises(IndexError, match="token"):
        ops.check_device_error()
    ops.check_device_error()
    with d.device(1):  # a backward's thread, say
        ops._call("opus_fake", 1, 0x202)
    with pytest.raises(IndexError, match="token"):
        ops.check_device_error()
    ops._call("opus_fake", 0, 0x107)
    ops._call("opus_fake", 1, 0x202)
    with pytest.raises(RuntimeError, match="0x107"):
        ops.check_device_error()
    with pytest.raises(IndexError):  # not lost to the other's
        ops.check_device_error()
    assert d.words == {0: 0, 1: 0} and d.current == 0
