"""_lib.on_device on a machine without a GPU: a launch goes to the device of the tensor."""
import contextlib

import torch

from operators import _lib


class _On:
    def __init__(self, index):
        self.index = index
        self.device = torch.device("cuda", index)

    def get_device(self):
        return self.index


def test_the_tensors_device_is_made_current(monkeypatch):
    entered = []

    @contextlib.contextmanager
    def device(d):
        entered.append(d)
        yield
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", device)
    with _lib.on_device(_On(0)):
        pass
    assert entered == []
    with _lib.on_device(_On(1)):
        pass
    assert entered == [torch.device("cuda", 1)]
