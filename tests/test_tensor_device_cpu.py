"""A wrapper of the C ABI refuses tensors on different devices and says which."""
import pytest
import torch

from c3_b200 import _lib


class _On(torch.Tensor):
    device_index = -1

    def get_device(self):
        return self.device_index


def _on(index):
    t = torch.zeros(2).as_subclass(_On)
    t.device_index = index
    return t


@_lib.on_tensor_device
def op(*args, **kwargs):
    return "called"


def test_the_devices_are_named():
    assert op(torch.zeros(2), [torch.zeros(1)], x=None) == "called"
    for args, kwargs in (((_on(2), _on(0)), {}), (([_on(2)], torch.zeros(1)), {"dY": (_on(0), None)}),
                         ((), {"a": _on(0), "b": [_on(0), _on(2)]})):
        with pytest.raises(_lib.C3CUError) as e:
            op(*args, **kwargs)
        assert e.value.code == -1 and "different devices: cuda:[0, 2]" in str(e.value)
    with pytest.raises(_lib.C3CUError, match=r"cuda:\[0, 1, 2\]"):
        op(_on(2), _on(0), _on(1))
