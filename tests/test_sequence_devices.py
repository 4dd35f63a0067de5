"""Arrays of another GPU are refused before a kernel can reach for them: `DeviceArray`s know their
device, as other libraries' arrays do."""
import numpy as np
import pytest

from salt_b200 import device as D
from salt_b200 import sequence

AT = 1 << 20


class SomeLibrarys:
    device = "cuda:1"


def on(device, *shape):
    """An array of that device's memory that is never read; None: a pointer from elsewhere."""
    owner = object.__new__(D._Allocation)
    owner.device = device
    return D.DeviceArray(AT, shape, np.float32, owner)


@pytest.mark.parametrize("name", ["x", "weight", "out", "residual", "rstd"])
def test_norm_refuses_arrays_of_another_device(monkeypatch, name):
    monkeypatch.setattr(sequence, "_here", lambda: 0)
    shape = {"weight": (8,), "rstd": (2,)}
    arrays = {k: on(0, *shape.get(k, (2, 8))) for k in ("x", "weight", "out", "residual", "rstd")}
    arrays[name] = on(1, *shape.get(name, (2, 8)))
    with pytest.raises(ValueError, match=f"{name}: not on the current device"):
        sequence.rms_norm(**arrays)


def test_views_keep_their_device():
    a = on(1, 4, 8)
    assert a[1:3].device == a[2].device == a.view(np.int32).device == 1
    assert D.DeviceArray(AT, (4,), np.float32, None).device is None
    assert D.DeviceArray(AT, (4,), np.float32, SomeLibrarys()).device is None


def test_views_of_another_device_are_refused(monkeypatch):
    monkeypatch.setattr(sequence, "_here", lambda: 0)
    with pytest.raises(ValueError, match="x: not on the current device"):
        sequence.rms_norm(on(1, 3, 2, 8)[1], on(0, 8), out=on(0, 2, 8))


@pytest.mark.gpu
def test_allocations_know_their_device():
    here = D.current_device()
    a = D.zeros((3, 4), np.float32)
    assert a.device == here and a[1:].device == here
    assert D.to_device(np.ones(3), np.float32).device == here
