"""CPU-only: what cannot be done while a graph is captured is refused by the stream of the tensors' device, whichever device is current."""
import contextlib
import importlib

import pytest

grouped = importlib.import_module("3deecelltracker_amd.grouped")
gradients = importlib.import_module("3deecelltracker_amd.gradients")


class Device:
    def __init__(self, index):
        self.index = index


class Torch:
    """Two devices; `captured` is the one whose current stream is being captured"""
    current, captured = 0, 0
    int32 = "int32"

    class Tensor:
        pass

    def __init__(self):
        outer = self

        class C:
            _cuda_getDevice = staticmethod(lambda: outer.current)
            _cuda_isCurrentStreamCapturing = staticmethod(lambda: outer.current == outer.captured)

        @contextlib.contextmanager
        def device(d):
            before, outer.current = outer.current, d.index
            yield
            outer.current = before

        class Cuda:
            is_current_stream_capturing = C._cuda_isCurrentStreamCapturing
        Cuda.device = staticmethod(device)
        self._C, self.cuda = C, Cuda

    def tensor(self, values, **kw):
        class Uploaded:
            to = staticmethod(lambda *a, **k: list(values))
        return Uploaded()


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("device", [0, 1])
def test_offsets_on_the_host(monkeypatch, current, device):
    t = Torch()
    t.current = current
    monkeypatch.setattr(grouped, "_env", lambda: (t, {}, None))
    if device == t.captured:
        with pytest.raises(ValueError, match="captured"):
            grouped.offsets_device([0, 2, 3], 2, 3, Device(device))
    else:
        assert grouped.offsets_device([0, 2, 3], 2, 3, Device(device)) == [0, 2, 3]
    assert t.current == current


@pytest.mark.parametrize("current", [0, 1])
def test_a_gradient_set(monkeypatch, current):
    t = Torch()
    t.current = current
    monkeypatch.setattr(gradients, "_env", lambda: (t, {}, None))
    monkeypatch.setattr(gradients, "_checked", lambda g, o: ([], [], Device(0)))
    with pytest.raises(ValueError, match="capture"):
        gradients.GradientSet([])


@pytest.mark.parametrize("offsets", [[0, 2.5, 10], [0, float("nan"), 10], [0, float("inf"), 10], [0, None, 10], [[0, 2], [2, 10], [10, 10]], [0, "2", 10]], ids=str)
def test_offsets_that_are_not_whole_numbers(monkeypatch, offsets):
    """None of them may be rounded in silence"""
    monkeypatch.setattr(grouped, "_env", lambda: (Torch(), {}, None))
    with pytest.raises(ValueError, match="whole numbers"):
        grouped.offsets_device(offsets, 2, 10, Device(1))


@pytest.mark.parametrize("offsets", [[0, 2, 10], (0, 2, 10), [0.0, 2.0, 10.0], "int64", "float64"], ids=str)
def test_offsets_that_are(monkeypatch, offsets):
    import numpy as np
    monkeypatch.setattr(grouped, "_env", lambda: (Torch(), {}, None))
    if isinstance(offsets, str):
        offsets = np.array([0, 2, 10], dtype=offsets)
    got = grouped.offsets_device(offsets, 2, 10, Device(1))
    assert got == [0, 2, 10] and all(type(v) is int for v in got)
