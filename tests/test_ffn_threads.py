"""CPU-only: the matching network's weights when training steps, uploads and matches meet on several host threads (the library and the training
step are stand-ins that say when they run)."""
import contextlib
import ctypes
import importlib
import threading

import numpy as np
import pytest

ffn_mod = importlib.import_module("3deecelltracker_amd.ffn")
_dev = importlib.import_module("3deecelltracker_amd._dev")
_lib = importlib.import_module("3deecelltracker_amd._lib")
WAIT = 0.3          # how long a thread is given to do what it must not do


class Training:
    """Counts steps; `during_step` and `during_weights` run in the middle of either"""

    def __init__(self):
        self.version, self.stepping, self.torn = 0, False, 0
        self.during_step = self.during_weights = lambda: None

    def step(self, x, y):
        self.stepping = True
        self.version += 1
        self.during_step()
        self.stepping = False
        return 0.5

    def weights(self):
        self.torn += self.stepping
        version = self.version
        self.during_weights()
        return {"version": version}


@pytest.fixture
def model(monkeypatch):
    import torch
    monkeypatch.setattr(_lib, "require_gpu", lambda: torch)
    monkeypatch.setattr(_dev, "to_dev", lambda a, dtype, device=None: torch.as_tensor(a, dtype=dtype))
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    m = ffn_mod.FFN(device=0)

    def upload(w):
        m._loaded, m._weights = ("handle", w.get("version")), w
        return m
    monkeypatch.setattr(m, "_upload", upload)
    m._training = Training()
    return m


def _step(m):
    m.train_on_batch(np.zeros((2, 122), np.float32), np.zeros(2, np.float32))


def _beside(call):
    """call() on another thread, given some time; -> the thread"""
    t = threading.Thread(target=call)
    t.start()
    t.join(WAIT)
    return t


def test_a_step_during_an_upload_is_not_lost(model):
    _step(model)
    threads = []

    def once():
        model._training.during_weights = lambda: None
        threads.append(_beside(lambda: _step(model)))
    model._training.during_weights = once
    first = model._handle                                  # brings step 1; step 2 arrives while it is being copied
    threads[0].join()
    assert first[1] in (1, 2) and model._training.version == 2
    assert model._handle == ("handle", 2)


def test_weights_are_not_copied_in_the_middle_of_a_step(model):
    _step(model)
    threads, seen = [], []

    def once():
        model._training.during_step = lambda: None
        threads.append(_beside(lambda: seen.append(model._handle)))
    model._training.during_step = once
    _step(model)
    threads[0].join()
    assert model._training.torn == 0 and model._handle == ("handle", 2) and seen == [("handle", 2)]


def test_the_update_is_waited_for_before_another_thread_may_copy_it(model):
    """The loss comes from the training thread's stream; until it is there, the update may still run"""
    threads = []

    class Loss:
        def __float__(self):
            threads.append(_beside(lambda: model._handle))
            assert model._loaded is None, "copied before the update was waited for"
            return 0.5
    model._training.step = lambda x, y: Loss()
    _step(model)
    threads[0].join()
    assert model._loaded == ("handle", 0)


class Library:
    """Handles as numbers; a call reports which of them live while it runs"""

    def __init__(self):
        self.alive, self.made, self.inside = set(), 0, None
        keep = self

        class Entry:
            def __call__(self, handle, *rest):
                ctypes.c_void_p.from_param(handle)         # what ctypes asks of an argument
                number = getattr(handle, "_as_parameter_", handle).value
                if keep.inside:
                    keep.inside()
                assert number in keep.alive, f"handle {number} was destroyed during a call"
                return 0
        self.ct_ffn_pairgrid = Entry()
        self.ct_ffn_predict = lambda handle, *rest: self.asked.append(handle._as_parameter_.value) or (self.inside and self.inside()) or 0
        self.asked = []

    def ct_ffn_num_weights(self):
        return 3

    def ct_ffn_workspace_bytes(self, n, m):
        return 16

    def ct_ffn_predict_workspace_bytes(self, rows):
        return 16

    def ct_ffn_create(self, w, n, device, out):
        self.made += 1
        self.alive.add(self.made)
        out._obj.value = self.made
        return 0

    def ct_ffn_destroy(self, handle):
        self.alive.discard(getattr(handle, "value", handle))


@pytest.fixture
def library(monkeypatch):
    import torch
    lib = Library()
    monkeypatch.setattr(_lib, "require_gpu", lambda: torch)
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(_dev, "stream", lambda d: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(ffn_mod, "flatten_ffn_weights", lambda w: np.zeros(w["size"], np.float32))
    return lib


def test_a_match_in_flight_keeps_its_weights(library):
    import torch
    m = ffn_mod.FFN(device=0)
    m.set_weights_dict({"size": 3})
    library.inside = lambda: m.set_weights_dict({"size": 3})
    m.pairgrid_device(torch.zeros(4, 61), torch.zeros(4, 61))
    library.inside = None
    assert library.alive == {2}                            # and the first handle is gone once the call has returned
    m.pairgrid_device(torch.zeros(4, 61), torch.zeros(4, 61))
    del m
    assert library.alive == set()


def test_weights_that_are_refused_change_nothing(library):
    m = ffn_mod.FFN(device=0)
    m.set_weights_dict({"size": 3})
    m._training = training = Training()
    training.weights = lambda: {"size": 3, "trained": True}
    m._stale = True                                        # a step ahead of the library's handle
    with pytest.raises(ValueError):
        m.set_weights_dict({"size": 4})
    assert m._training is training
    assert m._handle._as_parameter_.value == 2 and m._weights["trained"]


def test_reading_the_handle_leaves_the_current_device_alone(library, monkeypatch):
    import torch
    current = [0]

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d
        yield
        current[0] = before
    create = library.ct_ffn_create

    def create_there(w, n, where, out):
        current[0] = where                                 # what the library does
        return create(w, n, where, out)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(library, "ct_ffn_create", create_there)
    m = ffn_mod.FFN(device=3)
    m.set_weights_dict({"size": 3})
    assert current == [3]                                  # (as ever: points that are uploaded next go where the weights are)
    m._training = Training()
    m._training.weights = lambda: {"size": 3}
    current[0], m._stale = 1, True
    assert m._handle is not None and current == [1] and library.made == 2


def test_a_model_without_weights_can_be_copied(library):
    import copy
    import pickle
    for m in (copy.deepcopy(ffn_mod.FFN(device=0)), pickle.loads(pickle.dumps(ffn_mod.FFN(device=0)))):
        m.set_weights_dict({"size": 3})
        assert m._handle is not None and m._device == 0


def test_a_prediction_in_pieces_has_one_set_of_weights(library, monkeypatch):
    import torch
    monkeypatch.setattr(_dev, "to_dev", lambda a, dtype, device=None: torch.as_tensor(a, dtype=dtype))
    m = ffn_mod.FFN(device=0)
    m.set_weights_dict({"size": 3})
    library.inside = lambda: m.set_weights_dict({"size": 3}) and None      # what a training step on another thread amounts to
    m.predict(np.zeros(((1 << 18) + 1, 122), np.float32))
    assert library.asked == [1, 1] and library.alive == {3}
