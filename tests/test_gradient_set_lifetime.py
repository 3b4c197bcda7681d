"""CPU-only: what GradientSet tells the allocator.  Its table holds the addresses that the kernels write to, so the memory must stay the table's while a
stream or a graph may still read it.  Torch, the library and the tensors are stand-ins that note what they are asked."""
import contextlib
import gc
import importlib
import weakref

import pytest

gradients = importlib.import_module("3deecelltracker_amd.gradients")


class Tensor:
    def __init__(self, where=64):
        self.where, self.streams = where, []

    def record_stream(self, s):
        self.streams.append(s)

    def numel(self):
        return 4

    def data_ptr(self):
        return self.where

    dtype = "float32"


class Device:
    index = 0


class Torch:
    """One device; `stream` is the current one, `capturing` whether it is captured"""
    stream, capturing, float32, uint8 = 1, False, "float32", "uint8"

    def __init__(self):
        outer = self

        class C:
            _cuda_getDevice = staticmethod(lambda: 0)
            _cuda_getCurrentRawStream = staticmethod(lambda index: outer.stream)
            _cuda_isCurrentStreamCapturing = staticmethod(lambda: outer.capturing)

        class Cuda:
            device = staticmethod(lambda d: contextlib.nullcontext())
            is_current_stream_capturing = staticmethod(lambda: outer.capturing)

            @staticmethod
            def current_stream(d=None):
                class S:
                    synchronize = staticmethod(lambda: None)
                    cuda_stream = outer.stream

                    def __eq__(self, other):
                        return self.cuda_stream == getattr(other, "cuda_stream", other)
                return S()
        self._C, self.cuda = C, Cuda

    def empty(self, *a, **k):
        return Tensor()


class Library:
    ct_gradset_table_bytes = staticmethod(lambda n: 40 * (n + 1))
    ct_gradset_workspace_bytes = staticmethod(lambda: 64)
    ct_gradset_chunks = staticmethod(lambda n, sizes: n)
    ct_gradset_write = staticmethod(lambda *a: 0)
    ct_gradset_norm = staticmethod(lambda *a: 0)
    ct_gradset_clip = staticmethod(lambda *a: 0)


@pytest.fixture
def t(monkeypatch):
    t = Torch()
    monkeypatch.setattr(gradients, "_env", lambda: (t, {"float32": 0}, Library))
    monkeypatch.setattr(gradients, "_checked", lambda g, o: (list(g), list(g if o is None else o), Device))
    monkeypatch.setattr(gradients._dev, "workspace", lambda n, d=None: Tensor())
    monkeypatch.setattr(gradients._dev, "stream", lambda d=None: t.stream)
    return t


def test_the_list_is_held_for_every_stream_that_reads_it(t):
    g, o = Tensor(), Tensor(128)
    s = gradients.GradientSet([g], out=[o])
    s.clip(1.0)
    assert s._table.streams == [] and g.streams == []      # its own stream: the allocator knows
    for stream in (2, 3, 2, 1):
        t.stream = stream
        s.clip(1.0); s.norm()
    for a in (s._table, g, o):
        assert a.streams == [2, 3]


def test_a_graph_keeps_the_list_that_it_reads(t):
    before = len(gradients._captured) if hasattr(gradients, "_captured") else 0
    s, plain = gradients.GradientSet([Tensor()]), gradients.GradientSet([Tensor()])
    plain.clip(1.0)
    t.capturing = True
    s.clip(1.0); s.norm()
    gradients.clip_by_global_norm([Tensor()], 1.0)         # its table is the graph's own and written by the graph
    t.capturing = False
    held, dropped = weakref.ref(s._table), weakref.ref(plain._table)
    del s, plain
    gc.collect()
    assert held() is not None and dropped() is None
    assert len(gradients._captured) == before + 1
    gradients._captured.pop()


@pytest.mark.gpu
def test_a_set_that_is_dropped_while_another_stream_clips():
    import torch
    big = torch.randn(4096, 4096, device="cuda")
    grads = [torch.full((n,), 3.0, device="cuda") for n in (100003, 5, 4099)]
    out = [torch.empty_like(g) for g in grads]
    s = gradients.GradientSet(grads, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(30):
            big = big @ big * 1e-4                         # some ms of work in front of the clip
        norm = s.clip(1.0)
    where, size = s._table.data_ptr(), s._table.numel()
    del s
    others = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(50)]
    assert side.query() or all(o.data_ptr() != where for o in others)
    torch.cuda.synchronize()
    want = 3.0 * sum(g.numel() for g in grads) ** 0.5
    assert abs(float(norm) - want) <= want * 2.0 ** -23
    assert all(bool(((o * norm - 3.0).abs() <= 3.0 * 2.0 ** -21).all()) for o in out)


@pytest.mark.gpu
def test_a_graph_that_outlives_its_set():
    import torch
    grads = [torch.ones(n, device="cuda") for n in (100003, 5, 4099)]
    out = [torch.zeros_like(g) for g in grads]
    s = gradients.GradientSet(grads, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = s.clip(1.0)
    size = s._table.numel()
    del s
    others = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(50)]
    for value in (2.0, 0.001, 5.0):
        for g in grads:
            g.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        want = value * sum(g.numel() for g in grads) ** 0.5
        assert abs(float(norm) - want) <= want * 2.0 ** -23
        assert all(bool(((o * max(want, 1.0) - value).abs() <= value * 2.0 ** -21).all()) for o in out)
    assert all(bool((o == 255).all()) for o in others)
