"""The norm over all gradients of a model, and clipping by it (csrc/ct_gradnorm.hip).

    GradientSet(grads, out=None)            a list of gradient tensors that stay where they are, step after step
        .norm()  .clip(clip_norm)
    clip_by_global_norm(grads, clip_norm)   the same for a list that is used once

Keras' global_clipnorm: every gradient times clip_norm / max(norm, clip_norm); a norm that is not finite makes every value NaN."""
from __future__ import annotations

import ctypes as C
import math

from . import _dev, _lib
from .grouped import _capturing, _env, _no_grad

_captured: list = []          # the tables that a graph reads: it may be replayed after its set is gone (40 bytes a tensor each)


def _dense(a):
    """Whether the tensor fills the span of memory it lies in, whatever the order of its indices."""
    expect = 1
    for st, size in sorted((st, size) for size, st in zip(a.shape, a.stride()) if size > 1):
        if st != expect:
            return False
        expect *= size
    return True


def _checked(grads, out):
    t, kinds, _ = _env()
    grads = list(grads)
    out = grads if out is None else list(out)
    if len(out) != len(grads):
        raise ValueError(f"out: {len(out)} tensors for {len(grads)} gradients")
    device = None
    for i, (g, o) in enumerate(zip(grads, out)):
        for a in (g, o):
            if not isinstance(a, t.Tensor) or not a.is_cuda:
                raise ValueError(f"gradient {i}: expected a tensor on the GPU")
            if a.dtype not in kinds:
                raise ValueError(f"gradient {i}: values of type {a.dtype} are not supported (float32, bfloat16, float16)")
            device = a.device if device is None else device
            if a.device != device:
                raise ValueError(f"gradient {i}: is on {a.device}, others are on {device}")
            _no_grad(t, f"gradient {i}", a, ", but norm and clip are not part of torch's graph: pass it detached")
            if a.numel() and not _dense(a):
                raise ValueError(f"gradient {i}: shape {tuple(a.shape)} with strides {tuple(a.stride())} leaves gaps or overlaps itself")
        if g is not o and (g.dtype != o.dtype or g.shape != o.shape or (g.numel() > 1 and [s for n, s in zip(g.shape, g.stride()) if n > 1] !=
                                                                         [s for n, s in zip(o.shape, o.stride()) if n > 1])):
            raise ValueError(f"out {i}: {o.dtype} {tuple(o.shape)} {tuple(o.stride())} is not laid out as its gradient {g.dtype} {tuple(g.shape)} {tuple(g.stride())}")
    # what is written may be its own gradient, and meets nothing else
    spans = []
    for i, (g, o) in enumerate(zip(grads, out)):
        if not g.numel():
            continue
        size = g.numel() * g.element_size()
        spans.append((o.data_ptr(), o.data_ptr() + size, i, True))
        if g.data_ptr() != o.data_ptr():
            spans.append((g.data_ptr(), g.data_ptr() + size, i, False))
    spans.sort()
    reach, reach_written, who = 0, 0, None
    for begin, end, i, written in spans:
        if begin < (reach if written else reach_written):
            raise ValueError(f"gradient {i}: its memory is also that of gradient {who}; a tensor that is written must stand in the list once")
        if end > reach:
            reach, who = end, i
        if written:
            reach_written = max(reach_written, end)
    return grads, out, device


class GradientSet:
    """The gradients of one model as a list that .norm() and .clip() take whole: two launches for any number of tensors.

    grads: float32, bfloat16 and float16 tensors of one device, mixed as they come, of any shape (also without values); each must fill its
    memory (contiguous, or with its indices in another order).  out: where clip() writes, tensors of the same type and layout; left out,
    the gradients are clipped in place.  The set holds the tensors; it has to be made anew when one of them is replaced.  Making it waits for
    the current stream (the list is then ready for every stream), so it cannot be made while a graph is captured; its calls can be.  A set may
    be dropped while its calls are on their way on any stream; a graph that captured one needs the gradients and `out` to stay, as graphs do."""

    def __init__(self, grads, out=None):
        self._init(grads, out)
        if self._device is not None:
            _env()[0].cuda.current_stream(self._device).synchronize()

    def _init(self, grads, out, once=False):
        t, kinds, L = self._t, _, self._lib = _env()
        self.grads, self.out, self._device = _checked(grads, out)
        self._n = len(self.grads)
        if self._device is None:                              # an empty list: its norm is zero, on the current device
            self._device = t.device("cuda", t.cuda.current_device())
        if not once and _capturing(t, self._device):
            raise ValueError("GradientSet: make the set before the capture begins")
        n, m = self._n, max(self._n, 1)
        sizes = (C.c_int64 * m)(*[g.numel() for g in self.grads])
        types = (C.c_int * m)(*[kinds[g.dtype] for g in self.grads])
        ins = (C.c_void_p * m)(*[g.data_ptr() for g in self.grads])
        outs = (C.c_void_p * m)(*[o.data_ptr() for o in self.out])
        self._chunks = L.ct_gradset_chunks(n, sizes)
        self._keeps, self._streams = once, {t._C._cuda_getCurrentRawStream(self._device.index)}
        with t.cuda.device(self._device):
            self._table = _dev.workspace(L.ct_gradset_table_bytes(n), self._device)
            _lib.check(L.ct_gradset_write(n, ins, outs, sizes, types, self._table.data_ptr(), self._table.numel(), _dev.stream(self._device)),
                       "ct_gradset_write")
        self._ws, self._at = L.ct_gradset_workspace_bytes(), self._table.data_ptr()

    def _used_on(self, t, stream):
        """The memory that a call on a stream other than the list's own reads and writes is not handed out again before that stream is through"""
        current = t.cuda.current_stream()
        for a in {id(a): a for a in (self._table, *self.grads, *self.out)}.values():
            a.record_stream(current)
        self._streams.add(stream)

    def _call(self, call, *args):
        t, device = self._t, self._device
        if t._C._cuda_getDevice() != device.index:
            with t.cuda.device(device):
                return self._call(call, *args)
        stream = t._C._cuda_getCurrentRawStream(device.index)
        if t._C._cuda_isCurrentStreamCapturing():
            if not self._keeps:
                _captured.append(self._table)
                self._keeps = True
        elif stream not in self._streams:
            self._used_on(t, stream)
        # the scalar and the partial sums, new for each call: two streams, or two graphs, share none
        scalar, ws = t.empty((), dtype=t.float32, device=device), t.empty(self._ws, dtype=t.uint8, device=device)
        rc = call(self._at, self._n, self._chunks, *args, scalar.data_ptr(), ws.data_ptr(), self._ws, stream)
        if rc:
            _lib.check(rc, call.__name__)
        return scalar

    def norm(self):
        """The l2 norm over all values, a float32 scalar on the device (asynchronous)."""
        return self._call(self._lib.ct_gradset_norm)

    def clip(self, clip_norm: float):
        """Scale the gradients to at most `clip_norm` (into `out`, or in place) -> their norm before that, a float32 scalar on the device."""
        clip_norm = float(clip_norm)
        if not (clip_norm > 0.0 and math.isfinite(clip_norm)):
            raise ValueError(f"clip_norm must be positive and finite, got {clip_norm}")
        return self._call(self._lib.ct_gradset_clip, clip_norm)


def clip_by_global_norm(grads, clip_norm: float, out=None):
    """-> (clipped gradients, norm): a GradientSet that is used once, on the current stream, without waiting for it (so it can be captured).
    out: as for GradientSet; left out, the gradients are clipped in place and returned."""
    one = GradientSet.__new__(GradientSet)
    one._init(grads, out, once=True)
    return one.out, one.clip(clip_norm)
