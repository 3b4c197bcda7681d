"""Host-side mirror of the reference's ``CellTracker/ffn.py`` inference surface.

    FFN()                      reference ffn.py:225-265 (callable, .predict, .load_weights)
    initial_matching_ffn(...)  reference ffn.py:268-327
    normalize_points(...)      reference ffn.py:330-374

The kNN shape features, the two dense layers and the all-pairs score kernel run in
csrc/ct_match.hip.  The (m*n) x 122 pair grid the reference tiles on the host is never built
(it is only materialised when a *foreign* model object exposing `.predict` is passed in).
"""
from __future__ import annotations

import ctypes as C
import threading
from pathlib import Path
from typing import Tuple, Union

import numpy as np

from . import _dev, _lib
from .arch import FFN_FEAT, FFN_K_PTRS

RATIO_SEG_ERROR = 0.15
FFN_WEIGHTS_NAME = "weights_training_"
k_ptrs = FFN_K_PTRS
NUMBER_FEATURES = FFN_FEAT


def flatten_ffn_weights(w: dict) -> np.ndarray:
    parts = [w["w1"]] + [w["bn1"][k] for k in ("gamma", "beta", "mean", "var")] + [w["w2"]] + \
            [w["bn2"][k] for k in ("gamma", "beta", "mean", "var")] + [w["w3"], w["b3"]]
    return np.ascontiguousarray(np.concatenate([np.asarray(p, dtype=np.float32).ravel() for p in parts]))


class _Loaded:
    """A handle of the library as ctypes passes it.  A call that was given it keeps it: it is destroyed when the last one has returned, not when
    other weights take its place (its memory is freed behind everything that the device has been asked to do by then)."""

    def __init__(self, handle):
        self._as_parameter_ = handle
        self._destroy = _lib.lib().ct_ffn_destroy

    def __del__(self):
        self._destroy(self._as_parameter_)


class FFN:
    """Dense(61->512, no bias)+BN+LeakyReLU shared by both halves, concat, Dense(1024->512, no
    bias)+BN+LeakyReLU, Dense(512->1)+sigmoid -- evaluated by the HIP library."""

    def __init__(self, device: int | None = None):
        self._loaded = None            # the library's handle (_Loaded)
        self._stale = False            # the training weights are ahead of it
        self._training = None
        self._device = device
        self._weights = None
        self._lock = threading.RLock()         # held wherever the weights change: training steps, uploads, new weights

    def __getstate__(self):                    # (a model without weights can be copied and sent to a worker; a handle refuses)
        return {k: v for k, v in self.__dict__.items() if k != "_lock"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._lock = threading.RLock()

    @property
    def _handle(self):
        if self._stale:
            with self._lock:                   # (matches run on several host threads: the first one brings the weights, the others wait)
                if self._stale:
                    with _lib.require_gpu().cuda.device(self._device):       # (creating a handle makes its device current: loading weights does, reading them does not)
                        self._upload(self._training.weights())
                    self._stale = False
        return self._loaded

    def set_weights_dict(self, w: dict):
        with self._lock:
            self._upload(w)                    # (weights that do not fit are refused: everything is as it was then, training too)
            self._training, self._stale = None, False
            return self

    def _upload(self, w: dict):
        t = _lib.require_gpu()
        if self._device is None:
            self._device = t.cuda.current_device()
        flat = flatten_ffn_weights(w)
        L = _lib.lib()
        if flat.size != L.ct_ffn_num_weights():
            raise ValueError(f"FFN weight count {flat.size} != {L.ct_ffn_num_weights()}")
        h = C.c_void_p()
        _lib.check(L.ct_ffn_create(flat.ctypes.data, flat.size, self._device, C.byref(h)), "ct_ffn_create")
        self._loaded = _Loaded(h)
        self._weights = w
        return self

    def load_weights(self, path):
        path = Path(path)
        if not path.exists():
            raise OSError(f"Unable to open file {path}")
        if path.suffix == ".npz":
            z = np.load(path)
            w = {"w1": z["w1"], "w2": z["w2"], "w3": z["w3"], "b3": z["b3"],
                 "bn1": {k: z[f"bn1_{k}"] for k in ("gamma", "beta", "mean", "var")},
                 "bn2": {k: z[f"bn2_{k}"] for k in ("gamma", "beta", "mean", "var")}}
            return self.set_weights_dict(w)
        try:
            import h5py  # noqa: F401
        except ImportError as e:
            raise OSError(f"cannot read {path}: Keras .h5 import needs h5py, which is not installed") from e
        from .keras_h5 import read_ffn_h5
        return self.set_weights_dict(read_ffn_h5(path))

    def compile(self, learning_rate: float = 1e-3, beta_1: float = 0.9, beta_2: float = 0.999, epsilon: float = 1e-7, global_clipnorm: float | None = None):
        """Start training from the present weights: Adam, binary cross-entropy, all gradients clipped together by `global_clipnorm` (Keras' names and
        defaults; the loop around it, reference ffn.py:56-222, is the caller's)."""
        from .ffn_training import FFNTraining
        with self._lock:
            self._require()
            self._training = FFNTraining(self._weights, f"cuda:{self._device}", learning_rate, beta_1, beta_2, epsilon, global_clipnorm)

    def train_on_batch(self, x, y) -> float:
        """One update from x -- (P,122), or the two halves [ (P,61), (P,61) ] -- and labels y (P,) or (P,1) in [0, 1]; numpy or torch -> the loss
        before it.  predict() and the matching calls use the new weights."""
        t = _lib.require_gpu()
        if self._training is None:
            raise ValueError("FFN is not being trained: call compile() first")
        if isinstance(x, (list, tuple)):
            x = t.cat([_dev.to_dev(h, t.float32, f"cuda:{self._device}") for h in x], dim=1)
        x = _dev.to_dev(x, t.float32, f"cuda:{self._device}")
        y = _dev.to_dev(y, t.float32, f"cuda:{self._device}").reshape(-1)
        if x.ndim != 2 or x.shape[1] != 2 * FFN_FEAT or x.shape[0] < 2 or y.shape[0] != x.shape[0]:
            raise ValueError(f"expected at least two rows (P, {2 * FFN_FEAT}) and as many labels, got {tuple(x.shape)} and {tuple(y.shape)}")
        with self._lock:
            if self._training is None:
                raise ValueError("FFN is not being trained: its weights were replaced meanwhile")
            with t.cuda.device(x.device):
                loss = self._training.step(x, y)
            self._stale = True
            return float(loss)                                            # (waits for the update: weights() may read it on another stream)

    def save_weights(self, path):
        with self._lock:
            self._handle                                                  # (training weights come back first)
            w = self._weights
        if w is None:
            raise ValueError("model has no weights")
        out = {"w1": w["w1"], "w2": w["w2"], "w3": w["w3"], "b3": w["b3"]}
        for b in ("bn1", "bn2"):
            for k in ("gamma", "beta", "mean", "var"):
                out[f"{b}_{k}"] = w[b][k]
        np.savez(path, **out)

    def _require(self):
        if self._handle is None:
            raise ValueError("FFN has no weights: call load_weights() or set_weights_dict() first")

    def pairgrid_device(self, feat_ref_d, feat_tgt_d):
        """feat_* fp32 device [n][61], [m][61] -> corr fp32 device [m][n] (async)."""
        t = _lib.require_gpu(); L = _lib.lib()
        self._require()
        n, m = feat_ref_d.shape[0], feat_tgt_d.shape[0]
        corr = _dev.empty((m, n), t.float32, feat_ref_d.device)
        ws = _dev.workspace(L.ct_ffn_workspace_bytes(n, m), feat_ref_d.device)
        _lib.check(L.ct_ffn_pairgrid(self._handle, feat_ref_d.data_ptr(), n, feat_tgt_d.data_ptr(), m, corr.data_ptr(),
                                     ws.data_ptr(), ws.numel(), _dev.stream(feat_ref_d.device)), "ct_ffn_pairgrid")
        return corr

    def predict(self, x, batch_size=None, verbose=0, **_):
        """x: (P,122) array, or the legacy two-input list [ (P,61), (P,61) ] (track.py:175) -> (P,1) float32."""
        t = _lib.require_gpu(); L = _lib.lib()
        self._require()
        if isinstance(x, (list, tuple)):
            x = np.concatenate([np.asarray(x[0]), np.asarray(x[1])], axis=1)
        x = np.asarray(x)
        if x.ndim != 2 or x.shape[1] != 2 * FFN_FEAT:
            raise ValueError(f"expected input of shape (P, {2 * FFN_FEAT}), got {x.shape}")
        out = np.empty((x.shape[0], 1), dtype=np.float32)
        handle = self._handle                  # one for all pieces: a training step beside them does not mix two sets of weights in one result
        step = 1 << 18
        for s in range(0, x.shape[0], step):
            xd = _dev.to_dev(x[s:s + step], t.float32, f"cuda:{self._device}")
            rows = xd.shape[0]
            od = _dev.empty((rows,), t.float32, xd.device)
            ws = _dev.workspace(L.ct_ffn_predict_workspace_bytes(rows), xd.device)
            _lib.check(L.ct_ffn_predict(handle, xd.data_ptr(), rows, od.data_ptr(), ws.data_ptr(), ws.numel(),
                                        _dev.stream(xd.device)), "ct_ffn_predict")
            out[s:s + rows, 0] = od.cpu().numpy()
        return out

    __call__ = predict


def initial_matching_device(ffn_model: FFN, ref_d, tgt_d, k: int = FFN_K_PTRS):
    """ref_d, tgt_d: fp64 device [n][3], [m][3] -> corr fp32 device [m][n]."""
    return ffn_model.pairgrid_device(_dev.knn_features(ref_d, k), _dev.knn_features(tgt_d, k))


def initial_matching_ffn(ffn_model, ref: np.ndarray, tgt: np.ndarray, k_ptrs: int, two_inputs: bool = False) -> np.ndarray:
    """reference ffn.py:268-327 -> (m, n) float32, corr[t, r]."""
    ref_d, tgt_d = _dev.points_dev(ref), _dev.points_dev(tgt)
    if isinstance(ffn_model, FFN):
        return initial_matching_device(ffn_model, ref_d, tgt_d, k_ptrs).cpu().numpy()
    # foreign model object: features on the GPU, pair grid laid out exactly like the reference's
    fr = _dev.knn_features(ref_d, k_ptrs).cpu().numpy()
    ft = _dev.knn_features(tgt_d, k_ptrs).cpu().numpy()
    n, m = fr.shape[0], ft.shape[0]
    left = np.broadcast_to(fr[None], (m, n, fr.shape[1])).reshape(m * n, -1)
    right = np.broadcast_to(ft[:, None], (m, n, ft.shape[1])).reshape(m * n, -1)
    grid = [left, right] if two_inputs else np.concatenate([left, right], axis=1)
    return np.reshape(ffn_model.predict(grid, batch_size=1024), (m, n))


def normalize_points(points: np.ndarray, return_para: bool = False) -> Union[np.ndarray, Tuple[np.ndarray, Tuple]]:
    """reference ffn.py:330-374: centre, divide by 3 x std (ddof 0) of the projection on the first principal axis
    (device kernel: mean, 3x3 scatter matrix, largest eigenvalue by Jacobi rotations)."""
    points = np.asarray(points)
    if points.ndim != 2:
        raise ValueError(f"Points should be a 2D table, but get {points.ndim}D")
    if points.shape[1] != 3:
        raise ValueError(f"Points should have 3D coordinates, but get {points.shape[1]}D")
    out_d, para_d = _dev.normalize_points(_dev.points_dev(points))
    para = para_d.cpu().numpy()
    norm_points = out_d.cpu().numpy()
    return (norm_points, (para[:3].copy(), float(para[3]))) if return_para else norm_points
