"""The greedy assignment in one persistent launch against a launch for every phase, on ordinary streams (test_gpu_match.py has the same beside streams
that are restricted to four CUs, which not every machine grants), and what a refused stream leaves behind."""
import ctypes as C
import importlib
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
REPO = Path(__file__).resolve().parent.parent
_lib = importlib.import_module("3deecelltracker_amd._lib")

CHILD = r"""
import sys, importlib, numpy as np, torch
sys.path.insert(0, sys.argv[1])
_dev = importlib.import_module("3deecelltracker_amd._dev")
rng = np.random.default_rng(11)
cases = [rng.uniform(0, 1, s).astype(np.float32) for s in ((600, 600), (540, 600), (600, 431), (113, 90), (25, 21), (1, 7), (2000, 2000))]
cases += [np.round(rng.uniform(0, 1, (300, 300)) * 8).astype(np.float32) / 8, np.full((64, 64), 0.05, np.float32)]       # ties everywhere; none above the threshold
out = {}
for i, c in enumerate(cases):
    for mode in (0, 1):
        pairs, n, prior = _dev.greedy_match(torch.from_numpy(c).cuda(), 0.1 if mode == 0 else 0.5, mode)
        out[f"pairs {i} {mode}"] = pairs[:int(n.item())].cpu().numpy()
        out[f"prior {i} {mode}"] = prior.cpu().numpy()
np.savez(sys.argv[2], **out)
"""


def test_one_launch_equals_a_launch_for_every_phase(tmp_path):
    found = []
    for form in ("1", "0"):
        path = str(tmp_path / f"{form}.npz")
        r = subprocess.run([sys.executable, "-c", CHILD, str(REPO), path], capture_output=True, text=True, timeout=300, env=dict(os.environ, CT_GREEDY_PERSISTENT=form), cwd=REPO)
        assert r.returncode == 0, r.stderr[-2000:]
        found.append(np.load(path))
    assert sorted(found[0].files) == sorted(found[1].files) and len(found[0].files) == 36
    for k in found[0].files:
        assert np.array_equal(found[0][k], found[1][k]), k
    assert len(found[0]["pairs 0 0"]) > 300 and len(found[0]["pairs 8 0"]) == 0


def test_a_stream_that_is_refused_leaves_no_error_behind():
    import torch
    grouped = importlib.import_module("3deecelltracker_amd.grouped")
    L, stream = _lib.lib(), C.c_void_p()
    x, w, off = torch.ones(3, 8, device="cuda"), torch.ones(1, 8, 4, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    rc = L.ct_stream_create_cu_range(0, 0, 4, C.byref(stream))
    assert bool((grouped.product(x, w, off) == 8).all())                 # (a launch reports the last error of its thread)
    if rc == 0:
        assert L.ct_stream_destroy(stream) == 0
