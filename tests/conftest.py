import importlib
import os
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent
if str(REPO) not in sys.path:
    sys.path.insert(0, str(REPO))
os.environ.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
# the frame-loop tests keep 5-6 HIP streams busy: more hardware queues than the default 4 (read when HIP initialises; the package itself only warns)
os.environ.setdefault("GPU_MAX_HW_QUEUES", "16")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


# tests that need a stream restricted to some of the CUs; a machine may refuse those (hipExtStreamCreateWithCUMask: out of memory)
CU_MASK_TESTS = ("test_persistent_greedy_equals_the_launch_per_phase_form",)


def pytest_runtest_setup(item):
    if getattr(item, "originalname", item.name) in CU_MASK_TESTS:
        import ctypes as C
        import torch
        lib = importlib.import_module("3deecelltracker_amd._lib").lib()
        if not torch.cuda.is_available():
            return
        stream = C.c_void_p()
        rc = lib.ct_stream_create_cu_range(0, 0, 4, C.byref(stream))
        if rc:
            pytest.skip(f"this machine refuses streams with a CU mask: {lib.ct_error_string(rc).decode()} (the same without masked streams: test_greedy_forms.py)")
        lib.ct_stream_destroy(stream)


@pytest.fixture(scope="session")
def ct():
    """The product package (its directory name is not a Python identifier)."""
    return importlib.import_module("3deecelltracker_amd")


@pytest.fixture(scope="session")
def golden_dir():
    return REPO / "tests" / "golden"
