import os
import sys

import pytest

# CPU threads that wait for each other sleep instead of spinning (before torch loads its OpenMP runtime; child processes inherit it).  Several ranks with a
# thread per CPU each take turns on the CPUs, and a spinning thread keeps the one it waits for from running: the float64 CPU reference of three
# MobileNetV2 ranks, 8 threads each on 8 CPUs, 5.4 s instead of more than 300.
os.environ.setdefault("OMP_WAIT_POLICY", "PASSIVE")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")
    # a clean checkout has no built artefacts (they are git-ignored): build libaadg_hip.so (hipcc cross-compiles
    # without a GPU) and the oracle before collecting; both are no-ops when up to date
    try:
        from aadg_amd import build as _b
        _b.build_hip()
        from oracle import oracle as _o
        _o.build()
    except Exception as e:  # noqa: BLE001 -- tests that need the artefacts will fail loudly on their own
        print("conftest: build step failed: %s" % e)


@pytest.fixture(scope="session")
def oracle():
    from oracle import oracle as O
    O.lib()
    return O


@pytest.fixture(scope="session")
def hip():
    """The HIP path: fails loudly (never skips) when the library or the GPU is missing."""
    import torch
    from aadg_amd import _lib
    _lib.load()
    assert torch.cuda.is_available(), "gpu-marked tests need a GPU"
    return _lib
