import os
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

GOLDEN = Path(__file__).resolve().parent / "golden"


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a) and the built extension")


def pytest_runtest_setup(item):
    """vLLM keeps its first answer to questions that environment variables decide (functools.cache).  Tests set their own, so
    no answer stays from one test to the next, in any order."""
    module = sys.modules.get("vllm.utils.deep_gemm")
    for f in list(vars(module).values()) if module is not None else ():
        clear = getattr(f, "cache_clear", None)
        if callable(clear):
            clear()


def cuda_ok() -> bool:
    try:
        import torch

        return torch.cuda.is_available()
    except Exception:  # pragma: no cover
        return False


@pytest.fixture(scope="session")
def golden():
    import numpy as np

    def load(name):
        return dict(np.load(GOLDEN / f"{name}.npz"))

    return load
