import sys
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
PKG_ROOT = ROOT / "transformers-qwen3-moe-fused_b200"
for p in (str(ROOT), str(PKG_ROOT)):
    if p not in sys.path:
        sys.path.insert(0, p)

GOLDEN = ROOT / "tests" / "golden"


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run with -m gpu on a B200)")


@pytest.fixture(scope="session")
def golden():
    def load(name: str):
        return np.load(GOLDEN / f"{name}.npz")

    return load


@pytest.fixture(scope="session")
def cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def kernel_choice_restored(request):
    """A GPU test that fails while it forces a kernel family does not hand that on to the next one."""
    yield
    if request.node.get_closest_marker("gpu"):
        lib = sys.modules.get("qwen3_moe_fused._lib")
        if lib is not None and lib._lib is not None:
            lib.set_gemm_path(lib.PATH_AUTO)
