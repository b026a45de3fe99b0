import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG_PY = os.path.join(REPO, "batmobile-evo_amd", "python")
for p in (REPO, PKG_PY):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP kernels)")


def gpu_available():
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


# Modules that hand C entries addresses that lead nowhere, to be refused
HOST_CALLS = ("test_abi", "test_block_host", "test_layers_host", "test_host_no_gpu")


@pytest.hookimpl(trylast=True)                  # behind the choice by -m and -k
def pytest_collection_modifyitems(config, items):
    if not any("gpu" in item.keywords for item in items) or not gpu_available():
        os.environ["HIP_VISIBLE_DEVICES"] = "-1"    # a lost refusal ends as an error code, not on a GPU
        skip = pytest.mark.skip(reason="no GPU in this environment")
        bad = [item for item in items if "gpu" in item.keywords]
    else:
        skip = pytest.mark.skip(reason='its addresses lead nowhere: run with -m "not gpu", without a GPU')
        bad = [item for item in items if item.module.__name__ in HOST_CALLS]
    for item in bad:
        item.add_marker(skip)


@pytest.fixture(scope="session")
def bm():
    """The compiled extension; fails loudly when it is not built."""
    import torch  # noqa: F401
    import _batmobile
    return _batmobile


@pytest.fixture(scope="session")
def dev():
    import torch
    return torch.device("cuda:0")
