import gc
import os
import sys

import pytest

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (os.path.join(_ROOT, "legate-boost_amd"), os.path.join(_ROOT, "tests"), _ROOT):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


def pytest_collection_modifyitems(config, items):
    # GPU tests are only meaningful where a device exists; everything else runs on CPU.
    try:
        import torch

        has_gpu = torch.cuda.is_available()
    except Exception:  # pragma: no cover
        has_gpu = False
    if has_gpu:
        return
    skip = pytest.mark.skip(reason="no GPU in this environment")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(autouse=True, scope="module")
def _nothing_is_left_to_the_next_module():
    """Device memory that a module's tests have left in reference cycles, and the scratch that the calls keep, is given back at its end:
    a later test that watches torch.cuda.memory_allocated() would see it go whenever the collector runs."""
    yield
    ops = sys.modules.get("lbtree.ops")
    if ops is not None:
        ops.release_workspace()
    gc.collect()
