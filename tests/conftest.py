import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200)")


def pytest_collection_modifyitems(config, items):
    try:
        import torch
        has_gpu = torch.cuda.is_available()
    except Exception:
        has_gpu = False
    if has_gpu:
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(autouse=True)
def waits_of_shared_prefixes(request):
    """Kernels whose bounded waits ran out leave rows unwritten and say so in a word on the device: no test passes by them."""
    yield
    if request.node.path.name.startswith("test_shared_prefix") and "gpu" in request.keywords:
        from ginfer_b200.ops import gemm_bf16
        gemm_bf16.check_errors()
