import os
import sys

# (before anything initialises the GPU: see mdmm/__init__.py)
os.environ.setdefault('DEBUG_CLR_GRAPH_PACKET_CAPTURE', '0')

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import helpers  # noqa: E402,F401  (puts the repo root and the package dir on sys.path)


def pytest_configure(config):
    config.addinivalue_line('markers', 'gpu: needs a real MI355X (run with -m gpu on the GPU box)')


def pytest_collection_modifyitems(config, items):
    import torch
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason='no GPU in this container')
    for item in items:
        if 'gpu' in item.keywords:
            item.add_marker(skip)


@pytest.fixture(autouse=True)
def _oracle_bias_sums(request):
    """The replay tests skip parameters whose gradient is exactly zero (a convolution's bias in front of a BatchNorm) by the
    size of the oracle's rounding noise there, below 1e-4 of the largest gradient.  The CPU library's bias sum runs through
    each thread's share element by element: its noise is 1.6e-3 of the largest gradient with 16 threads and 1.9e-2 with one
    (240 frames; a left-out modality's constant batch multiplies it by 1 / sqrt(eps) = 316 a norm), ATen's own cascaded sum
    3.9e-5 with any number of threads.  So these tests' oracle runs on ATen's convolutions."""
    if request.node.path.name != 'test_replay_gpu.py':
        yield
        return
    import torch
    with torch.backends.mkldnn.flags(enabled=False):
        yield
