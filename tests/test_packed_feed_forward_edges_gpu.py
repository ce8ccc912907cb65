"""The GPU tests of packed_feed_forward_edges.py, in a process of their own (PyTorch
has to be imported before the library, see test_packed_gpu.py). Directly:

    python -m pytest tests/packed_feed_forward_edges.py -x -v
"""
import pytest

import test_packed_gpu

pytestmark = pytest.mark.gpu


def test_in_a_process_of_its_own(gpu, capfd):
    test_packed_gpu.test_in_a_process_of_its_own(gpu, capfd, "packed_feed_forward_edges.py")
