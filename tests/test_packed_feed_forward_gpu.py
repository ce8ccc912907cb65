"""The GPU tests of packed_feed_forward.py, in a process of their own (PyTorch
has to be imported before the library, see test_packed_gpu.py). Directly:

    python -m pytest tests/packed_feed_forward.py -x -v
"""
import pytest

import test_packed_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("file", ["packed_feed_forward.py"])
def test_in_a_process_of_its_own(gpu, capfd, file):
    test_packed_gpu.test_in_a_process_of_its_own(gpu, capfd, file)
