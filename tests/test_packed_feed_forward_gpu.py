"""The GPU tests of packed_feed_forward.py and packed_block.py, each in a process
of its own (PyTorch has to be imported before the library, see test_packed_gpu.py).
Directly:

    python -m pytest tests/packed_feed_forward.py tests/packed_block.py -x -v
"""
import pytest

import test_packed_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("file", ["packed_feed_forward.py", "packed_block.py"])
def test_in_a_process_of_its_own(gpu, capfd, file):
    test_packed_gpu.test_in_a_process_of_its_own(gpu, capfd, file)
