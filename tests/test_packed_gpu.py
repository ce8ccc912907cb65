"""The GPU tests of the operators on packed batches, packed_operators.py and
packed_chain.py, each in a process of its own: they hold device memory and
compute the float64 references with PyTorch, which brings a HIP runtime of its
own and has to be imported before the library (the two then share that one; the
other way round PyTorch finds no device), while the tests of this process run the
library on the system's runtime. Directly:

    python -m pytest tests/packed_operators.py tests/packed_chain.py -x -v
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("file", ["packed_operators.py", "packed_chain.py"])
def test_in_a_process_of_its_own(gpu, capfd, file):
    with capfd.disabled():  # its progress and failures are seen as they come
        print(f"\n{file}:", flush=True)
        code = subprocess.run([sys.executable, "-u", "-m", "pytest", os.path.join(HERE, file), "-x", "-q", "-p", "no:cacheprovider"],
                              cwd=os.path.dirname(HERE), timeout=600).returncode
    assert code == 0, f"{file} failed: its output is above"
