"""Arrays in LDS that kernels access 16 bytes at a time say so in their declaration:
an array of floats is aligned to four bytes by itself, and that the compiler places
it better is not its promise."""
import glob
import os
import re

import pytest

from test_dma_wait_order import KERNELS

WIDE = r"\((?:const )?(?:typename )?(?:Num<T>::)?(?:float4_t|half8_t|uint4_t|v8)\s*\*\)[\s&(]*"


def unaligned(source):
    """Names of the arrays that are accessed in 16 bytes but not declared so."""
    bad = []
    for declared in re.findall(r"__shared__ ([^;]*);", source):
        if "aligned(16)" in declared:
            continue
        names = re.findall(r"(\w+)(?=\[)", re.sub(r"\[[^\]]*\]", "[]", declared))
        bad += [name for name in names if re.search(WIDE + name + r"\b", source)]
    return bad


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(KERNELS, "*.hip")) + glob.glob(os.path.join(KERNELS, "*.hpp"))),
                         ids=os.path.basename)
def test_wide_accesses_are_declared(path):
    with open(path) as f:
        assert not unaligned(f.read())


def test_the_check_finds_them():
    use = "*(float4_t*)&sum[w][4 * l] = v; x = *(const v8*)(codes + 8);"
    assert unaligned("__shared__ float sum[N][20], other[3];" + use) == ["sum"]
    assert unaligned("__shared__ char codes[N > 1 ? N : 8];" + use) == ["codes"]
    assert unaligned("__shared__ int codes_of[4], x[9];" + use) == []
    assert unaligned("__shared__ __attribute__((aligned(16))) float sum[N][20];" + use) == []
