"""The static check of test_packed_waits_live.py (register loads beside DMA loads)
on the kernels of the feed-forward half of a packed block, whose DMA loads come from
buffers as well (`buffer_load_dwordx4 ... lds`); and no packed float32 arithmetic,
which the build turns off."""
import os
import re

import pytest

import test_packed_waits
import test_packed_waits_live
from test_dma_wait_order import KERNELS
from test_packed_waits import LOAD, USE, hipcc, kernels_of  # noqa: F401


def is_dma(ins):
    return ins.startswith("global_load_lds") or (ins.startswith("buffer_load") and " lds" in ins)


@pytest.fixture(autouse=True)
def loads_from_buffers_too(monkeypatch):
    monkeypatch.setattr(test_packed_waits, "is_dma", is_dma)
    monkeypatch.setattr(test_packed_waits_live, "is_dma", is_dma)


@pytest.mark.parametrize("src,kernels,with_dma", [
    ("packed_gated.hip", ("packed_product_kernel", "packed_product_few_kernel", "packed_gated_few_kernel"), ("packed_product_kernel",)),
    ("packed_quantised.hip", ("packed_product_kernel", "packed_product_few_kernel"), ("packed_product_kernel",)),
    ("packed_norm.hip", ("packed_norm_kernel",), ()),
    ("packed_quantise.hip", ("packed_quantise_kernel", "packed_dequantise_kernel"), ()),
])
def test_register_loads_beside_dma_loads(hipcc, tmp_path, src, kernels, with_dma):  # noqa: F811
    found = {}
    for name, kernel in kernels_of(os.path.join(KERNELS, src), str(tmp_path / "k.s"), KERNELS).items():
        bad = test_packed_waits_live.violations(kernel)
        assert not bad, f"{name}: {bad[:3]}"
        assert not any(re.match(r"v_pk_(add|mul|fma)_f32", i) for i in kernel[0]), name
        found[name] = sum(is_dma(i) for i in kernel[0])
    for kernel in kernels:
        assert any(kernel in k and (n > 0) == (kernel in with_dma) for k, n in found.items()), (kernel, found)


BUFFER = "buffer_load_dwordx4 v4, s[4:7], s3 offen lds"


@pytest.mark.parametrize("code,caught", [
    ([LOAD, BUFFER, "s_waitcnt vmcnt(1)", USE], True),
    ([LOAD, BUFFER, "s_waitcnt vmcnt(0)", USE], False),
    ([BUFFER, LOAD, "s_waitcnt vmcnt(0)", USE], False),
    (["buffer_load_dword v1, v2, s[4:7], 0 offen", BUFFER, "s_waitcnt vmcnt(1)", USE], True),
])
def test_the_check_knows_loads_from_buffers(code, caught):
    assert bool(test_packed_waits_live.violations((code + ["s_endpgm"], {}))) == caught
