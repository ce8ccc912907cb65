"""The static check of test_packed_waits.py (register loads beside DMA loads in
the kernels on packed batches), with every register of a load followed for
itself: a load stays on its way for those of its registers that nothing has
written since, and operands with modifiers (-v1, |v1|, abs(v1)) and accumulator
registers count as well."""
import os
import re

import pytest

from test_dma_wait_order import KERNELS, VMEM
from test_packed_waits import DMA, LOAD, USE, hipcc, is_dma, kernels_of  # noqa: F401


def registers(operand):
    """The vector registers of an operand, those of the accumulator file as ("a", n)."""
    operand = re.sub(r"^(neg|abs|sext)\((.*)\)$", r"\2", operand.strip().lstrip("-").strip("|").lstrip("-"))
    m = re.fullmatch(r"([va])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m.group(1), n) for n in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.fullmatch(r"([va])(\d+)", operand)
    return {(m.group(1), int(m.group(2)))} if m else set()


class Instruction:
    def __init__(self, text, at, labels):
        self.text, op = text, text.split()[0]
        parts = text.split(None, 1)
        args = [registers(o.strip().split()[0]) for o in parts[1].split(",") if o.strip()] if len(parts) > 1 else []
        vector = not op.startswith("s_")
        self.dma = is_dma(text)
        self.load = bool(VMEM.match(text)) and "load" in op and not self.dma
        self.full = bool(re.match(r"s_waitcnt.*vmcnt\(0\)", text))
        stores = self.dma or op.startswith(("global_store", "buffer_store", "ds_write", "scratch_store", "v_cmp"))
        # Reads what it writes, or leaves a part of it.
        accumulates = op.startswith(("v_fmac", "v_mac", "v_permlane32_swap", "v_swap", "v_dot2c", "v_writelane")) or "d16" in op \
            or "sdwa" in op or "dst_sel" in text
        self.writes = args[0] if vector and args and not stores and not accumulates else set()
        self.reads = set().union(*(args if stores or accumulates else args[1:])) if vector and args else set()
        self.loaded = args[0] if self.load and args else set()
        target = [labels[text.split()[1]]] if op.startswith(("s_branch", "s_cbranch")) else []
        self.next = target if op == "s_branch" else [] if op == "s_endpgm" else [at + 1] + target


def violations(kernel):
    """Register loads of which a register is used behind a later DMA load without
    a full wait, each with such a use."""
    code = [Instruction(text, i, kernel[1]) for i, text in enumerate(kernel[0])]
    bad = []
    for i, load in enumerate(code):
        if not load.load or not load.loaded:
            continue
        seen, stack = set(), [(i + 1, False, frozenset(load.loaded))]
        while stack:
            at, dma, live = stack.pop()
            if at >= len(code) or (at, dma, live) in seen:
                continue
            seen.add((at, dma, live))
            ins = code[at]
            if ins.full:
                continue
            if ins.reads & live:
                if dma:
                    bad.append((load.text, ins.text))
                    break
                continue  # used, and so waited for, in front of any DMA load
            live -= ins.writes | ins.loaded
            if live:
                stack += [(n, dma or ins.dma, live) for n in ins.next]
    return bad


@pytest.mark.parametrize("src,kernels", [("packed_attention.hip", ("packed_attention_kernel", "packed_attention_few_kernel")),
                                         ("packed_linear.hip", ("packed_shrink_kernel", "packed_linear_few_kernel",
                                                                "packed_linear_kernel"))])
def test_register_loads_beside_dma_loads(hipcc, tmp_path, src, kernels):  # noqa: F811
    found = {}
    for name, kernel in kernels_of(os.path.join(KERNELS, src), str(tmp_path / "k.s"), KERNELS).items():
        bad = violations(kernel)
        assert not bad, f"{name}: {bad[:3]}"
        found[name] = sum(is_dma(i) for i in kernel[0])
    for kernel in kernels:
        assert any(kernel in k and n > 0 for k, n in found.items()), (kernel, found)


WIDE = "global_load_dwordx4 v[10:13], v[2:3], off"


@pytest.mark.parametrize("code,labels,caught", [
    ([LOAD, DMA, "s_waitcnt vmcnt(1)", USE], {}, True),
    ([LOAD, DMA, "s_waitcnt vmcnt(0)", USE], {}, False),
    ([LOAD, "s_waitcnt vmcnt(0)", USE, DMA], {}, False),
    # operands with modifiers
    ([LOAD, DMA, "s_waitcnt vmcnt(1)", "v_fma_f32 v6, v7, v8, -v1"], {}, True),
    ([LOAD, DMA, "s_waitcnt vmcnt(1)", "v_fma_f32 v6, v7, |v1|, v8"], {}, True),
    ([LOAD, DMA, "s_waitcnt vmcnt(1)", "v_max_f32_e64 v6, -|v1|, v8"], {}, True),
    ([LOAD, DMA, "s_waitcnt vmcnt(1)", "v_fma_f32 v6, v7, v8, -v5"], {}, False),
    # one register of a wide load written anew, another used
    ([WIDE, DMA, "s_waitcnt vmcnt(1)", "v_mov_b32_e32 v10, 0", "v_add_u32_e32 v6, v11, v6"], {}, True),
    ([WIDE, DMA, "s_waitcnt vmcnt(1)", "v_mov_b32_e32 v10, 0", "v_add_u32_e32 v6, v10, v6"], {}, False),
    ([WIDE, DMA, "s_waitcnt vmcnt(1)", "v_mov_b32_e32 v10, 0", "s_waitcnt vmcnt(0)", "v_add_u32_e32 v6, v11, v6"], {}, False),
    # one written on one of two paths only
    ([LOAD, DMA, "s_cbranch_scc0 .LBB0_1", "v_mov_b32_e32 v1, 0", USE], {".LBB0_1": 4}, True),
    # accumulator registers
    (["global_load_dwordx4 a[0:3], v[2:3], off", DMA, "s_waitcnt vmcnt(1)", "v_accvgpr_read_b32 v6, a2"], {}, True),
])
def test_the_check_catches_a_missing_wait(code, labels, caught):
    assert bool(violations((code + ["s_endpgm"], labels))) == caught
