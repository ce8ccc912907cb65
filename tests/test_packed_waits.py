"""Static check of the kernels on packed batches for register loads beside DMA
loads, on the gfx950 assembly this build produces (CPU only: hipcc
cross-compiles).

Their blocks come into LDS by DMA (`global_load_lds_dwordx4`), with waits that
let the N newest loads stay in flight (`s_waitcnt vmcnt(N)`). DMA loads land in
order among themselves, so where N is no more than the number of DMA loads
issued behind the awaited one, it has landed, whatever else is in flight. But
nothing orders a register load against a DMA load (test_dma_wait_order.py), while
the compiler takes a register load for returned once a counted wait behind it
would say so if all loads returned in order. So a register load that is used
behind a DMA load which was issued after it needs a full wait (vmcnt(0)) in
between. Every register load of every kernel is followed to its uses along every
path of the emitted code."""
import os
import re
import subprocess

import pytest

from test_dma_wait_order import FLAGS, HIPCC, KERNELS, VMEM


def is_dma(ins):
    return ins.startswith("global_load_lds")


def registers(operand):
    m = re.fullmatch(r"v\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.fullmatch(r"v(\d+)", operand)
    return {int(m.group(1))} if m else set()


def kernels_of(src, out, include):
    """Per kernel its instructions and the index that each label stands for."""
    subprocess.check_call([HIPCC, *FLAGS, "-I", include, src, "-o", out], stderr=subprocess.DEVNULL)
    kernels, cur = {}, None
    for line in open(out):
        m = re.match(r"^(_Z\S+):", line)
        if m and "kernel" in m.group(1):
            cur = kernels[m.group(1)] = ([], {})
            continue
        if line.startswith(".Lfunc_end"):
            cur = None
        if cur is None:
            continue
        m = re.match(r"^(\.LBB\w+):", line)
        if m:
            cur[1][m.group(1)] = len(cur[0])
        s = line.split(";")[0].strip()
        if s and not s.startswith((";", ".")):
            cur[0].append(s)
    return kernels


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
        accumulates = op.startswith(("v_fmac", "v_permlane32_swap", "v_dot2c"))
        self.writes = args[0] if vector and args and not stores else set()
        self.reads = set().union(*(args if stores or accumulates else args[1:])) if vector and args else set()
        target = [labels[text.split()[1]]] if op.startswith(("s_branch", "s_cbranch")) else []
        self.next = target if op == "s_branch" else [] if op == "s_endpgm" else [at + 1] + target


def violations(kernel):
    """Register loads whose value is used behind a later DMA load without a full
    wait, each with such a use."""
    code = [Instruction(text, i, kernel[1]) for i, text in enumerate(kernel[0])]
    bad = []
    for i, load in enumerate(code):
        if not load.load:
            continue
        seen, stack = set(), [(i + 1, False)]
        while stack:
            at, dma = stack.pop()
            if at >= len(code) or (at, dma) in seen:
                continue
            seen.add((at, dma))
            ins = code[at]
            if ins.full:
                continue
            if ins.reads & load.writes:
                if dma:
                    bad.append((load.text, ins.text))
                    break
                continue  # used, and so waited for, in front of any DMA load
            if ins.writes & load.writes:
                continue
            stack += [(n, dma or ins.dma) for n in ins.next]
    return bad


@pytest.fixture(scope="module")
def hipcc():
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not found")


@pytest.mark.parametrize("src,kernels", [("packed_attention.hip", ("packed_attention_kernel", "packed_attention_few_kernel")),
                                         ("packed_linear.hip", ("packed_shrink_kernel", "packed_linear_few_kernel",
                                                                "packed_linear_kernel"))])
def test_register_loads_beside_dma_loads(hipcc, tmp_path, src, kernels):
    found = {}
    for name, kernel in kernels_of(os.path.join(KERNELS, src), str(tmp_path / "k.s"), KERNELS).items():
        bad = violations(kernel)
        assert not bad, f"{name}: {bad[:3]}"
        assert not any(re.match(r"v_pk_(add|mul|fma)_f32", i) for i in kernel[0]), name
        found[name] = sum(is_dma(i) for i in kernel[0])
    for kernel in kernels:
        assert any(kernel in k and n > 0 for k, n in found.items()), (kernel, found)


LOAD, DMA, USE = "global_load_dword v1, v[2:3], off", "global_load_lds_dwordx4 v[4:5], off", "v_add_u32_e32 v6, v1, v6"


@pytest.mark.parametrize("code,labels,caught", [
    ([LOAD, DMA, "s_waitcnt vmcnt(1)", USE], {}, True),
    ([LOAD, DMA, "s_waitcnt vmcnt(0)", USE], {}, False),
    ([LOAD, "s_waitcnt vmcnt(0)", DMA, "s_waitcnt vmcnt(1)", USE], {}, False),
    ([LOAD, "s_waitcnt vmcnt(0)", USE, DMA], {}, False),
    ([DMA, LOAD, "s_waitcnt vmcnt(0)", USE], {}, False),
    # a full wait on one of two paths, and the use in the next turn of a loop
    ([LOAD, DMA, "s_cbranch_scc0 .LBB0_1", "s_waitcnt vmcnt(0)", USE], {".LBB0_1": 4}, True),
    ([LOAD, "s_waitcnt vmcnt(0)", USE, LOAD, DMA, "s_waitcnt vmcnt(1)", "s_cbranch_scc0 .LBB0_1"], {".LBB0_1": 2}, True),
    ([LOAD, DMA, "global_load_dwordx4 v[0:3], v[2:3], off", "s_waitcnt vmcnt(0)", USE], {}, False),
    ([LOAD, DMA, "ds_write_b32 v7, v1"], {}, True),
    ([LOAD, DMA, "global_store_dword v[8:9], v1, off"], {}, True),
])
def test_the_check_catches_a_missing_wait(code, labels, caught):
    assert bool(violations((code + ["s_endpgm"], labels))) == caught
