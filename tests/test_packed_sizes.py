"""Sizes that the operators on packed batches take (CPU only: every argument is
checked before the engine is looked at, so a null engine shows that the checks
passed)."""
import importlib.util
import os
import random

import pytest

import dinov3_hrx as d
from dinov3_hrx import packed

from test_packed import ATTENTION, message

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# --- rotation ----------------------------------------------------------------

@pytest.mark.parametrize("neighbours", [0, 1])
@pytest.mark.parametrize("dim,rotated", [(64, 64), (64, 32), (128, 48), (80, 80), (80, 40), (80, 16), (16, 8), (8, 8), (24, 24), (40, 40),
                                         (112, 56)])
def test_rotation_takes(neighbours, dim, rotated):
    assert message("rotation", neighbours=neighbours, head_dim=dim, rotated=rotated, x_stride=4 * dim, out_stride=4 * dim) == "null engine"


@pytest.mark.parametrize("dim,rotated", [(80, 24), (80, 8), (80, 72), (24, 12), (40, 20), (64, 40), (16, 0), (8, 4)])
def test_rotation_refuses(dim, rotated):
    assert "rotated must be" in message("rotation", head_dim=dim, rotated=rotated, x_stride=4 * dim, out_stride=4 * dim)


def test_the_timed_ranges_are_taken():
    # Every call that the range of the timed cases can make, with addresses that
    # nothing reads.
    pytest.importorskip("torch")
    spec = importlib.util.spec_from_file_location("timed_operators", os.path.join(ROOT, "perf", "operators.py"))
    timed = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(timed)
    rng = random.Random(17)
    seen = {}
    for case in timed.listed() + [timed.draw(rng) for _ in range(3000)]:
        if case["op"] == "attention":
            q, k = timed._lengths(case["queries"]), timed._lengths(case["keys"])
            name, dim = "attention", case["head_dim"]
            change = dict(causal=case["causal"], sequences=len(q), heads=case["heads"], kv_heads=case["kv_heads"], head_dim=dim,
                          q_rows=sum(q), k_rows=sum(k), longest_q=max(q), longest_k=max(k), q_stride=case["heads"] * dim,
                          out_stride=case["heads"] * dim, k_stride=case["kv_heads"] * dim, v_stride=case["kv_heads"] * dim,
                          workspace_bytes=1 << 40)
        elif case["op"] == "linear":
            lengths = timed._lengths(case["lengths"])
            name = "linear"
            change = dict(sequences=len(lengths), rows=sum(lengths), inputs=case["inputs"], outputs=case["outputs"], rank=case["rank"],
                          adapters=case["adapters"], x_stride=case["inputs"], w_stride=case["inputs"], y_stride=case["outputs"],
                          workspace_bytes=1 << 40)
        else:
            lengths = timed._lengths(case["lengths"])
            name, dim = "rotation", case["head_dim"]
            change = dict(neighbours=case["neighbours"], rows=sum(lengths), heads=case["heads"], head_dim=dim, rotated=case["rotated"],
                          places=max(lengths), x_stride=case["row"], out_stride=case["heads"] * dim)
        assert message(name, **change) == "null engine", case
        seen[name, case.get("rotated") == 40] = seen.get((name, case.get("rotated") == 40), 0) + 1
    assert all(seen.get(k, 0) > 20 for k in (("attention", False), ("linear", False), ("rotation", False), ("rotation", True))), seen


# --- no queries --------------------------------------------------------------

@pytest.mark.parametrize("k_rows", [0, 1, 512, 513, 1 << 20])
@pytest.mark.parametrize("longest_k", [0, 1, 513, 1 << 20])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (32, 8, 128), (1, 1, 8)])
def test_attention_without_queries_needs_nothing(k_rows, longest_k, heads, kv, dim):
    sizes = dict(q_rows=0, k_rows=k_rows, longest_k=longest_k, heads=heads, kv_heads=kv, head_dim=dim, q=0, out=0, q_stride=heads * dim,
                 out_stride=heads * dim, k_stride=kv * dim, v_stride=kv * dim, workspace=0, workspace_bytes=0)
    assert d.packed_workspace("attention", packed.Attention(**{**ATTENTION, **sizes})) == 0
    assert message("attention", **sizes) == "null engine"
