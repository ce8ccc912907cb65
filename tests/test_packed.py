"""Refusals of the operators on packed batches (CPU only: every argument is
checked before the engine is looked at, so a null engine shows which check
answers), and the workspace functions."""
import ctypes

import pytest

import dinov3_hrx as d
from dinov3_hrx import packed

A = 1 << 20  # an aligned address; nothing here reads it

LINEAR = dict(type=packed.F16, sequences=3, rows=100, inputs=64, outputs=128, rank=16, adapters=2, x=A, w=A, bias=A, a=A, b=A,
              scale=A, y=A, x_stride=64, w_stride=64, y_stride=128, starts=A, adapter=A, workspace=A, workspace_bytes=1 << 20)
ROTATION = dict(type=packed.BF16, rows=10, heads=4, head_dim=64, rotated=64, places=10, x=A, out=2 * A, x_stride=256,
                out_stride=256, cos=A, sin=A, index=A)
ATTENTION = dict(type=packed.F16, causal=1, sequences=3, heads=8, kv_heads=2, head_dim=64, q_rows=100, k_rows=100, scale=0.125,
                 q=A, k=A, v=A, out=A, q_stride=512, k_stride=128, v_stride=128, out_stride=512, q_starts=A, k_starts=A,
                 workspace=A, workspace_bytes=1 << 30)
CALLS = {"linear": (packed.Linear, LINEAR), "rotation": (packed.Rotation, ROTATION),
         "attention": (packed.Attention, ATTENTION)}


def message(name, **change):
    kind, fields = CALLS[name]
    call = kind(**{**fields, **change})
    run = getattr(d._lib, f"dhx_packed_{name}_run")
    assert run(None, ctypes.byref(call), None) == 1
    return d._lib.dhx_last_error(None).decode()


@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_reach_the_engine(name):
    assert message(name) == "null engine"
    assert getattr(d._lib, f"dhx_packed_{name}_run")(None, None, None) == 1
    assert d._lib.dhx_last_error(None).decode() == "null argument"


REFUSED = [
    ("linear", dict(type=2), "type must be DHX_F16 or DHX_BF16"),
    ("linear", dict(sequences=0), "sequences must be positive"),
    ("linear", dict(inputs=60), "inputs must be a positive multiple of 8"),
    ("linear", dict(inputs=0), "inputs must be a positive multiple of 8"),
    ("linear", dict(outputs=4), "outputs must be a positive multiple of 8"),
    ("linear", dict(rank=0), "rank must be a positive multiple of 8"),
    ("linear", dict(rank=264), "rank must be at most 256"),
    ("linear", dict(adapters=0), "adapters must be positive"),
    ("linear", dict(rows=1 << 31), "rows must be at most"),
    ("linear", dict(rows=(1 << 27) + 1), "rows must be at most"),
    ("linear", dict(rows=1 << 27, outputs=1 << 20), "the number of tiles of 256 x 256 outputs must be at most"),
    ("linear", dict(x=0), "x is a null device pointer"),
    ("linear", dict(w=A + 8), "w must be 16-byte aligned"),
    ("linear", dict(bias=A + 4), "bias must be 16-byte aligned"),
    ("linear", dict(scale=0), "scale is a null device pointer"),
    ("linear", dict(starts=0), "starts is a null device pointer"),
    ("linear", dict(adapter=A + 2), "adapter must be 4-byte aligned"),
    ("linear", dict(x_stride=56), "x_stride must be at least 64"),
    ("linear", dict(w_stride=68), "w_stride must be a multiple of 8"),
    ("linear", dict(y_stride=1 << 23), "y_stride must be at most"),
    ("linear", dict(workspace_bytes=100), "the workspace has 100 bytes"),
    ("linear", dict(workspace=0), "workspace is a null device pointer"),
    ("linear", dict(workspace=A + 8), "workspace must be 16-byte aligned"),
    ("rotation", dict(type=7), "type must be DHX_F16 or DHX_BF16"),
    ("rotation", dict(neighbours=2), "neighbours must be 0 or 1"),
    ("rotation", dict(heads=0), "heads must be positive"),
    ("rotation", dict(head_dim=60), "head_dim must be a positive multiple of 8"),
    ("rotation", dict(rotated=24), "rotated must be a positive multiple of 16"),
    ("rotation", dict(rotated=80), "rotated must be at most head_dim"),
    ("rotation", dict(places=0), "places must be positive"),
    ("rotation", dict(x=A + 2), "x must be 16-byte aligned"),
    ("rotation", dict(cos=0), "cos is a null device pointer"),
    ("rotation", dict(index=0), "index is a null device pointer"),
    ("rotation", dict(x_stride=248), "x_stride must be at least 256"),
    ("rotation", dict(out=A, out_stride=264), "in place, out_stride must be x_stride"),
    ("attention", dict(type=3), "type must be DHX_F16 or DHX_BF16"),
    ("attention", dict(causal=2), "causal must be 0 or 1"),
    ("attention", dict(reserved=1), "reserved must be 0"),
    ("attention", dict(sequences=0), "sequences must be positive"),
    ("attention", dict(kv_heads=0), "kv_heads must be positive"),
    ("attention", dict(heads=7), "heads must be a multiple of kv_heads"),
    ("attention", dict(head_dim=136), "head_dim must be at most 128"),
    ("attention", dict(head_dim=68), "head_dim must be a positive multiple of 8"),
    ("attention", dict(scale=0.0), "scale must be positive and finite"),
    ("attention", dict(scale=-1.0), "scale must be positive and finite"),
    ("attention", dict(scale=float("nan")), "scale must be positive and finite"),
    ("attention", dict(scale=float("inf")), "scale must be positive and finite"),
    ("attention", dict(k=0), "k is a null device pointer"),
    ("attention", dict(out=A + 8), "out must be 16-byte aligned"),
    ("attention", dict(k_starts=0), "k_starts is a null device pointer"),
    ("attention", dict(q_stride=500), "q_stride must be a multiple of 8"),
    ("attention", dict(v_stride=56), "v_stride must be at least 64"),
    ("attention", dict(q_head_stride=60), "head strides must be multiples of 8"),
    ("attention", dict(k_head_stride=56), "head strides must be at least head_dim"),
    ("attention", dict(out_stride=504), "out_stride and out_head_stride make heads overlap"),
    ("attention", dict(q_rows=1 << 30), "q_rows * (heads / kv_heads) must be at most"),
    ("attention", dict(scale=2.0 ** 21), "scale must be at most 2^20"),
    ("attention", dict(k_rows=(1 << 31) - 300), "q_rows + k_rows must be at most"),
    ("attention", dict(sequences=1 << 24), "the number of row tiles must be at most"),
]


@pytest.mark.parametrize("name,change,text", REFUSED)
def test_refused(name, change, text):
    assert text in message(name, **change)


def test_no_rows_need_no_memory():
    assert message("linear", rows=0, x=0, y=0) == "null engine"
    assert message("rotation", rows=0, x=0, out=0, index=0) == "null engine"
    assert message("attention", k_rows=0, k=0, v=0) == "null engine"
    assert message("attention", q_rows=0, q=0, out=0) == "null engine"


def test_heads_in_matrices_of_their_own():
    # [heads][rows][head_dim]: the distance between rows is head_dim.
    assert message("attention", out_stride=64, out_head_stride=100 * 64, q_stride=64, q_head_stride=100 * 64) == "null engine"
    assert "overlap" in message("attention", out_stride=64, out_head_stride=99 * 64)


def test_workspaces():
    kind, fields = CALLS["linear"]
    need = d.packed_workspace("linear", kind(**fields))
    assert need >= 100 * 4 + 100 * 16 * 2
    assert message("linear", workspace_bytes=need) == "null engine"
    assert "the call needs" in message("linear", workspace_bytes=need - 1)
    # The sizes alone are needed, and they are checked.
    assert d.packed_workspace("linear", kind(**{**fields, "x": 0, "workspace": 0, "workspace_bytes": 0})) == need
    with pytest.raises(d.DINOv3Error, match="rank must be"):
        d.packed_workspace("linear", kind(**{**fields, "rank": 12}))
    kind, fields = CALLS["attention"]
    for rows, sequences, longest in ((100, 3, 100), (1, 1, 8192), (64, 64, 1 << 20), (1 << 20, 1, 1 << 20)):
        sizes = {**fields, "q_rows": rows, "sequences": sequences, "longest_k": longest, "k_rows": longest * sequences}
        need = d.packed_workspace("attention", kind(**sizes))
        if need:
            assert "the call needs" in message("attention", **{**sizes, "workspace_bytes": need - 1})
            assert message("attention", **{**sizes, "workspace_bytes": need}) == "null engine"
        else:
            assert message("attention", **{**sizes, "workspace": 0, "workspace_bytes": 0}) == "null engine"
    with pytest.raises(d.DINOv3Error, match="heads must be"):
        d.packed_workspace("attention", kind(**{**fields, "heads": 3}))
