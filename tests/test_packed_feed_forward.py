"""Refusals of the operators of the feed-forward half of a packed block (CPU only:
every argument is checked before the engine is looked at, so a null engine shows
which check answers), their workspaces, and that the whole range of the timed
cases is taken."""
import ctypes
import importlib.util
import os
import random

import pytest

import dinov3_hrx as d
from dinov3_hrx import packed

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20  # an aligned address; nothing here reads it

NORM = dict(type=packed.F16, stream_type=packed.F16, post=packed.RMS, pre=packed.LAYER, rows=100, channels=384, sequences=3, post_eps=1e-5,
            pre_eps=0.0, x=A, y=2 * A, x_out=3 * A, h=4 * A, post_weight=A, pre_weight=A, pre_bias=A, scale=A, gate=A, x_stride=384,
            y_stride=384, x_out_stride=384, h_stride=384, gate_stride=384, starts=A)
QUANTISATION = dict(type=packed.BF16, rows=10, columns=1000, x=A, codes=A, scales=A, x_stride=1000, codes_stride=512, scales_stride=32)
QUANTISED_LINEAR = dict(type=packed.BF16, sequences=3, rows=1000, inputs=1000, outputs=1280, x=A, w=A, w_scales=A, bias=A, y=A, x_stride=1000,
                        y_stride=1280, w_stride=512, scales_stride=32, starts=A, workspace=A, workspace_bytes=1 << 30)
GATED = dict(type=packed.F16, activation=packed.SILU, rows=1000, inputs=64, outputs=1280, x=A, gate=A, up=A, out=A, x_stride=64,
             out_stride=1280, w_stride=64)
GATED_FOUR = dict(GATED, gate_scales=A, up_scales=A, w_stride=32, scales_stride=16, workspace=A, workspace_bytes=1 << 20)
CALLS = {"norm": ("norm", packed.Norm, NORM), "quantise": ("quantise", packed.Quantisation, QUANTISATION),
         "dequantise": ("dequantise", packed.Quantisation, QUANTISATION),
         "quantised_linear": ("quantised_linear", packed.QuantisedLinear, QUANTISED_LINEAR),
         "gated": ("gated", packed.Gated, GATED), "gated_four": ("gated", packed.Gated, GATED_FOUR)}


def message(name, **change):
    function, kind, fields = CALLS[name]
    call = kind(**{**fields, **change})
    assert getattr(d._lib, f"dhx_packed_{function}_run")(None, ctypes.byref(call), None) == 1
    return d._lib.dhx_last_error(None).decode()


@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_reach_the_engine(name):
    assert message(name) == "null engine"
    assert getattr(d._lib, f"dhx_packed_{CALLS[name][0]}_run")(None, None, None) == 1
    assert d._lib.dhx_last_error(None).decode() == "null argument"


PLAIN = dict(y=0, x_out=0, post=0, post_weight=0, scale=0, gate=0)  # a norm without y
REFUSED = [
    ("norm", dict(type=2), "type must be DHX_F16 or DHX_BF16"),
    ("norm", dict(stream_type=packed.BF16), "stream_type must be type or DHX_F32"),
    ("norm", dict(stream_type=3), "stream_type must be type or DHX_F32"),
    ("norm", dict(post=3), "post and pre must be"),
    ("norm", dict(pre=7), "post and pre must be"),
    ("norm", dict(rows=(1 << 31) - 256), "rows must be at most"),
    ("norm", dict(channels=0), "channels must be a positive multiple of 8"),
    ("norm", dict(channels=60), "channels must be a positive multiple of 8"),
    ("norm", dict(channels=32776), "channels must be at most 32768"),
    ("norm", dict(post_eps=-1e-6), "post_eps and pre_eps must be finite and not negative"),
    ("norm", dict(pre_eps=float("nan")), "post_eps and pre_eps must be finite and not negative"),
    ("norm", dict(pre_eps=float("inf")), "post_eps and pre_eps must be finite and not negative"),
    ("norm", dict(x=0), "x is a null device pointer"),
    ("norm", dict(y=2 * A + 8), "y must be 16-byte aligned"),
    ("norm", dict(x_out=0), "x_out is a null device pointer"),
    ("norm", dict(h=0), "h is a null device pointer"),
    ("norm", dict(pre=0, pre_weight=0, pre_bias=0), "h needs a norm in pre"),
    ("norm", dict(pre=0, h=0), "pre_weight and pre_bias need a norm in pre"),
    ("norm", dict(post=0), "post_weight and post_bias need a norm in post"),
    ("norm", dict(x_stride=376), "x_stride must be at least 384"),
    ("norm", dict(y_stride=388), "y_stride must be a multiple of 8"),
    ("norm", dict(x_out_stride=1 << 23), "x_out_stride must be at most"),
    ("norm", dict(h_stride=0), "h_stride must be at least 384"),
    ("norm", dict(x_out=A, x_out_stride=392), "in place, x_out_stride must be x_stride"),
    ("norm", dict(h=2 * A, h_stride=392), "in place, h_stride must be y_stride"),
    ("norm", dict(h=3 * A), "h and x_out must not be the same"),
    ("norm", dict(scale=A + 4), "scale must be 16-byte aligned"),
    ("norm", dict(gate=A + 8), "gate must be 16-byte aligned"),
    ("norm", dict(gate_stride=100), "gate_stride must be a multiple of 8"),
    ("norm", dict(starts=0, sequences=0), "gate needs starts"),
    ("norm", dict(starts=0), "starts is a null device pointer"),
    ("norm", dict(sequences=0), "sequences must be positive"),
    ("norm", dict(starts=A + 2), "starts must be 4-byte aligned"),
    ("norm", dict(PLAIN, x_out=A), "without y there are no post, scale, gate and x_out, and pre is needed"),
    ("norm", dict(PLAIN, post=1), "without y there are no post"),
    ("norm", dict(PLAIN, scale=A), "without y there are no post"),
    ("norm", dict(PLAIN, gate=A), "without y there are no post"),
    ("norm", dict(PLAIN, pre=0, h=0, pre_weight=0, pre_bias=0), "without y there are no post"),
    ("quantise", dict(type=2), "type must be DHX_F16 or DHX_BF16"),
    ("quantise", dict(reserved=1), "reserved must be 0"),
    ("quantise", dict(columns=1004), "columns must be a positive multiple of 8"),
    ("quantise", dict(columns=0), "columns must be a positive multiple of 8"),
    ("quantise", dict(columns=(1 << 22) + 8, x_stride=1 << 22), "columns must be at most"),
    ("quantise", dict(x=0), "x is a null device pointer"),
    ("quantise", dict(codes=A + 8), "codes must be 16-byte aligned"),
    ("quantise", dict(scales=0), "scales is a null device pointer"),
    ("quantise", dict(x_stride=992), "x_stride must be at least 1000"),
    ("quantise", dict(codes_stride=496), "codes_stride must be at least 512"),
    ("quantise", dict(codes_stride=520), "codes_stride must be a multiple of 16"),
    ("quantise", dict(scales_stride=16, columns=520, codes_stride=512, x_stride=1000), "scales_stride must be at least 32"),
    ("quantise", dict(scales_stride=40), "scales_stride must be a multiple of 16"),
    ("quantise", dict(codes_stride=1 << 24), "codes_stride must be at most"),
    ("quantise", dict(sequences=2), "starts is a null device pointer"),
    ("dequantise", dict(columns=12), "columns must be a positive multiple of 8"),
    ("dequantise", dict(scales=A + 4), "scales must be 16-byte aligned"),
    ("quantised_linear", dict(type=2), "type must be DHX_F16 or DHX_BF16"),
    ("quantised_linear", dict(rows=(1 << 27) + 1), "rows must be at most"),
    ("quantised_linear", dict(rows=1 << 27, outputs=1 << 20), "the number of tiles of 256 x 128 outputs must be at most"),
    ("quantised_linear", dict(inputs=60), "inputs must be a positive multiple of 8"),
    ("quantised_linear", dict(outputs=0), "outputs must be a positive multiple of 8"),
    ("quantised_linear", dict(w=0), "w is a null device pointer"),
    ("quantised_linear", dict(w_scales=A + 8), "w_scales must be 16-byte aligned"),
    ("quantised_linear", dict(bias=A + 4), "bias must be 16-byte aligned"),
    ("quantised_linear", dict(y=0), "y is a null device pointer"),
    ("quantised_linear", dict(w_stride=496), "w_stride must be at least 512"),
    ("quantised_linear", dict(scales_stride=24), "scales_stride must be a multiple of 16"),
    ("quantised_linear", dict(y_stride=1272), "y_stride must be at least 1280"),
    ("quantised_linear", dict(starts=0), "starts is a null device pointer"),
    ("quantised_linear", dict(workspace_bytes=100), "the workspace has 100 bytes"),
    ("quantised_linear", dict(workspace=A + 8), "workspace must be 16-byte aligned"),
    ("gated", dict(type=5), "type must be DHX_F16 or DHX_BF16"),
    ("gated", dict(activation=5), "activation must be one of"),
    ("gated", dict(reserved=1), "reserved must be 0"),
    ("gated", dict(gate_scales=A), "gate_scales and up_scales come together"),
    ("gated", dict(up_scales=A), "gate_scales and up_scales come together"),
    ("gated", dict(up=0), "up is a null device pointer"),
    ("gated", dict(gate=A + 2), "gate must be 16-byte aligned"),
    ("gated", dict(up_bias=A + 8), "up_bias must be 16-byte aligned"),
    ("gated", dict(out=0), "out is a null device pointer"),
    ("gated", dict(w_stride=56), "w_stride must be at least 64"),
    ("gated", dict(out_stride=1272), "out_stride must be at least 1280"),
    ("gated_four", dict(w_stride=16), "w_stride must be at least 32"),
    ("gated_four", dict(scales_stride=0), "scales_stride must be at least 16"),
    ("gated_four", dict(up_scales=A + 1), "up_scales must be 16-byte aligned"),
    ("gated_four", dict(workspace_bytes=0), "the workspace has 0 bytes"),
]


@pytest.mark.parametrize("name,change,text", REFUSED)
def test_refused(name, change, text):
    assert text in message(name, **change)


def test_what_may_be_missing():
    for name, change in (("norm", dict(rows=0, x=0, y=0, x_out=0, h=0)), ("norm", PLAIN), ("norm", dict(gate=0, starts=0, sequences=0)),
                         ("norm", dict(pre=0, h=0, pre_weight=0, pre_bias=0)), ("norm", dict(x_out=A, h=2 * A)),
                         ("norm", dict(stream_type=packed.F32)), ("quantise", dict(rows=0, x=0, codes=0, scales=0)),
                         ("quantise", dict(starts=A, sequences=1)), ("quantised_linear", dict(bias=0, starts=0, sequences=0)),
                         ("quantised_linear", dict(rows=0, x=0, y=0, workspace=0, workspace_bytes=0)),
                         ("gated", dict(rows=0, x=0, out=0)), ("gated", dict(starts=A, sequences=9, gate_bias=A))):
        assert message(name, **change) == "null engine", (name, change)


def test_workspaces():
    for name, least in (("quantised_linear", 1000 * (512 + 32)), ("gated_four", 1000 * (32 + 16))):
        function, kind, fields = CALLS[name]
        need = d.packed_workspace(function, kind(**fields))
        assert need >= least
        assert message(name, workspace_bytes=need) == "null engine"
        assert "the call needs" in message(name, workspace_bytes=need - 1)
        assert d.packed_workspace(function, kind(**{**fields, "x": 0, "workspace": 0, "workspace_bytes": 0})) == need
        with pytest.raises(d.DINOv3Error, match="inputs must be"):
            d.packed_workspace(function, kind(**{**fields, "inputs": 12}))
    assert d.packed_workspace("gated", packed.Gated(**GATED)) == 0
    # Few rows are quantised by the product itself.
    assert d.packed_workspace("gated", packed.Gated(**{**GATED_FOUR, "rows": 24})) == 0
    assert message("gated_four", rows=24, workspace=0, workspace_bytes=0) == "null engine"
    assert d.packed_workspace("quantised_linear", packed.QuantisedLinear(**{**QUANTISED_LINEAR, "rows": 1})) == 0
    assert d._lib.dhx_packed_gated_workspace(None, None) == 1


def test_the_timed_ranges_are_taken():
    # Every call that the range of the timed cases can make, with addresses that
    # nothing reads.
    pytest.importorskip("torch")
    spec = importlib.util.spec_from_file_location("more_timed_operators", os.path.join(ROOT, "perf", "more_operators.py"))
    timed = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(timed)
    rng = random.Random(23)
    seen = {}
    for case in timed.listed() + [timed.draw(rng) for _ in range(3000)]:
        op, t = case["op"], {"f16": packed.F16, "bf16": packed.BF16, "f32": packed.F32}[case["type"]]
        if op == "norm":
            n, c, gated = len(timed._lengths(case["lengths"])), case["channels"], case["gated"]
            kinds = {"none": 0, "rms": 1, "layer": 2}
            name, post, pre = "norm", kinds[case["post"]], kinds[case["pre"]]
            change = dict(type=t, stream_type=packed.F32 if case["stream"] == "f32" else t, post=post, pre=pre, channels=c, sequences=n,
                          rows=sum(timed._lengths(case["lengths"])), h=4 * A if pre else 0, post_weight=A if post else 0,
                          pre_weight=A if pre else 0, pre_bias=A if pre == 2 else 0, gate=A if gated else 0,
                          x_stride=c, y_stride=c, x_out_stride=c, h_stride=c, gate_stride=c)
        elif op == "quantise":
            c = case["columns"]
            name, change = "quantise", dict(type=t, rows=case["rows"], columns=c, x_stride=c, codes_stride=(c + 31) // 32 * 16,
                                            scales_stride=timed._pad(c))
        else:
            lengths, i, o = timed._lengths(case["lengths"]), case["inputs"], case["outputs"]
            change = dict(type=t, sequences=len(lengths), rows=sum(lengths), inputs=i, outputs=o, x_stride=i, starts=A)
            if op == "linear4" or case["four"]:
                change.update(w_stride=(i + 31) // 32 * 16, scales_stride=timed._pad(i), workspace_bytes=1 << 40)
            else:
                change.update(w_stride=i)
            name = "quantised_linear" if op == "linear4" else "gated_four" if case["four"] else "gated"
            change["y_stride" if op == "linear4" else "out_stride"] = o
        assert message(name, **change) == "null engine", case
        seen[name] = seen.get(name, 0) + 1
    assert len(seen) == 5 and all(n > 200 for n in seen.values()), seen
