"""The operators on packed batches (include/dinov3_packed.h): a projection with
low-rank adapters, the position rotation, and attention, over the rows of many
sequences that lie back to back. A call is described once, with device
addresses as integers, and run by an Engine any number of times:

    from dinov3_hrx import Engine, packed
    call = packed.Attention(type=packed.BF16, causal=1, sequences=n, heads=32, kv_heads=8, head_dim=128, ...)
    bytes = engine.packed_attention_workspace(call)   # the caller's device memory
    engine.packed_attention(call, stream)             # queued, not waited for

The fields and their rules are those of the header. A program that uses PyTorch
imports it before this package: the two then share PyTorch's HIP runtime, while
the other way round each would have its own."""
from __future__ import annotations

import ctypes

F16, BF16 = 0, 1

_u32, _u64, _p = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_void_p


class Linear(ctypes.Structure):
    """dhx_packed_linear."""
    _fields_ = [("type", _u32), ("sequences", _u32), ("rows", _u64), ("inputs", _u32), ("outputs", _u32), ("rank", _u32),
                ("adapters", _u32), ("x", _p), ("w", _p), ("bias", _p), ("a", _p), ("b", _p), ("scale", _p), ("y", _p),
                ("x_stride", _u64), ("w_stride", _u64), ("y_stride", _u64), ("starts", _p), ("adapter", _p),
                ("workspace", _p), ("workspace_bytes", _u64)]


class Rotation(ctypes.Structure):
    """dhx_packed_rotation."""
    _fields_ = [("type", _u32), ("neighbours", _u32), ("rows", _u64), ("heads", _u32), ("head_dim", _u32),
                ("rotated", _u32), ("places", _u32), ("x", _p), ("out", _p), ("x_stride", _u64), ("out_stride", _u64),
                ("cos", _p), ("sin", _p), ("index", _p)]


class Attention(ctypes.Structure):
    """dhx_packed_attention."""
    _fields_ = [("type", _u32), ("causal", _u32), ("sequences", _u32), ("heads", _u32), ("kv_heads", _u32),
                ("head_dim", _u32), ("q_rows", _u64), ("k_rows", _u64), ("longest_q", _u32), ("longest_k", _u32),
                ("scale", ctypes.c_float), ("reserved", _u32), ("q", _p), ("k", _p), ("v", _p), ("out", _p),
                ("q_stride", _u64), ("k_stride", _u64), ("v_stride", _u64), ("out_stride", _u64),
                ("q_head_stride", _u64), ("k_head_stride", _u64), ("v_head_stride", _u64), ("out_head_stride", _u64),
                ("lse", _p), ("q_starts", _p), ("k_starts", _p), ("workspace", _p), ("workspace_bytes", _u64)]


def declare(lib) -> None:
    """Argument types of the C functions."""
    for name, call in (("linear", Linear), ("rotation", Rotation), ("attention", Attention)):
        getattr(lib, f"dhx_packed_{name}_run").argtypes = [_p, ctypes.POINTER(call), _p]
        if call is not Rotation:
            getattr(lib, f"dhx_packed_{name}_workspace").argtypes = [ctypes.POINTER(call), ctypes.POINTER(_u64)]
