"""Calls of the feed-forward half of a packed block that lie at the edge of what is
taken (CPU only: a null engine shows which check answers), and the documents'
examples of them."""
import ast
import os
import re

import pytest

import test_packed_feed_forward as calls
from test_dma_wait_order import KERNELS
from dinov3_hrx import packed
from test_packed_feed_forward import PLAIN, A, message

X, Y = calls.NORM["x"], calls.NORM["y"]


@pytest.mark.parametrize("change,text", [
    (dict(h=X, h_stride=392), "h in the place of x must have its type, and h_stride be x_stride"),
    (dict(h=X, stream_type=packed.F32), "h in the place of x must have its type"),
    (dict(PLAIN, h=X, h_stride=768), "h in the place of x must have its type"),
    (dict(PLAIN, h=X, stream_type=packed.F32), "h in the place of x must have its type"),
    (dict(x_out=Y, x_out_stride=392), "x_out in the place of y must have its type, and x_out_stride be y_stride"),
    (dict(x_out=Y, stream_type=packed.F32), "x_out in the place of y must have its type"),
    (dict(x_out=Y, h=Y), "h and x_out must not be the same"),
    (dict(x_out=X, h=X), "h and x_out must not be the same"),
])
def test_outputs_in_the_place_of_inputs_refused(change, text):
    # Rows of another size or distance would be written over rows that are not yet read.
    assert text in message("norm", **change)


def test_outputs_in_the_place_of_inputs_taken():
    for change in (dict(h=X), dict(x_out=Y), dict(h=X, x_out=Y), dict(PLAIN, h=X), dict(x_out=X, h=Y), dict(x_out=X, h=Y, stream_type=packed.F32),
                   dict(rows=0, x=0, y=A, x_out=A, h=0, stream_type=packed.F32)):
        assert message("norm", **change) == "null engine", change


def test_the_documents_examples_name_their_stream():
    # The null stream, which a call without one means, does not wait for PyTorch's other
    # streams, nor they for it: an example on the current stream passes it in every call.
    found = 0
    for document in ("README", "INTEGRATION"):
        with open(os.path.join(calls.ROOT, document + ".md")) as f:
            blocks = re.findall(r"```python\n(.*?)```", f.read(), re.S)
        for block in blocks:
            for node in ast.walk(ast.parse(block)):
                name = getattr(getattr(node, "func", None), "attr", "")
                if name.startswith("packed_") and not name.endswith("_workspace"):
                    found += 1
                    assert len(node.args) == 2, f"{document}: {name} without a stream"
    assert found >= 3


def test_launchers_hand_on_nothing_unread():
    # Each field of what a product's launcher hands on is read by the launches.
    with open(os.path.join(KERNELS, "packed_product.hpp")) as f:
        source = f.read()
    fields = re.search(r"struct Product \{(.*?)\n\};", source, re.S).group(1)
    names = re.findall(r"[ *](\w+)[,;]", re.sub(r"//.*", "", fields))
    assert len(names) > 15
    for name in names:
        assert re.search(rf"\bp\.{name}\b", source), name
