"""Timed cases of the feed-forward half of a block on packed batches, through
the public calls: the norms, the gated projection, and products with weights
held in 4 bits.

A packed batch holds the rows of many sequences (images of different sizes,
prompts, single tokens) back to back, as in operators.py. The operators:

  "norm"      x' = x + gate[s] * scale * post(y), h = pre(x'): the residual step
              behind a block, with the norm of the block's output before it and the
              norm of the next block's input behind it (either may be missing;
              LayerNorm or root mean square);
  "gated"     act(x Wg^T + bg) * (x Wu^T + bu), weights in the type of x or in 4
              bits (then x is quantised alike within the call);
  "quantise"  rows to 4-bit values with a scale per 32 of them, and back;
  "linear4"   x Wq^T + bias, the weights Wq in 4 bits and x quantised alike
              within the call.

4-bit values: e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), times 2^e of
the block of 32 along a row that they lie in, e = floor(log2 of the block's largest
magnitude) - 2; nearest, ties to even, what is past 6 becomes 6.

With `own` false, `run` computes them in elementary float32 operations; with
`own` true, it makes the calls of dinov3_hrx's engine.

A case's lengths are a text: "201*64" is 64 sequences of 201 rows, "5,0,17" are
three of 5, 0 and 17.
"""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "dinov3-loom_amd"))

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LARGEST_FLOPS = 1.1e12       # no drawn case costs more than the largest listed one
LARGEST_BYTES = 400e6
BLOCK = 32                   # values that share a scale
MIXED = "2048,731,1,64,1533,129,977,350,2311,48"  # prompts of many requests
RAGGED = "201*7,581,33,1029*3,1,0,405,2309"       # images of different sizes
ODD = "77,0,1,513,1279,300,64,65"                 # ragged prompts, one of one token and one without any


def _norm(name, type, stream, lengths, channels, post, pre, scaled, gated):
    return {"name": name, "op": "norm", "type": type, "stream": stream, "lengths": lengths, "channels": channels,
            "post": post, "pre": pre, "scaled": scaled, "gated": gated}


def _gated(name, type, lengths, inputs, outputs, activation, biased, four):
    return {"name": name, "op": "gated", "type": type, "lengths": lengths, "inputs": inputs, "outputs": outputs,
            "activation": activation, "biased": biased, "four": four}


def _quantise(name, type, rows, columns):
    return {"name": name, "op": "quantise", "type": type, "rows": rows, "columns": columns}


def _linear4(name, type, lengths, inputs, outputs, biased):
    return {"name": name, "op": "linear4", "type": type, "lengths": lengths, "inputs": inputs, "outputs": outputs,
            "biased": biased}


def listed():
    return [
        # One new token of each of 24 requests, norms on both sides of the block:
        # latency.
        _norm("norm_single", "bf16", "bf16", "1*24", 4096, "rms", "rms", False, False),
        # A batch of 224x224 images: LayerScale and the next LayerNorm.
        _norm("norm_images", "f16", "f16", "201*64", 384, "none", "layer", True, False),
        # Prompts with a gate per request, the residual kept in float32.
        _norm("norm_prompts", "bf16", "f32", MIXED, 4096, "rms", "rms", True, True),
        # Single tokens through a large feed-forward: the weights' bytes.
        _gated("gated_single", "bf16", "1*24", 4096, 8192, "silu", False, False),
        # A batch of images through this model's own feed-forward.
        _gated("gated_images", "f16", "201*64", 384, 1536, "silu", True, False),
        # Prompts through a large one.
        _gated("gated_prompts", "bf16", "4096,1024,511,513,2048", 4096, 8192, "silu", False, False),
        # Odd sizes, weights in 4 bits.
        _gated("gated_odd_four", "bf16", ODD, 1000, 2728, "gelu", True, True),
        # Activations of odd rows, whose last block is short.
        _quantise("quantise_odd", "f16", 2299, 1000),
        # The weights of a layer.
        _quantise("quantise_weights", "bf16", 8192, 4096),
        # Single tokens: the weights' bytes, a quarter of 16-bit ones.
        _linear4("linear4_single", "bf16", "1*24", 4096, 4096, False),
        # Ragged images through the down projection.
        _linear4("linear4_ragged", "f16", RAGGED, 1536, 384, True),
        # Prompts through a large projection.
        _linear4("linear4_prompts", "bf16", "4096,1024*6,511,513,2048*2,1024", 4096, 4096, False),
    ]


def _lengths(text):
    out = []
    for part in text.split(","):
        n, _, times = part.partition("*")
        out += [int(n)] * int(times or 1)
    return out


def _spread(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def _split(rng, rows):
    """A text of lengths, `rows` rows together."""
    if rng.random() < 0.25:
        return "1*%d" % rows if rows <= 96 else str(rows)
    n = min(rows, _spread(rng, 1, 64))
    shares = [rng.expovariate(1.0) + 0.02 for _ in range(n)]
    got = [int(rows * s / sum(shares)) for s in shares]
    got[rng.randrange(n)] += rows - sum(got)
    return ",".join(str(n) for n in got)


def _draw_norm(rng):
    type = rng.choice(("f16", "bf16"))
    kinds = ("none", "rms", "layer")
    post = rng.choice(kinds)
    return _norm("", type, rng.choice((type, type, "f32")), _split(rng, _spread(rng, 1, 16384)), 8 * _spread(rng, 8, 1024), post,
                 rng.choice(kinds[1:] if post == "none" else kinds), rng.random() < 0.5, rng.random() < 0.4)


def _draw_gated(rng):
    return _gated("", rng.choice(("f16", "bf16")), _split(rng, _spread(rng, 1, 12864)), 8 * _spread(rng, 16, 512),
                  8 * _spread(rng, 16, 1024), rng.choice(("silu", "silu", "gelu", "gelu_tanh", "relu", "sigmoid")),
                  rng.random() < 0.5, rng.random() < 0.5)


def _draw_quantise(rng):
    return _quantise("", rng.choice(("f16", "bf16")), _spread(rng, 1, 16384), 8 * _spread(rng, 4, 1024))


def _draw_linear4(rng):
    return _linear4("", rng.choice(("f16", "bf16")), _split(rng, _spread(rng, 1, 16384)), 8 * _spread(rng, 16, 512),
                    8 * _spread(rng, 16, 512), rng.random() < 0.5)


def draw(rng):
    while True:
        case = rng.choice((_draw_norm, _draw_gated, _draw_quantise, _draw_linear4))(rng)
        del case["name"]
        cost = work(case)
        if cost["flops"] <= LARGEST_FLOPS and cost["bytes"] <= LARGEST_BYTES:
            return case


def _four_bytes(rows, columns):
    """Bytes of a 4-bit matrix: half a byte a value, and a scale per block of a row."""
    blocks = (columns + BLOCK - 1) // BLOCK
    return rows * (columns // 2 + blocks)


def work(case):
    if case["op"] == "quantise":  # values in, 4 bits out and in, values out
        r, c = case["rows"], case["columns"]
        return {"bytes": 4 * r * c + 2 * _four_bytes(r, c), "flops": 4 * r * c}
    lengths = _lengths(case["lengths"])
    rows = sum(lengths)
    if case["op"] == "norm":
        c = case["channels"]
        stream = 4 if case["stream"] == "f32" else 2
        vectors = (case["post"] != "none") + (case["pre"] != "none") + case["scaled"]
        vectors += (case["post"] == "layer") + (case["pre"] == "layer")
        return {"bytes": rows * c * (2 * stream + 2 + 2 * (case["pre"] != "none")) + 4 * c * vectors + 4 * c * len(lengths) * case["gated"],
                "flops": rows * c * (2 + 6 * (case["post"] != "none") + 6 * (case["pre"] != "none"))}
    i, o = case["inputs"], case["outputs"]
    many = 2 if case["op"] == "gated" else 1
    four = case["op"] == "linear4" or case["four"]
    weights = many * (_four_bytes(o, i) if four else 2 * o * i)
    return {"bytes": 2 * rows * (i + o) + weights + 4 * o * many * case["biased"], "flops": 2 * many * rows * i * o}


def _row_sequences(case):
    """The sequence of each row."""
    n = torch.tensor(_lengths(case["lengths"]))
    return torch.repeat_interleave(torch.arange(n.numel()), n).cuda()


def _pad(columns):
    """Columns of the scales' rows: one per block, rows of whole 16 bytes."""
    return ((columns + BLOCK - 1) // BLOCK + 15) // 16 * 16


def _inputs(case, seed):
    """The tensors of a case, from its seed."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    if case["op"] == "quantise":
        # Some channels are larger than the others, as activations' are.
        wide = 1 + 7 * (torch.rand(case["columns"], generator=g, device="cuda") < 0.02)
        return {"x": (normal(case["rows"], case["columns"]) * wide).to(t)}
    rows = sum(_lengths(case["lengths"]))
    if case["op"] == "norm":
        c = case["channels"]
        x = {"x": (normal(rows, c, scale=2.0) + 0.25).to(TYPES[case["stream"]]), "y": normal(rows, c).to(t)}
        for side in ("post", "pre"):
            if case[side] != "none":
                x[side + "_weight"] = 1 + normal(c, scale=0.2)
            if case[side] == "layer":
                x[side + "_bias"] = normal(c, scale=0.2)
        if case["scaled"]:
            x["scale"] = normal(c, scale=0.3)
        if case["gated"]:
            x["gate"] = normal(len(_lengths(case["lengths"])), c)
        return x
    i, o = case["inputs"], case["outputs"]
    x = {"x": normal(rows, i).to(t)}
    for w in ("gate", "up") if case["op"] == "gated" else ("w",):
        if case["op"] == "linear4" or case["four"]:
            # 4-bit codes of normal values (two in a byte, the first in its low half; a
            # row's last block filled up with zeros) and the blocks' scale bytes, 127 + e.
            blocks = (i + BLOCK - 1) // BLOCK
            codes = torch.zeros(o, blocks * BLOCK, dtype=torch.uint8, device="cuda")
            value = normal(o, i, scale=2.0)
            size = value.abs()
            grid = sum((size >= limit).to(torch.uint8) for limit in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
            codes[:, :i] = grid + 8 * (value < 0)
            x[w] = codes[:, 0::2] + 16 * codes[:, 1::2]
            e = torch.randint(-2, 2, (o, _pad(i)), generator=g, device="cuda") - round(math.log2(2 * i ** 0.5))
            x[w + "_scales"] = (127 + e).to(torch.uint8)
        else:
            x[w] = normal(o, i, scale=i ** -0.5).to(t)
        if case["biased"]:
            x[w + "_bias"] = normal(o, scale=0.1)
    return x


_engine = None


def _engine_of():
    global _engine
    if _engine is None:
        from dinov3_hrx import Engine
        _engine = Engine(0)
    return _engine


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, "in": x}
    if case["op"] != "quantise":
        lengths = _lengths(case["lengths"])
        state["starts"] = torch.tensor([0] + lengths).cumsum(0).int().cuda()
        if case["op"] == "norm" and case["gated"]:
            state["sequence"] = _row_sequences(case)
    if own:
        from dinov3_hrx import packed
        state["engine"] = e = _engine_of()
        types = {"f16": packed.F16, "bf16": packed.BF16, "f32": packed.F32}
        t = types[case["type"]]
        at = {name: v.data_ptr() for name, v in x.items()}
        rows = x["x"].shape[0]
        if case["op"] == "norm":
            c = case["channels"]
            kinds = {"none": packed.NONE, "rms": packed.RMS, "layer": packed.LAYER}
            out = {"x": torch.empty_like(x["x"])}
            if case["pre"] != "none":
                out["h"] = torch.empty_like(x["y"])
            state["call"] = packed.Norm(
                type=t, stream_type=types[case["stream"]], post=kinds[case["post"]], pre=kinds[case["pre"]], rows=rows, channels=c,
                sequences=len(lengths), post_eps=1e-5, pre_eps=1e-5, x=at["x"], y=at["y"], x_out=out["x"].data_ptr(),
                h=out["h"].data_ptr() if "h" in out else 0, x_stride=c, y_stride=c, x_out_stride=c, h_stride=c, gate_stride=c,
                starts=state["starts"].data_ptr(),
                **{k: at.get(k, 0) for k in ("post_weight", "post_bias", "pre_weight", "pre_bias", "scale", "gate")})
            need = 0
        elif case["op"] == "quantise":
            c = case["columns"]
            state["codes"] = torch.empty(rows, (c + BLOCK - 1) // BLOCK * 16, dtype=torch.uint8, device="cuda")
            state["scales"] = torch.empty(rows, _pad(c), dtype=torch.uint8, device="cuda")
            out = torch.empty_like(x["x"])
            state["call"], state["back"] = (packed.Quantisation(
                type=t, rows=rows, columns=c, x=v.data_ptr(), x_stride=c, codes=state["codes"].data_ptr(),
                codes_stride=state["codes"].shape[1], scales=state["scales"].data_ptr(), scales_stride=state["scales"].shape[1])
                for v in (x["x"], out))
            need = 0
        else:
            i, o = case["inputs"], case["outputs"]
            out = torch.empty(rows, o, dtype=x["x"].dtype, device="cuda")
            four = case["op"] == "linear4" or case["four"]
            sizes = dict(type=t, sequences=len(lengths), rows=rows, inputs=i, outputs=o, x=at["x"], x_stride=i, starts=state["starts"].data_ptr(),
                         w_stride=x["w" if case["op"] == "linear4" else "gate"].shape[1], scales_stride=_pad(i) if four else 0)
            if case["op"] == "gated":
                kinds = {"silu": packed.SILU, "gelu": packed.GELU, "gelu_tanh": packed.GELU_TANH, "relu": packed.RELU,
                         "sigmoid": packed.SIGMOID}
                state["call"] = packed.Gated(
                    activation=kinds[case["activation"]], gate=at["gate"], up=at["up"], gate_scales=at.get("gate_scales", 0),
                    up_scales=at.get("up_scales", 0), gate_bias=at.get("gate_bias", 0), up_bias=at.get("up_bias", 0),
                    out=out.data_ptr(), out_stride=o, **sizes)
                need = e.packed_gated_workspace(state["call"])
            else:
                state["call"] = packed.QuantisedLinear(
                    w=at["w"], w_scales=at["w_scales"], bias=at.get("w_bias", 0), y=out.data_ptr(), y_stride=o, **sizes)
                need = e.packed_quantised_linear_workspace(state["call"])
        if need:
            state["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
            state["call"].workspace, state["call"].workspace_bytes = state["workspace"].data_ptr(), need
        state["out"] = out
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        e, stream = state["engine"], torch.cuda.current_stream().cuda_stream
        if op == "norm":
            e.packed_norm(state["call"], stream)
        elif op == "gated":
            e.packed_gated(state["call"], stream)
        elif op == "linear4":
            e.packed_quantised_linear(state["call"], stream)
        else:
            e.packed_quantise(state["call"], stream)
            e.packed_dequantise(state["back"], stream)
        return state["out"]
    return {"norm": _plain_norm, "gated": _plain_gated, "quantise": _plain_quantise, "linear4": _plain_linear4}[op](state)


def _plain_normed(x, side, kind, v):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-5) * x[side + "_weight"]
    return v + x[side + "_bias"] if kind == "layer" else v


def _plain_norm(state):
    case, x = state["case"], state["in"]
    z = _plain_normed(x, "post", case["post"], x["y"].float())
    if case["scaled"]:
        z = z * x["scale"]
    if case["gated"]:
        z = z * x["gate"][state["sequence"]]
    new = x["x"].float() + z
    out = {"x": new.to(x["x"].dtype)}
    if case["pre"] != "none":
        out["h"] = _plain_normed(x, "pre", case["pre"], new).to(x["y"].dtype)
    return out


def _plain_rounded(v):
    """The 4-bit values that the rows of v stand for once quantised, as float32."""
    rows, columns = v.shape
    whole = torch.zeros(rows, (columns + BLOCK - 1) // BLOCK * BLOCK, device="cuda")
    whole[:, :columns] = v
    blocks = whole.view(rows, -1, BLOCK)
    top = blocks.abs().amax(2, keepdim=True)
    e = torch.frexp(top.clamp_min(2.0 ** -126))[1] - 3  # frexp: from 0.5 to 1
    step = torch.ldexp(torch.ones_like(top), e.clamp_min(-120))  # the inputs' blocks are far above
    size = blocks.abs() / step
    value = 0.5 * ((size > 0.25).float() + (size >= 0.75) + (size > 1.25) + (size >= 1.75)) + (size > 2.5) + (size >= 3.5) + 2.0 * (size > 5)
    return (torch.where(blocks < 0, -value, value) * step).view(rows, -1)[:, :columns]


def _plain_weights(codes, scales, columns):
    """The values of 4-bit weights, as float32."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda")
    table = torch.cat([table, -table])
    both = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], 2)
    rows = both.shape[0]
    blocks = both.view(rows, -1, BLOCK)
    step = torch.exp2(scales[:, :blocks.shape[1]].float() - 127)
    return (blocks * step[:, :, None]).view(rows, -1)[:, :columns]


def _plain_quantise(state):
    x = state["in"]["x"]
    return _plain_rounded(x.float()).to(x.dtype)


def _plain_product(x, rows, w):
    columns = rows.shape[1]
    weights = _plain_weights(x[w], x[w + "_scales"], columns) if w + "_scales" in x else x[w].float()
    y = rows @ weights.t()
    return y + x[w + "_bias"] if w + "_bias" in x else y


def _plain_gated(state):
    case, x = state["case"], state["in"]
    rows = x["x"].float()
    if case["four"]:
        rows = _plain_rounded(rows)
    g, u = _plain_product(x, rows, "gate"), _plain_product(x, rows, "up")
    if case["activation"] == "silu":
        g = g / (1 + torch.exp(-g))
    elif case["activation"] == "sigmoid":
        g = 1 / (1 + torch.exp(-g))
    elif case["activation"] == "relu":
        g = g.clamp_min(0)
    elif case["activation"] == "gelu":
        g = 0.5 * g * (1 + torch.erf(g * 2 ** -0.5))
    else:
        g = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    return (g * u).to(x["x"].dtype)


def _plain_linear4(state):
    x = state["in"]
    return _plain_product(x, _plain_rounded(x["x"].float()), "w").to(x["x"].dtype)


def _exact_rounded(v):
    """4-bit rounding of float64 rows: to whole multiples of half the power of two below each value."""
    columns = v.shape[1]
    blocks = torch.nn.functional.pad(v, (0, -columns % BLOCK)).unflatten(1, (-1, BLOCK))
    top = blocks.abs().max(2, keepdim=True).values
    scale = torch.where(top > 0, torch.floor(torch.log2(top.clamp_min(1e-300))) - 2, torch.zeros_like(top))
    # log2 of a value just under a power of two may round up to it.
    scale = scale - (top * torch.exp2(-scale) < 4).double() * (top > 0)
    m = blocks * torch.exp2(-scale)
    step = torch.exp2(torch.floor(torch.log2(m.abs().clamp_min(1))) - 1)
    return (torch.round(m / step) * step).clamp(-6, 6).mul(torch.exp2(scale)).flatten(1)[:, :columns]


def _exact_weights(codes, scales, columns):
    """e2m1 by its parts: sign, two bits of exponent, one of mantissa."""
    c = torch.stack([codes.long() % 16, codes.long() // 16], 2).flatten(1)[:, :columns]
    sign, exponent, mantissa = 1 - 2 * (c // 8), c // 2 % 4, c % 2
    value = torch.where(exponent == 0, 0.5 * mantissa.double(), (1 + 0.5 * mantissa.double()) * torch.exp2(exponent.double() - 1))
    return sign * value * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)[:, :columns]


def _exact_normed(v, kind, weight, bias):
    if kind == "none":
        return v
    if kind == "layer":
        var, mean = torch.var_mean(v, 1, correction=0, keepdim=True)
        return (v - mean) / torch.sqrt(var + 1e-5) * weight + bias
    return v / torch.sqrt(v.square().sum(1, keepdim=True) / v.shape[1] + 1e-5) * weight


def exact(case, seed):
    """The operators by their definitions in float64."""
    x = _inputs(case, seed)
    if case["op"] == "quantise":
        return _exact_rounded(x["x"].double())
    if case["op"] == "norm":
        x = {name: v.double() for name, v in x.items()}
        z = _exact_normed(x["y"], case["post"], x.get("post_weight"), x.get("post_bias"))
        out, at, rows = {}, 0, []
        for s, n in enumerate(_lengths(case["lengths"])):
            rows.append(z[at:at + n] * x.get("scale", 1.0) * (x["gate"][s] if case["gated"] else 1.0))
            at += n
        out["x"] = x["x"] + torch.cat(rows)
        if case["pre"] != "none":
            out["h"] = _exact_normed(out["x"], case["pre"], x.get("pre_weight"), x.get("pre_bias"))
        return out
    rows = x["x"].double()
    i = case["inputs"]
    if case["op"] == "linear4" or case["four"]:
        rows = _exact_rounded(rows)

    def product(w):
        scales = x.get(w + "_scales")
        weights = x[w].double() if scales is None else _exact_weights(x[w], scales, i)
        return torch.nn.functional.linear(rows, weights, x[w + "_bias"].double() if case["biased"] else None)

    if case["op"] == "linear4":
        return product("w")
    g, u = product("gate"), product("up")
    name = case["activation"]
    if name in ("silu", "sigmoid"):
        g = torch.sigmoid(g) * (g if name == "silu" else 1)
    elif name == "relu":
        g = torch.relu(g)
    else:
        g = torch.nn.functional.gelu(g, approximate="tanh" if name == "gelu_tanh" else "none")
    return g * u
