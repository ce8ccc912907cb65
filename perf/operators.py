"""Timed cases of the operators on packed batches, through their public calls.

A packed batch holds the rows of many sequences (images of different sizes,
prompts, single tokens) back to back: sequence s has the rows starts[s] ..
starts[s + 1] - 1. Three operators work on it:

  "linear"     a projection that all sequences share, y = x W^T + bias, plus the
               low-rank adapter of each sequence's own request, scale (x A^T) B^T;
  "rotate"     the position rotation of the heads of each row, with the angles
               of the row's own place in its image or prompt;
  "attention"  softmax attention inside each sequence, with grouped heads,
               causal or not, and any number of queries and keys.

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

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
LARGEST_FLOPS = 1.1e12       # no drawn case costs more than the largest listed one
LARGEST_BYTES = 330e6
EXACT_FLOPS = 2e12           # beyond this the 64-bit form takes too long
PLAIN_SCORES = 1 << 28       # scores that the plain attention holds at a time


def _attention(name, type, queries, keys, heads, kv_heads, head_dim, causal):
    return {"name": name, "op": "attention", "type": type, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "causal": causal}


def _linear(name, type, lengths, inputs, outputs, rank, adapters, bare):
    return {"name": name, "op": "linear", "type": type, "lengths": lengths, "inputs": inputs, "outputs": outputs,
            "rank": rank, "adapters": adapters, "bare": bare}


def _rotate(name, type, lengths, heads, row, head_dim, rotated, prefix, neighbours):
    return {"name": name, "op": "rotate", "type": type, "lengths": lengths, "heads": heads, "row": row,
            "head_dim": head_dim, "rotated": rotated, "prefix": prefix, "neighbours": neighbours}


def listed():
    return [
        # One 224x224 image (196 patches and 5 prefix tokens): latency.
        _attention("attention_image", "f16", "201", "201", 6, 6, 64, False),
        # A server's batch of images of different sizes, 224 to 1024 pixels.
        _attention("attention_images", "f16", "201*24,581*8,261,1029*6,331,405,2309,4101", "201*24,581*8,261,1029*6,331,405,2309,4101",
                   6, 6, 64, False),
        # A head size between the kernels' own, ragged prompts, one of one
        # token and one without any.
        _attention("attention_odd", "bf16", "77,0,1,513,1279,300,64,65", "77,0,1,513,1279,300,64,65", 16, 16, 80, True),
        # Prompts of many requests, grouped heads.
        _attention("attention_prompts", "bf16", "2048,731,1,64,1533,129,977,350,2311,48", "2048,731,1,64,1533,129,977,350,2311,48",
                   32, 8, 128, True),
        # One long prompt.
        _attention("attention_long", "bf16", "16384", "16384", 16, 4, 128, True),
        # One new token of each of 48 requests against all its keys.
        _attention("attention_single", "bf16", "1*48", "8192,4097,6000*4,1,130,2048*16,777*8,3500*10,1025*6", 32, 8, 128, True),
        # Single tokens through an adapted projection, a request each.
        _linear("linear_single", "bf16", "1*24", 4096, 4096, 16, 24, 0),
        # A batch of images through the QKV projection, eight fine-tuned
        # variants of one backbone and some requests without one.
        _linear("linear_images", "f16", "201*64", 384, 1152, 16, 8, 8),
        # Ragged images through the down projection.
        _linear("linear_ragged", "f16", "201*7,581,33,1029*3,1,0,405,2309", 1536, 384, 8, 5, 3),
        # Prompts through a large projection.
        _linear("linear_prompts", "bf16", "4096,1024*6,511,513,2048*2,1024", 4096, 4096, 32, 6, 0),
        # The q and k heads of packed image rows, as the projection leaves them.
        _rotate("rotate_images", "f16", "201*64", 12, 1152, 64, 64, 5, False),
        # The same of prompts with grouped heads (32 and 8 of them), neighbours
        # paired.
        _rotate("rotate_prompts", "bf16", "2048,731,1,64,1533,129,977,350,2311,48", 40, 6144, 128, 128, 0, True),
    ]


def _lengths(text):
    out = []
    for part in text.split(","):
        n, _, times = part.partition("*")
        out += [int(n)] * int(times or 1)
    return out


def _text(lengths):
    return ",".join(str(n) for n in lengths)


def _spread(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def _split(rng, total, most):
    """Lengths of up to `most` sequences, `total` rows together."""
    n = min(total, _spread(rng, 1, most))
    shares = [rng.expovariate(1.0) + 0.02 for _ in range(n)]
    got = [int(total * s / sum(shares)) for s in shares]
    got[rng.randrange(n)] += total - sum(got)
    return got


def _draw_attention(rng):
    head_dim = rng.choice((64, 64, 64, 128, 128, 128, 32, 80, 96))
    kv_heads = rng.choice((1, 2, 3, 4, 6, 8, 12))
    heads = kv_heads * rng.choice((1, 1, 1, 2, 3, 4, 8))
    case = {"op": "attention", "type": rng.choice(("f16", "bf16")), "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "causal": rng.random() < 0.6}
    kind = rng.choice(("same", "same", "same", "few", "apart"))
    if kind == "same":  # whole images or prompts
        keys = _split(rng, _spread(rng, 16, 12000), 64)
        queries = keys
    elif kind == "few":  # single tokens, pooling queries
        keys = [_spread(rng, 1, 8192) for _ in range(_spread(rng, 1, 64))]
        few = rng.choice((1, 1, 1, 2, 5, 8))
        queries = [few] * len(keys)
    else:  # a prompt's next part, or queries of another kind; keys may be fewer
        keys = [_spread(rng, 1, 4096) for _ in range(_spread(rng, 1, 16))]
        queries = [_spread(rng, 1, 1024) for _ in keys]
        if rng.random() < 0.5:
            keys[rng.randrange(len(keys))] = 0
    return dict(case, queries=_text(queries), keys=_text(keys))


def _draw_linear(rng):
    rows = _spread(rng, 1, 16384)
    lengths = [1] * min(rows, 96) if rng.random() < 0.3 else _split(rng, rows, 64)
    sequences = len(lengths)
    return {"op": "linear", "type": rng.choice(("f16", "bf16")), "lengths": _text(lengths),
            "inputs": 8 * _spread(rng, 16, 512), "outputs": 8 * _spread(rng, 16, 512),
            "rank": rng.choice((8, 16, 16, 24, 32, 64)), "adapters": _spread(rng, 1, min(32, sequences)),
            "bare": rng.choice((0, 0, sequences // 4))}


def _draw_rotate(rng):
    head_dim = rng.choice((64, 64, 128, 128, 80, 32))
    rotated = head_dim if rng.random() < 0.7 else head_dim // 2
    heads = rng.choice((1, 6, 8, 12, 24, 32, 40))
    prefix = rng.choice((0, 0, 5))
    row = heads * head_dim + (rng.choice((0, 1, 6)) * head_dim)
    return {"op": "rotate", "type": rng.choice(("f16", "bf16")), "lengths": _text(_split(rng, _spread(rng, 16, 16384), 64)),
            "heads": heads, "row": row, "head_dim": head_dim, "rotated": rotated, "prefix": prefix,
            "neighbours": rng.random() < 0.5}


def draw(rng):
    while True:
        case = rng.choice((_draw_attention, _draw_attention, _draw_linear, _draw_linear, _draw_rotate))(rng)
        cost = work(case)
        if cost["flops"] <= LARGEST_FLOPS and cost["bytes"] <= LARGEST_BYTES:
            return case


def _visible(queries, keys, causal):
    """Pairs of a query and a key that it sees."""
    if not causal:
        return sum(q * k for q, k in zip(queries, keys))
    pairs = 0
    for q, k in zip(queries, keys):
        first = max(0, q - k)  # queries before it see nothing
        seen = q - first
        pairs += seen * k - seen * (seen - 1) // 2
    return pairs


def _adapter_of(case):
    """The adapter of each sequence: round robin, `bare` sequences have none."""
    n = len(_lengths(case["lengths"]))
    return [-1 if s < case["bare"] else (s * 5) % case["adapters"] for s in range(n)]


def work(case):
    if case["op"] == "attention":
        q, k, d = _lengths(case["queries"]), _lengths(case["keys"]), case["head_dim"]
        rows = 2 * sum(q) * case["heads"] + 2 * sum(k) * case["kv_heads"]
        return {"bytes": 2 * rows * d, "flops": 4 * d * case["heads"] * _visible(q, k, case["causal"])}
    lengths = _lengths(case["lengths"])
    rows = sum(lengths)
    if case["op"] == "linear":
        adapter = _adapter_of(case)
        adapted = sum(n for n, a in zip(lengths, adapter) if a >= 0)
        used = len({a for n, a in zip(lengths, adapter) if a >= 0 and n > 0})
        i, o, r = case["inputs"], case["outputs"], case["rank"]
        return {"bytes": 2 * (rows * (i + o) + i * o + used * r * (i + o)) + 4 * o,
                "flops": 2 * rows * i * o + 2 * adapted * r * (i + o)}
    h, d, r = case["heads"], case["head_dim"], case["rotated"]
    tables = max(lengths) * r // 2 * 8
    return {"bytes": 4 * rows * h * d + tables + 4 * rows, "flops": 3 * rows * h * r}


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _device_ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    """The tensors of a case, from its seed."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    if case["op"] == "attention":
        q, k, d = sum(_lengths(case["queries"])), sum(_lengths(case["keys"])), case["head_dim"]
        # Queries are scaled so that some keys carry most of a row's weight.
        return {"q": normal(q, case["heads"], d, scale=2.0), "k": normal(k, case["kv_heads"], d),
                "v": normal(k, case["kv_heads"], d)}
    lengths = _lengths(case["lengths"])
    rows = sum(lengths)
    if case["op"] == "linear":
        i, o, r, n = case["inputs"], case["outputs"], case["rank"], case["adapters"]
        return {"x": normal(rows, i), "w": normal(o, i, scale=i ** -0.5),
                "bias": torch.randn(o, generator=g, device="cuda") * 0.1, "a": normal(n, r, i, scale=i ** -0.5),
                "b": normal(n, o, r, scale=r ** -0.5), "scale": torch.rand(n, generator=g, device="cuda") + 0.5}
    # A row's q and k heads at the front of a longer row (v behind them).
    places = max(lengths)
    freq = 100.0 ** (-torch.arange(case["rotated"] // 2, dtype=torch.float64) / (case["rotated"] // 2))
    angle = torch.arange(places, dtype=torch.float64)[:, None] * freq
    return {"rows": normal(rows, case["row"]), "cos": angle.cos().float().cuda(), "sin": angle.sin().float().cuda()}


def _places(case):
    """The table row of each row: its place behind the prefix, -1 in the prefix."""
    return [p if p >= 0 else -1 for n in _lengths(case["lengths"]) for p in range(-case["prefix"], n - case["prefix"])]


_engine = None


def _engine_of():
    global _engine
    if _engine is None:
        from dinov3_hrx import Engine
        _engine = Engine(0)
    return _engine


def prepare(case, seed):
    state = {"case": case, "in": _inputs(case, seed)}
    x = state["in"]
    if case["op"] == "attention":
        q, k = _lengths(case["queries"]), _lengths(case["keys"])
        state["queries"], state["keys"] = _starts(q), _starts(k)
        state["q_starts"] = _device_ints(state["queries"])
        state["k_starts"] = state["q_starts"] if q == k else _device_ints(state["keys"])
    else:
        state["rows"] = _starts(_lengths(case["lengths"]))
        state["starts"] = _device_ints(state["rows"])
        if case["op"] == "linear":
            state["adapter"] = _adapter_of(case)
            state["ids"] = _device_ints(state["adapter"])
            rows = {}
            for s, a in enumerate(state["adapter"]):
                rows.setdefault(a, []).append((state["rows"][s], state["rows"][s + 1]))
            state["rows_of"] = {a: torch.cat([torch.arange(b, e, device="cuda") for b, e in spans])
                                for a, spans in rows.items() if a >= 0}
        else:
            state["index"] = _device_ints(_places(case))
    if own:
        from dinov3_hrx import packed
        state["engine"] = e = _engine_of()
        t = packed.F16 if case["type"] == "f16" else packed.BF16
        if case["op"] == "attention":
            d = case["head_dim"]
            out = torch.empty_like(x["q"])
            call = packed.Attention(
                type=t, causal=case["causal"], sequences=len(q), heads=case["heads"], kv_heads=case["kv_heads"], head_dim=d,
                q_rows=sum(q), k_rows=sum(k), longest_q=max(q), longest_k=max(k), scale=d ** -0.5,
                q=x["q"].data_ptr(), k=x["k"].data_ptr(), v=x["v"].data_ptr(), out=out.data_ptr(),
                q_stride=case["heads"] * d, k_stride=case["kv_heads"] * d, v_stride=case["kv_heads"] * d,
                out_stride=case["heads"] * d, q_starts=state["q_starts"].data_ptr(), k_starts=state["k_starts"].data_ptr())
            need = e.packed_attention_workspace(call)
        elif case["op"] == "linear":
            i, o, rows = case["inputs"], case["outputs"], sum(_lengths(case["lengths"]))
            out = torch.empty(rows, o, dtype=x["x"].dtype, device="cuda")
            call = packed.Linear(
                type=t, sequences=len(state["adapter"]), rows=rows, inputs=i, outputs=o, rank=case["rank"],
                adapters=case["adapters"], x=x["x"].data_ptr(), w=x["w"].data_ptr(), bias=x["bias"].data_ptr(),
                a=x["a"].data_ptr(), b=x["b"].data_ptr(), scale=x["scale"].data_ptr(), y=out.data_ptr(),
                x_stride=i, w_stride=i, y_stride=o, starts=state["starts"].data_ptr(), adapter=state["ids"].data_ptr())
            need = e.packed_linear_workspace(call)
        else:
            out = torch.empty(x["rows"].shape[0], case["heads"], case["head_dim"], dtype=x["rows"].dtype, device="cuda")
            call = packed.Rotation(
                type=t, neighbours=case["neighbours"], rows=x["rows"].shape[0], heads=case["heads"],
                head_dim=case["head_dim"], rotated=case["rotated"], places=x["cos"].shape[0], x=x["rows"].data_ptr(),
                out=out.data_ptr(), x_stride=case["row"], out_stride=case["heads"] * case["head_dim"],
                cos=x["cos"].data_ptr(), sin=x["sin"].data_ptr(), index=state["index"].data_ptr())
            need = 0
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        if case["op"] != "rotate":
            call.workspace, call.workspace_bytes = workspace.data_ptr(), need
        state.update(out=out, call=call, workspace=workspace)
    return state


def run(state):
    case = state["case"]
    if own:
        e, stream = state["engine"], torch.cuda.current_stream().cuda_stream
        if case["op"] == "attention":
            e.packed_attention(state["call"], stream)
        elif case["op"] == "linear":
            e.packed_linear(state["call"], stream)
        else:
            e.packed_rotate(state["call"], stream)
        return state["out"]
    return {"attention": _plain_attention, "linear": _plain_linear, "rotate": _plain_rotate}[case["op"]](state)


def _plain_attention(state):
    case, x = state["case"], state["in"]
    heads, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    group = heads // kv
    out = torch.zeros(x["q"].shape, dtype=torch.float32, device="cuda")
    q_all = x["q"].float() * d ** -0.5
    k_all, v_all = x["k"].float(), x["v"].float()
    for s in range(len(state["queries"]) - 1):
        q0, q1, k0, k1 = state["queries"][s], state["queries"][s + 1], state["keys"][s], state["keys"][s + 1]
        lq, lk = q1 - q0, k1 - k0
        if lq == 0 or lk == 0:
            continue
        k = k_all[k0:k1].permute(1, 2, 0).contiguous()  # [kv][d][lk]
        v = v_all[k0:k1].permute(1, 0, 2).contiguous()  # [kv][lk][d]
        step = max(1, PLAIN_SCORES // (heads * lk))
        for b in range(0, lq, step):
            e = min(lq, b + step)
            q = q_all[q0 + b:q0 + e].view(e - b, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * (e - b), d)
            p = torch.matmul(q, k).view(kv, group, e - b, lk)
            if case["causal"]:
                last = torch.arange(b, e, device="cuda")[:, None] + (lk - lq)
                p.masked_fill_(torch.arange(lk, device="cuda") > last, -math.inf)
            top = p.amax(-1, keepdim=True).clamp_min(-3e38)  # a row that sees nothing
            p = p.sub_(top).exp_()
            total = p.sum(-1, keepdim=True).clamp_min(1e-30)
            o = torch.matmul(p.view(kv, group * (e - b), lk), v).view(kv, group, e - b, d) / total
            out[q0 + b:q0 + e] = o.permute(2, 0, 1, 3).reshape(e - b, heads, d)
    return out.to(x["q"].dtype)


def _plain_linear(state):
    x = state["in"]
    rows = x["x"].float()
    y = rows @ x["w"].float().t() + x["bias"]
    for a, at in state["rows_of"].items():
        y[at] += x["scale"][a] * (rows[at] @ x["a"][a].float().t() @ x["b"][a].float().t())
    return y.to(x["x"].dtype)


def _plain_rotate(state):
    case, x = state["case"], state["in"]
    h, d, r = case["heads"], case["head_dim"], case["rotated"]
    rows = x["rows"][:, :h * d].float().view(-1, h, d)
    at = state["index"].long()
    turned = (at >= 0)[:, None, None]
    c, s = x["cos"][at.clamp_min(0)][:, None], x["sin"][at.clamp_min(0)][:, None]
    out = rows.clone()
    first = slice(0, r, 2) if case["neighbours"] else slice(0, r // 2)
    second = slice(1, r, 2) if case["neighbours"] else slice(r // 2, r)
    x1, x2 = rows[..., first], rows[..., second]
    out[..., first] = torch.where(turned, x1 * c - x2 * s, x1)
    out[..., second] = torch.where(turned, x2 * c + x1 * s, x2)
    return out.to(x["rows"].dtype)


def exact(case, seed):
    """The operators by their definitions in float64."""
    if work(case)["flops"] > EXACT_FLOPS:
        return None
    x = {name: t.double() for name, t in _inputs(case, seed).items()}
    if case["op"] == "attention":
        q_lens, k_lens = _lengths(case["queries"]), _lengths(case["keys"])
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros_like(x["q"])
        q_at = k_at = 0
        for lq, lk in zip(q_lens, k_lens):
            skip = max(0, lq - lk) if case["causal"] else 0
            if lk and lq > skip:
                for h in range(case["heads"]):
                    # The queries that see a key, against all keys.
                    q = x["q"][q_at + skip:q_at + lq, h]
                    s = q @ x["k"][k_at:k_at + lk, h // group].t().contiguous() / math.sqrt(case["head_dim"])
                    if case["causal"]:
                        s = s + torch.full_like(s, -math.inf).triu(lk - (lq - skip) + 1)
                    e = torch.exp(s - s.max(1, keepdim=True).values)
                    out[q_at + skip:q_at + lq, h] = (e @ x["v"][k_at:k_at + lk, h // group]) / e.sum(1, keepdim=True)
            q_at, k_at = q_at + lq, k_at + lk
        return out
    if case["op"] == "linear":
        out, at = [], 0
        for n, a in zip(_lengths(case["lengths"]), _adapter_of(case)):
            w = x["w"] if a < 0 else x["w"] + x["scale"][a] * (x["b"][a] @ x["a"][a])
            out.append(x["x"][at:at + n] @ w.t().contiguous() + x["bias"])
            at += n
        return torch.cat(out)
    h, d, r = case["heads"], case["head_dim"], case["rotated"]
    rows = x["rows"][:, :h * d].reshape(-1, h, d)
    # Each pair as a complex number, times the complex number of its angle.
    pair = rows[..., :r].reshape(-1, h, r // 2, 2) if case["neighbours"] else rows[..., :r].reshape(-1, h, 2, r // 2).transpose(2, 3)
    place = torch.tensor(_places(case), device="cuda")
    turn = torch.complex(x["cos"], x["sin"])[place.clamp_min(0)]
    turn[place < 0] = 1.0
    turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn[:, None])
    turned = turned if case["neighbours"] else turned.transpose(2, 3)
    return torch.cat([turned.reshape(-1, h, r), rows[..., r:]], -1)
