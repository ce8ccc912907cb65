"""The operators on packed batches as a block uses them together: norm, projection,
rotation, attention, projection, residual step with LayerScale and norm, gated
projections, projection down, residual step, on images of different sizes, each
stage checked against float64; the norm, the gated projections and the residual step
against the engine's own kernels on 224x224 images; captured into graphs and replayed
for other inputs and lengths; on streams side by side; every tile and route of the
products; far strides; more rows than workgroups; starts of any kind; failures."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import dinov3_hrx as d  # noqa: E402
from dinov3_hrx import packed  # noqa: E402

from conftest import from_frag, to_frag  # noqa: E402
from packed_chain import Block as Attention  # noqa: E402
from packed_feed_forward import (activation_want, at, four, gated_want, norm_want, pad16, product_want, quantisation, quantised,  # noqa: E402
                                 quantised_want, run_gated, run_linear4, run_norm, step_want, values, weights4)
from packed_operators import F, attention_want, gen, half_step, ints, linear_want, normal, run_attention, run_linear, starts_of, within  # noqa: E402
from test_kernels_gpu import K_LN, K_RESID, K_SWIGLU, _keys, pack_gateup  # noqa: E402

pytestmark = pytest.mark.gpu
HIDDEN, FF, HEADS, DIM, PREFIX = 384, 1536, 6, 64, 5


@pytest.fixture(scope="module")
def eng(gpu):
    e = d.Engine(0)
    yield e
    e.close()


class Block:
    """A block's buffers for `rows` rows and `sequences`; bits: of the feed-forward
    weights."""

    def __init__(self, e, dt, rows, sequences, seed, bits=16, wide=False):
        g = gen(seed)
        self.attention = Attention(dt, rows, sequences, seed)
        self.e, self.dt, self.bits, self.rows = e, dt, bits, rows
        self.x = torch.empty(rows, HIDDEN, dtype=torch.float32 if wide else dt, device="cuda")
        self.h = self.attention.x  # what the projection to q, k and v reads
        self.starts = self.attention.starts
        vector = lambda n=HIDDEN: torch.randn(n, generator=g, device="cuda") * 0.2  # noqa: E731
        self.norms = [{"pre_weight": 1 + vector(), "pre_bias": vector()} for _ in range(3)]
        self.scales = [vector() for _ in range(2)]
        self.biases = [vector(FF), vector(FF), vector()]
        if bits == 4:
            self.gate, self.up, self.down = (weights4(e, g, o, i, dt) for o, i in ((FF, HIDDEN), (FF, HIDDEN), (HIDDEN, FF)))
        else:
            self.gate, self.up, self.down = (normal(g, dt, o, i, scale=i ** -0.5) for o, i in ((FF, HIDDEN), (FF, HIDDEN), (HIDDEN, FF)))
            self.none = torch.zeros(1, 8, FF, device="cuda").to(dt), torch.zeros(1, HIDDEN, 8, device="cuda").to(dt)
            self.bare = ints([-1] * sequences)
        self.act = torch.empty(rows, FF, dtype=dt, device="cuda")
        self.out = torch.empty(rows, HIDDEN, dtype=dt, device="cuda")
        self.ws = [torch.empty(1 << 22, dtype=torch.uint8, device="cuda") for _ in range(2)]

    def fill(self, lengths, ids, seed):
        st = self.attention.fill(lengths, ids, seed)
        self.x.copy_(normal(gen(seed + 1), torch.float32, self.rows, HIDDEN, scale=2.0))
        return st

    def first(self, stream=0):
        run_norm(self.e, self.x, None, None, self.h, "none", "layer", starts=self.starts, stream=stream, **self.norms[0])

    def step(self, i, stream=0):
        run_norm(self.e, self.x, self.attention.out if i == 1 else self.out, self.x, self.h, "none", "layer", scale=self.scales[i - 1],
                 starts=self.starts, stream=stream, **self.norms[i])

    def gated(self, stream=0):
        four_bits = self.bits == 4
        run_gated(self.e, self.h, self.gate[0] if four_bits else self.gate, self.up[0] if four_bits else self.up, *self.biases[:2], self.act,
                  "silu", (self.gate[1], self.up[1]) if four_bits else None, self.starts, self.ws[0], stream)

    def project(self, stream=0):
        if self.bits == 4:
            run_linear4(self.e, self.act, *self.down[:2], self.biases[2], self.out, self.starts, self.ws[1], stream)
        else:
            run_linear(self.e, self.act, self.down, self.biases[2], *self.none, torch.ones(1, device="cuda") if stream == 0 else self.scales[0],
                       self.out, self.starts, self.bare, stream=stream, workspace=self.ws[1])

    def run(self, stream=0):
        self.first(stream)
        self.attention.run(self.e, stream, (0, 0))
        self.step(1, stream)
        self.gated(stream)
        self.project(stream)
        self.step(2, stream)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits,wide", [(16, False), (4, True), (4, False)])
@pytest.mark.parametrize("lengths", [[201, 6, 581, 1, 0, 101, 1029], [1, 0, 7]])
def test_block_stage_by_stage(eng, dt, bits, wide, lengths):
    ids = [(s * 2) % 4 - 1 for s in range(len(lengths))]
    b = Block(eng, dt, sum(lengths) + 30, len(lengths), 3, bits, wide)
    st = b.fill(lengths, ids, 4)
    n = st[-1]
    start = b.x.clone()
    for t in (b.h, b.act, b.out, b.attention.out):
        t.fill_(7.0)
    b.first()
    torch.cuda.synchronize()
    _, (want, e) = step_want(b.x[:n], None, "none", "layer", b.norms[0], None)
    within(b.h[:n], want, e, dt)
    b.attention.run(eng, hints=(0, 0))  # checked stage by stage in packed_chain.py
    before = b.x.clone()
    b.step(1)
    torch.cuda.synchronize()
    (want, e), (want_h, eh) = step_want(before[:n], b.attention.out[:n], "none", "layer", dict(b.norms[1], scale=b.scales[0]), None)
    within(b.x[:n], want, e, b.x.dtype)
    within(b.h[:n], want_h, eh, dt)
    b.gated()
    torch.cuda.synchronize()
    w = [t[2] if bits == 4 else t.double() for t in (b.gate, b.up, b.down)]
    given = lambda t: values(*(v.cuda() for v in quantised_want(t)), t.shape[1]) if bits == 4 else t.double()  # noqa: E731
    want, e = gated_want("silu", given(b.h[:n]), w[0], w[1], b.biases[0], b.biases[1])
    within(b.act[:n], want, e, dt)
    b.project()
    torch.cuda.synchronize()
    want, e = product_want(given(b.act[:n]), w[2], b.biases[2])
    within(b.out[:n], want, e, dt)
    before = b.x.clone()
    b.step(2)
    torch.cuda.synchronize()
    (want, e), (want_h, eh) = step_want(before[:n], b.out[:n], "none", "layer", dict(b.norms[2], scale=b.scales[1]), None)
    within(b.x[:n], want, e, b.x.dtype)
    within(b.h[:n], want_h, eh, dt)
    for t in (b.h, b.act, b.out):  # rows of no sequence
        assert (t[n:] == 7.0).all()
    assert torch.equal(b.x[n:], start[n:])
    # And all of them queued at once.
    alone = b.x.clone(), b.h.clone()
    b.x.copy_(start)
    b.run()
    torch.cuda.synchronize()
    assert torch.equal(b.x, alone[0]) and torch.equal(b.h, alone[1])


def test_against_the_engines_own_kernels(eng):
    # LayerNorm, SwiGLU and the residual step in the engine's fragment order, on the
    # rows of two 224x224 images, and the packed ones on the same: both sides are within
    # the arithmetic's bound and one rounding of the definition.
    rows = 402
    g = gen(21)
    x = normal(g, torch.float16, rows, HIDDEN, scale=2.0)
    gamma, beta = 1 + torch.randn(HIDDEN, generator=g, device="cuda") * 0.2, torch.randn(HIDDEN, generator=g, device="cuda") * 0.2
    gate, up = (normal(g, torch.float16, FF, HIDDEN, scale=0.05) for _ in range(2))
    gb, ub = (torch.randn(FF, generator=g, device="cuda") * 0.2 for _ in range(2))
    down, db = normal(g, torch.float16, HIDDEN, FF, scale=0.03), torch.randn(HIDDEN, generator=g, device="cuda") * 0.1
    ls = torch.rand(HIDDEN, generator=g, device="cuda") + 0.5
    frag = lambda t: eng.weight(to_frag(t.cpu().numpy()))  # noqa: E731
    plain = lambda t: eng.weight(np.ascontiguousarray(t.cpu().numpy()))  # noqa: E731
    u = half_step(torch.float16)

    def own(kernel, scalars, bindings, out, columns):
        key = next(_keys)
        eng.record(key, [(kernel, scalars, bindings)])
        eng.replay(key)
        eng.synchronize()
        padded = (rows + 31) // 32 * 32
        eng.reserve_readback(padded * columns * 2)
        return torch.from_numpy(np.array(from_frag(eng.read(out, np.float16, (padded * columns,)), rows, columns))).cuda()

    def both_near(mine, theirs, want, e):
        within(mine, want, e, torch.float16)
        # the engine's own tolerance (test_kernels_gpu.py) beside this side's bound
        assert ((mine.double() - theirs.double()).abs() <= e + 2e-3 + 2 * u * want.abs()).all()

    def room(columns):
        return eng.allocate((rows + 31) // 32 * 32 * columns * 2)

    h = torch.empty_like(x)
    run_norm(eng, x, None, None, h, "none", "layer", pre_weight=gamma, pre_bias=beta, eps=(1e-5, 1e-5))
    torch.cuda.synchronize()
    buffer = room(HIDDEN)
    theirs = own(K_LN, [rows], [frag(x), plain(gamma), plain(beta), buffer], buffer, HIDDEN)
    want, e = norm_want(x.double(), torch.zeros_like(x, dtype=torch.float64), "layer", 1e-5, gamma, beta)
    both_near(h, theirs, want, e)
    act = torch.empty(rows, FF, dtype=torch.float16, device="cuda")
    run_gated(eng, h, gate, up, gb, ub, act, "silu")
    torch.cuda.synchronize()
    w, b = pack_gateup(*(t.cpu().numpy() for t in (gate, up, gb, ub)))
    buffer = room(FF)
    theirs = own(K_SWIGLU, [rows], [frag(h), eng.weight(to_frag(w)), eng.weight(np.ascontiguousarray(b)), buffer], buffer, FF)
    want, e = gated_want("silu", h.double(), gate.double(), up.double(), gb, ub)
    both_near(act, theirs, want, e)
    out, new = torch.empty_like(x), torch.empty_like(x)
    none = torch.zeros(1, 8, FF, device="cuda").half(), torch.zeros(1, HIDDEN, 8, device="cuda").half()
    run_linear(eng, act, down, db, *none, torch.ones(1, device="cuda"), out, ints([0, rows]), ints([-1]))
    run_norm(eng, x, out, new, None, scale=ls, starts=ints([0, rows]))
    torch.cuda.synchronize()
    buffer = frag(x)
    theirs = own(K_RESID, [rows, FF], [frag(act), frag(down), plain(db), plain(ls), buffer], buffer, HIDDEN)
    want, e = product_want(act.double(), down.double(), db)
    e = ls.double() * (e + u * (want.abs() + e)) + 3 * F * (want.abs() * ls.double() + x.double().abs())  # out is rounded here
    both_near(new, theirs, x.double() + ls.double() * want, e)


@pytest.mark.parametrize("bits,capacity,sequences,batches", [
    (16, 1300, 9, [([201, 581], [0, 1]), ([1] * 9, [2, 1, 0, -1, 0, 1, 2, 0, 1]), ([1300], [1]), ([0, 300, 0, 17, 1], [0, 0, 1, 2, -1])]),
    (4, 1300, 9, [([201, 581], [0, 1]), ([5], [-1]), ([1300], [1])]),
    (4, 24, 24, [([1] * 24, [0] * 24), ([1] * 3, [1, -1, 2]), ([7, 0, 9], [0, 1, 2])]),
])
def test_graph_replayed_for_other_batches(eng, bits, capacity, sequences, batches):
    b, eager = (Block(eng, torch.bfloat16, capacity, sequences, 21, bits) for _ in range(2))
    b.fill([3], [0], 1)
    b.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(torch.cuda.current_stream().cuda_stream)
    for turn, (lengths, ids) in enumerate(batches * 3):
        for x in (b, eager):
            x.fill(lengths, ids, turn)
            for t in (x.act, x.out, x.attention.out, x.attention.qkv, x.attention.mixed):
                t.fill_(3.0)
        eager.run()
        junk = torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.x, eager.x) and torch.equal(b.h, eager.h) and torch.equal(b.act, eager.act), lengths
        n = sum(lengths)
        assert (b.act[n:] == 3.0).all() and (b.out[n:] == 3.0).all()
        del junk


def test_graphs_and_streams_side_by_side(eng):
    # Each with buffers and workspaces of its own, in flight at the same time.
    blocks = [Block(eng, torch.float16, 2400, 4, 31 + i, bits) for i, bits in enumerate((16, 4, 4))]
    start, want = [], []
    for i, b in enumerate(blocks):
        b.fill([[201, 1029, 6, 900], [1, 2000, 77, 301], [2, 3, 0, 1]][i], [0, 1, -1, 2], 40 + i)
        start.append(b.x.clone())
        b.run()
        torch.cuda.synchronize()
        want.append(b.x.clone())
    streams, graphs = [torch.cuda.Stream() for _ in blocks], []
    for b in blocks:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for turn in range(4):
        for b, x in zip(blocks, start):
            b.x.copy_(x)
        torch.cuda.synchronize()
        for b, s, g in zip(blocks, streams, graphs):
            with torch.cuda.stream(s):
                if turn % 2:
                    g.replay()
                else:
                    b.run(s.cuda_stream)
        torch.cuda.synchronize()
        for b, w in zip(blocks, want):
            n = int(b.starts[-1])
            assert torch.equal(b.x[:n], w[:n]), turn


def test_on_engine_regions_and_the_engines_stream(eng):
    rng = np.random.default_rng(3)
    x, y = (rng.normal(size=(50, 64)).astype(np.float16) for _ in range(2))
    regions = [eng.weight(a) for a in (x, y)]
    out, h = eng.allocate(x.nbytes), eng.allocate(x.nbytes)
    call = packed.Norm(type=packed.F16, stream_type=packed.F16, post=packed.NONE, pre=packed.RMS, rows=50, channels=64, pre_eps=1e-6,
                       x=eng.address(regions[0]), y=eng.address(regions[1]), x_out=eng.address(out), h=eng.address(h), x_stride=64,
                       y_stride=64, x_out_stride=64, h_stride=64)
    eng.packed_norm(call, eng.stream)
    eng.reserve_readback(x.nbytes)
    new, got = eng.read(out, np.float16, x.shape).astype(np.float64), eng.read(h, np.float16, x.shape).astype(np.float64)
    want = x.astype(np.float64) + y.astype(np.float64)
    assert (np.abs(new - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -25).all()
    normed = want / np.sqrt((want * want).mean(1, keepdims=True) + 1e-6)
    assert (np.abs(got - normed) <= 2.0 ** -11 * np.abs(normed) * 1.1 + 2.0 ** -25).all()


# --- routes ------------------------------------------------------------------

# One call on each tile (256 x 256, 128 x 128 in two and four stages, 128 x 64 in two
# and four, 64 x 64 in two and four) and on each form of the few-rows kernel (steps of
# 4, 8 and 16 blocks, more steps than waves, more outputs than workgroups take at
# once, several blocks of rows).
GATED = [(2300, 200, 2304), (300, 776, 5000), (3000, 136, 1504), (200, 776, 4000), (1000, 136, 1200), (50, 800, 264), (300, 136, 1000), (100, 800, 1000)]
FEW_GATED = [(16, 2056, 8200), (100, 1032, 520), (130, 1032, 520), (70, 1504, 1000), (40, 8200, 200), (3, 136, 1000), (1, 16, 8), (20, 1504, 8),
             (20, 1032, 8200), (100, 2056, 2000), (300, 800, 1000), (5, 136, 9000)]
GATED4 = [(2300, 1000, 2304), (3000, 136, 1504), (200, 2888, 4000), (1000, 136, 1200), (50, 2888, 264), (600, 136, 1000), (100, 2888, 1000)]
LINEAR4 = [(3400, 1000, 3304), (3000, 136, 2600), (300, 2888, 4104), (2000, 136, 2000), (50, 2888, 520), (700, 136, 1400), (100, 2888, 2000)]
FEW = [(3, 1000, 9000), (5, 8200, 304), (20, 1504, 504), (30, 2400, 104), (100, 304, 200), (24, 1000, 1000), (1, 16, 8),
       (100, 1000, 1000), (150, 1504, 1000), (100, 304, 2000), (100, 5000, 200), (40, 2400, 1000)]
CASES = [("gated", *c) for c in GATED + FEW_GATED] + [("gated4", *c) for c in GATED4 + FEW] + [("linear4", *c) for c in LINEAR4 + FEW]


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("kind,rows,inputs,outputs", CASES)
def test_routes(eng, t, kind, rows, inputs, outputs):
    dt = {"f16": torch.float16, "bf16": torch.bfloat16}[t]
    g = gen(rows + inputs)
    x = normal(g, dt, rows, inputs)
    bias = torch.randn(2, outputs, generator=g, device="cuda")
    out = torch.full((rows, outputs + 8), 7.0, device="cuda").to(dt)
    given = x.double()
    if kind != "gated":
        (gate, gs, gw), (up, us, uw) = (weights4(eng, g, outputs, inputs, dt) for _ in range(2))
        given = values(*(v.cuda() for v in quantised_want(x)), inputs)
    if kind == "linear4":
        run_linear4(eng, x, gate, gs, bias[0], out)
        want, e = product_want(given, gw, bias[0])
    elif kind == "gated4":
        run_gated(eng, x, gate, up, bias[0], bias[1], out, "gelu_tanh", (gs, us))
        want, e = gated_want("gelu_tanh", given, gw, uw, bias[0], bias[1])
    else:
        gate, up = (normal(g, dt, outputs, inputs, scale=inputs ** -0.5) for _ in range(2))
        run_gated(eng, x, gate, up, bias[0], bias[1], out, "silu")
        want, e = gated_want("silu", given, gate.double(), up.double(), bias[0], bias[1])
    torch.cuda.synchronize()
    within(out[:, :outputs], want, e, dt)
    assert (out[:, outputs:] == 7.0).all()


def test_the_same_call_gives_the_same_bits(eng):
    g = gen(2)
    for rows, inputs, outputs in ((24, 2048, 1000), (700, 1000, 1000), (2300, 520, 2304)):
        x = normal(g, torch.bfloat16, rows, inputs)
        (gate, gs, _), (up, us, _) = (weights4(eng, g, outputs, inputs, torch.bfloat16) for _ in range(2))
        outs = [torch.empty(rows, outputs, dtype=torch.bfloat16, device="cuda") for _ in range(6)]
        for out in outs:
            run_gated(eng, x, gate, up, None, None, out, "silu", (gs, us))
        torch.cuda.synchronize()
        assert all(torch.equal(out, outs[0]) for out in outs)


# --- far strides, many rows, starts of any kind --------------------------------

def test_rows_far_apart(eng):
    # Rows 8 MiB apart: offsets pass 32 bits.
    stride, rows = 1 << 22, 1100
    g = gen(5)
    far = torch.empty(rows * stride, dtype=torch.float16, device="cuda").view(rows, stride)
    x, y, new, h, act, out = (far[:, i * 512:i * 512 + 136] for i in range(6))
    x.copy_(normal(g, torch.float16, rows, 136))
    y.copy_(normal(g, torch.float16, rows, 136))
    run_norm(eng, x, y, new, h, "rms", "layer")
    torch.cuda.synchronize()
    (want, e), (want_h, eh) = step_want(x, y, "rms", "layer", {}, None)
    within(new, want, e, torch.float16)
    within(h, want_h, eh, torch.float16)
    weights = far[:136, 8192:8192 + 136]
    weights.copy_(normal(g, torch.float16, 136, 136, scale=0.1))
    gate, up = weights, normal(g, torch.float16, 136, stride, scale=0.1)[:, :136]
    for n in (20, rows):
        run_gated(eng, x[:n], gate, up, None, None, act[:n], "silu")
        torch.cuda.synchronize()
        want, e = gated_want("silu", x[:n].double(), gate.double(), up.double(), None, None)
        within(act[:n], want, e, torch.float16)
    raw = far.view(torch.uint8)
    codes, scales = raw[:, 40000:40000 + 80], raw[:, 50000:50000 + 16]
    back = far[:, 30000:30000 + 136]
    eng.packed_quantise(quantisation(x, codes, scales))
    eng.packed_dequantise(quantisation(back, codes, scales))
    torch.cuda.synchronize()
    want_codes, want_scales = quantised_want(x)
    assert torch.equal(codes.cpu(), want_codes) and torch.equal(scales.cpu(), want_scales)
    assert torch.equal(back.double().cpu(), values(want_codes, want_scales, 136))
    for n in (20, rows):
        run_linear4(eng, x[:n], codes[:136], scales[:136], None, out[:n])
        torch.cuda.synchronize()
        want, e = product_want(values(want_codes, want_scales, 136)[:n].cuda(), values(want_codes, want_scales, 136)[:136].cuda(), None)
        within(out[:n], want, e, torch.float16)


def test_float32_rows_far_apart(eng):
    stride, rows = 1 << 22, 600
    g = gen(6)
    far = torch.empty(rows * stride, dtype=torch.float32, device="cuda").view(rows, stride)
    x, new = far[:, :72], far[:, 1024:1024 + 72]
    x.copy_(torch.randn(rows, 72, generator=g, device="cuda"))
    y = normal(g, torch.bfloat16, rows, 72)
    h = torch.empty_like(y)
    run_norm(eng, x, y, new, h, "layer", "rms")
    torch.cuda.synchronize()
    (want, e), (want_h, eh) = step_want(x, y, "layer", "rms", {}, None)
    within(new, want, e, torch.float32)
    within(h, want_h, eh, torch.bfloat16)


def test_more_rows_than_workgroups(eng):
    # More than 2^21 workgroups of one row each: workgroups take a second row.
    rows, channels = (1 << 21) + 700, 520
    x = torch.zeros(rows, channels, dtype=torch.float16, device="cuda")
    y = torch.zeros_like(x)
    some = torch.cat([torch.arange(64, device="cuda"), torch.arange(rows - 764, rows, device="cuda")])
    x[some], y[some] = (normal(gen(9 + i), torch.float16, some.numel(), channels) for i in range(2))
    want, h = torch.empty(some.numel(), channels, dtype=torch.float16, device="cuda"), torch.empty(some.numel(), channels, dtype=torch.float16, device="cuda")
    run_norm(eng, x[some], y[some], want, h, "rms", "layer")
    run_norm(eng, x, y, x, y, "rms", "layer")
    torch.cuda.synchronize()
    assert torch.equal(x[some], want) and torch.equal(y[some], h) and not x[64:4096].any() and not y[64:4096].any()
    del x, y
    for rows, columns in (((1 << 21) + 300, 2056), ((1 << 23) + 300, 8)):
        x = torch.zeros(rows, columns, dtype=torch.bfloat16, device="cuda")
        some = torch.cat([torch.arange(64, device="cuda"), torch.arange(rows - 764, rows, device="cuda")])
        x[some] = normal(gen(11), torch.bfloat16, some.numel(), columns)
        codes, scales = quantised(eng, x)
        back = torch.full_like(x, 7.0)
        eng.packed_dequantise(quantisation(back, codes, scales))
        few_codes, few_scales = quantised(eng, x[some])
        torch.cuda.synchronize()
        assert torch.equal(codes[some], few_codes) and torch.equal(scales[some], few_scales)
        assert torch.equal(back[some].double(), values(few_codes, few_scales, columns)) and not back[64:4096].any()
        del x, codes, scales, back


@pytest.mark.parametrize("starts", [[0, -7, 30, 2 ** 31 - 1], [60, 20, 5, 0], [10, 10, 10, 10], [-5, -4, -3, -1], [50, 2 ** 30, 0, 64]])
def test_starts_of_any_kind_stay_inside(eng, starts):
    # Starts that decrease or lie outside: nothing outside the rows is touched.
    g = gen(2)
    for rows in (24, 64, 300):
        x, y = (normal(g, torch.float16, rows, 256) for _ in range(2))
        gate = torch.randn(3, 256, generator=g, device="cuda")
        w, w2 = (normal(g, torch.float16, 256, 256, scale=0.1) for _ in range(2))
        codes, scales = quantised(eng, w)
        guards = [torch.full((rows + 200, 256), 7.0, device="cuda").half() for _ in range(5)]
        mine = [t[100:100 + rows] for t in guards]
        bytes_ = [torch.full((rows + 200, n), 0xee, dtype=torch.uint8, device="cuda") for n in (128, 16)]
        run_norm(eng, x, y, mine[0], mine[1], "rms", "layer", gate=gate, starts=ints(starts))
        run_norm(eng, x, y, mine[0], mine[1], "rms", "layer", starts=ints(starts))
        run_gated(eng, x, w, w2, None, None, mine[2], "silu", starts=ints(starts))
        run_gated(eng, x, codes, codes, None, None, mine[3], "silu", (scales, scales), starts=ints(starts))
        run_linear4(eng, x, codes, scales, None, mine[4], starts=ints(starts))
        eng.packed_quantise(quantisation(x, *(t[100:100 + rows] for t in bytes_), ints(starts)))
        torch.cuda.synchronize()
        for t in guards:
            assert (t[:100] == 7.0).all() and (t[100 + rows:] == 7.0).all()
        for t in bytes_:
            assert (t[:100] == 0xee).all() and (t[100 + rows:] == 0xee).all()


def test_refusals_change_nothing_and_failures_poison(gpu):
    e = d.Engine(0)
    x = torch.ones(4, 64, device="cuda").half()
    out = torch.full_like(x, 7.0)
    run = lambda pre: run_norm(e, x, None, None, out, "none", pre)  # noqa: E731
    with pytest.raises(d.DINOv3Error, match="pre is needed"):
        e.packed_norm(packed.Norm(type=packed.F16, rows=4, channels=64, x=at(x), x_stride=64))
    for rows, outputs in ((64, 64), (400, 1000)):
        many, y = torch.ones(rows, 2056, device="cuda").half(), torch.full((rows, outputs), 7.0, device="cuda").half()
        codes, scales = quantised(e, torch.ones(outputs, 2056, device="cuda").half())
        call = packed.QuantisedLinear(type=packed.F16, rows=rows, inputs=2056, outputs=outputs, x=at(many), w=at(codes), w_scales=at(scales),
                                      y=at(y), x_stride=2056, y_stride=outputs, w_stride=codes.shape[1], scales_stride=scales.shape[1])
        if rows == 64:  # few rows need no workspace, and run without one
            assert e.packed_quantised_linear_workspace(call) == 0
            e.packed_quantised_linear(call)
            torch.cuda.synchronize()
            assert (y == 2056.0).all()
            continue
        assert e.packed_quantised_linear_workspace(call) > 0
        with pytest.raises(d.DINOv3Error, match="the call needs"):
            e.packed_quantised_linear(call)
        torch.cuda.synchronize()
        assert (out == 7.0).all() and (y == 7.0).all()
    run("rms")
    torch.cuda.synchronize()
    assert (out == 1.0).all()
    assert d._lib.dhx_test_fail_next_call(e._h) == 0
    with pytest.raises(d.DINOv3Error):
        run("rms")
    with pytest.raises(d.DINOv3Error, match="session is unusable after a GPU failure"):
        run("rms")
    e.close()
