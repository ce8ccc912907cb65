"""The operators on packed batches as they are used: a run of them together on
images of different sizes, each with its own request's adapter, checked stage by
stage against float64; the same against the engine's own kernels on a 224x224
image; captured into a graph and replayed for other inputs and other lengths;
on streams side by side; on engine regions; far strides; failures."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import dinov3_hrx as d  # noqa: E402
from dinov3_hrx import packed  # noqa: E402

from test_kernels_gpu import K_ATTN, K_QKV, _keys  # noqa: E402
from packed_operators import (F, attention_want, gen, half_step, ints, linear_want, normal, run_attention, run_linear,  # noqa: E402
                             run_rotation, starts_of, within)

pytestmark = pytest.mark.gpu
HEADS, DIM, HIDDEN, PREFIX = 6, 64, 384, 5


@pytest.fixture(scope="module")
def eng(gpu):
    e = d.Engine(0)
    yield e
    e.close()


class Block:
    """Projection to q, k, v, rotation of q and k in place, attention, output
    projection; every buffer and workspace of `rows` rows and `sequences`."""

    def __init__(self, dt, rows, sequences, seed, adapters=3, rank=16):
        g = gen(seed)
        s = HIDDEN ** -0.5
        self.dt, self.rows = dt, rows
        self.wq, self.bq = normal(g, dt, 3 * HIDDEN, HIDDEN, scale=s), torch.randn(3 * HIDDEN, generator=g, device="cuda") * 0.1
        self.wo, self.bo = normal(g, dt, HIDDEN, HIDDEN, scale=s), torch.randn(HIDDEN, generator=g, device="cuda") * 0.1
        self.aq, self.ao = (normal(g, dt, adapters, rank, HIDDEN, scale=s) for _ in range(2))
        self.dq, self.do = normal(g, dt, adapters, 3 * HIDDEN, rank, scale=0.25), normal(g, dt, adapters, HIDDEN, rank, scale=0.25)
        self.scale = torch.rand(adapters, generator=g, device="cuda") + 0.5
        places = 1100
        angle = torch.rand(places, DIM // 2, generator=g, device="cuda") * 6.28
        self.cos, self.sin = angle.cos(), angle.sin()
        self.x = normal(g, dt, rows, HIDDEN)
        self.starts, self.ids = ints([0] * (sequences + 1)), ints([-1] * sequences)
        self.index = ints([-1] * rows)
        self.qkv = torch.empty(rows, 3 * HIDDEN, dtype=dt, device="cuda")
        self.mixed, self.out = (torch.empty(rows, HIDDEN, dtype=dt, device="cuda") for _ in range(2))
        self.ws = [torch.empty(1 << 22, dtype=torch.uint8, device="cuda") for _ in range(3)]

    def fill(self, lengths, ids, seed):
        """Another batch in the same buffers; rows behind it keep what they have."""
        g = gen(seed)
        st = starts_of(lengths)
        self.x.copy_(normal(g, self.dt, self.rows, HIDDEN))
        n = self.starts.numel() - 1
        self.starts.copy_(ints(st + [st[-1]] * (n + 1 - len(st))))
        self.ids.copy_(ints(ids + [-1] * (n - len(ids))))
        index = [i - PREFIX if i >= PREFIX else -1 for m in lengths for i in range(m)]
        self.index.copy_(ints(index + [-1] * (self.rows - len(index))))
        return st

    def heads(self):
        return [t.unflatten(1, (HEADS, DIM)) for t in self.qkv.split(HIDDEN, 1)]

    def run(self, e, stream=0, hints=None):
        run_linear(e, self.x, self.wq, self.bq, self.aq, self.dq, self.scale, self.qkv, self.starts, self.ids, stream=stream,
                   workspace=self.ws[0])
        run_rotation(e, self.qkv, self.qkv, self.index, self.cos, self.sin, 2 * HEADS, DIM, DIM, 0, stream)
        q, k, v = self.heads()
        run_attention(e, q, k, v, self.mixed.unflatten(1, (HEADS, DIM)), self.starts, self.starts, 0, DIM ** -0.5, hints=hints,
                      stream=stream, workspace=self.ws[1])
        run_linear(e, self.mixed, self.wo, self.bo, self.ao, self.do, self.scale, self.out, self.starts, self.ids, stream=stream,
                   workspace=self.ws[2])


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_block_stage_by_stage(eng, dt):
    lengths, ids = [201, 6, 581, 1, 0, 101, 1029], [0, -1, 2, 1, 0, 1, 0]
    b = Block(dt, sum(lengths) + 40, len(lengths), 3)
    st = b.fill(lengths, ids, 4)
    n, spans = st[-1], [(st[s], st[s + 1], i) for s, i in enumerate(ids)]
    b.out.fill_(7.0)
    # The stages one by one, each on what the one before left.
    run_linear(eng, b.x, b.wq, b.bq, b.aq, b.dq, b.scale, b.qkv, b.starts, b.ids)
    torch.cuda.synchronize()
    want, bound = linear_want(b.x[:n], b.wq, b.bq, b.aq, b.dq, b.scale, spans)
    within(b.qkv[:n], want, bound, dt)
    before = b.qkv[:n].clone()
    run_rotation(eng, b.qkv, b.qkv, b.index, b.cos, b.sin, 2 * HEADS, DIM, DIM, 0)
    torch.cuda.synchronize()
    assert torch.equal(b.qkv[:n, 2 * HIDDEN:], before[:, 2 * HIDDEN:])
    qk, at = before[:, :2 * HIDDEN].double().view(n, 2 * HEADS, 2, DIM // 2), b.index[:n].long()
    c = torch.where(at[:, None] >= 0, b.cos.double()[at.clamp_min(0)], 1.0)[:, None]
    s = torch.where(at[:, None] >= 0, b.sin.double()[at.clamp_min(0)], 0.0)[:, None]
    x1, x2 = qk[:, :, 0], qk[:, :, 1]
    want = torch.stack([x1 * c - x2 * s, x2 * c + x1 * s], 2)
    bound = 3 * F * torch.stack([(x1 * c).abs() + (x2 * s).abs(), (x2 * c).abs() + (x1 * s).abs()], 2)
    within(b.qkv[:n, :2 * HIDDEN].reshape(n, 2 * HEADS, 2, DIM // 2), want, bound, dt)
    q, k, v = b.heads()
    mixed = b.mixed.unflatten(1, (HEADS, DIM))
    run_attention(eng, q, k, v, mixed, b.starts, b.starts, 0, DIM ** -0.5)
    torch.cuda.synchronize()
    for lo, hi, _ in spans:
        want, room, _, _ = attention_want(q[lo:hi], k[lo:hi], v[lo:hi], 0, DIM ** -0.5)
        within(mixed[lo:hi], want, room, dt)
    run_linear(eng, b.mixed, b.wo, b.bo, b.ao, b.do, b.scale, b.out, b.starts, b.ids)
    torch.cuda.synchronize()
    want, bound = linear_want(b.mixed[:n], b.wo, b.bo, b.ao, b.do, b.scale, spans)
    within(b.out[:n], want, bound, dt)
    assert (b.out[n:] == 7.0).all()
    # And all of them queued at once.
    alone = b.out.clone()
    b.out.fill_(7.0)
    b.run(eng)
    torch.cuda.synchronize()
    assert torch.equal(b.out, alone)


def test_against_the_engines_own_kernels(eng):
    # Two 224x224 images: QKV + RoPE and attention in the engine's fragment
    # layout, and the packed run of projection, rotation and attention. q, k and
    # v are rounded once there and twice here (q and k), so a score differs by at
    # most (u + 2u)(1 + u) sum|q k| on either side's rounding, v by 2u.
    images, grid, tpad, T = 2, 14, 256, 201
    g = gen(11)
    h = normal(g, torch.float16, images * T, HIDDEN)
    w = normal(g, torch.float16, 3 * HIDDEN, HIDDEN, scale=HIDDEN ** -0.5)
    bias = torch.randn(3 * HIDDEN, generator=g, device="cuda") * 0.1
    angle = torch.rand(grid * grid, 32, generator=g, device="cuda") * 6.28
    # The engine's tables are separable; the rows of a grid row share the first
    # 16 angles, those of a column the others.
    angle = angle.view(grid, grid, 32)
    angle = torch.cat([angle[:, :1, :16].expand(grid, grid, 16), angle[:1, :, 16:].expand(grid, grid, 16)], 2).reshape(-1, 32)
    cos, sin = angle.cos().contiguous(), angle.sin().contiguous()
    up = lambda a: eng.weight(np.ascontiguousarray(a))  # noqa: E731
    regions = [up(d.fragment_order(h.cpu().numpy())), up(d.fragment_order(w.cpu().numpy())), up(bias.cpu().numpy())]
    regions += [up(torch.cat([t, t], 1).cpu().numpy()) for t in (cos, sin)]
    qkv = [eng.allocate(images * HEADS * tpad * DIM * 2) for _ in range(3)]
    rows = (images * T + 31) // 32 * 32
    out = eng.allocate(rows * HIDDEN * 2)
    key = next(_keys)
    eng.record(key, [(K_QKV, [images, grid, tpad], regions + qkv), (K_ATTN, [images, grid, tpad], qkv + [out])])
    eng.replay(key)
    eng.synchronize()
    eng.reserve_readback(rows * HIDDEN * 2)
    own = torch.from_numpy(d.row_order(eng.read(out, np.float16, (rows * HIDDEN,)), images * T, HIDDEN)).cuda()

    packed_qkv = torch.empty(images * T, 3 * HIDDEN, dtype=torch.float16, device="cuda")
    none = torch.zeros(1, 8, HIDDEN, device="cuda").half(), torch.zeros(1, 3 * HIDDEN, 8, device="cuda").half()
    st = ints([0, T, 2 * T])
    run_linear(eng, h, w, bias, *none, torch.ones(1, device="cuda"), packed_qkv, st, ints([-1, -1]))
    index = ints([p - PREFIX if p >= PREFIX else -1 for _ in range(images) for p in range(T)])
    run_rotation(eng, packed_qkv, packed_qkv, index, cos, sin, 2 * HEADS, DIM, DIM, 0)
    mixed = torch.empty(images * T, HEADS, DIM, dtype=torch.float16, device="cuda")
    q, k, v = (t.unflatten(1, (HEADS, DIM)) for t in packed_qkv.split(HIDDEN, 1))
    run_attention(eng, q, k, v, mixed, st, st, 0, DIM ** -0.5)
    torch.cuda.synchronize()
    u = half_step(torch.float16)
    for i in range(images):
        rows_of = slice(i * T, (i + 1) * T)
        _, room, _, _ = attention_want(q[rows_of], k[rows_of], v[rows_of], 0, DIM ** -0.5)
        for head in range(HEADS):
            size = DIM ** -0.5 * (q[rows_of, head].double().abs() @ k[rows_of, head].double().abs().t().contiguous())
            weight = torch.softmax(DIM ** -0.5 * q[rows_of, head].double() @ k[rows_of, head].double().t().contiguous(), 1)
            off = 2 * torch.expm1(2 * 3.1 * u * size.amax(1, keepdim=True)) + 2 * 3.1 * u
            near = 2 * room[:, head] + off * (weight @ v[rows_of, head].double().abs()) + 2 * u * mixed[rows_of, head].double().abs()
            mine, theirs = mixed[rows_of, head].double(), own[rows_of, head * DIM:(head + 1) * DIM].double()
            assert ((mine - theirs).abs() <= near).all()


def test_graph_replayed_for_other_batches(eng):
    # One capture for up to 9 sequences and 1300 rows, replayed for batches of
    # other lengths and contents, with eager calls and other work in between.
    b, eager = (Block(torch.bfloat16, 1300, 9, 21) for _ in range(2))
    b.fill([201], [0], 1)
    hints = (0, 0)
    b.run(eng, hints=hints)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(eng, torch.cuda.current_stream().cuda_stream, hints)
    batches = [([201, 581], [0, 1]), ([1] * 9, [2, 1, 0, -1, 0, 1, 2, 0, 1]), ([1300], [1]), ([0, 300, 0, 17, 1], [0, 0, 1, 2, -1]), ([5], [-1])]
    for turn, (lengths, ids) in enumerate(batches * 2):
        for x in (b, eager):
            x.fill(lengths, ids, turn)
            x.out.fill_(3.0)
            x.qkv.fill_(3.0)
            x.mixed.fill_(3.0)
        eager.run(eng, hints=hints)
        junk = torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.out, eager.out) and torch.equal(b.mixed, eager.mixed), lengths
        n = sum(lengths)
        assert (b.out[n:] == 3.0).all() and (b.qkv[n:] == 3.0).all()
        del junk


def test_two_graphs_and_streams_side_by_side(eng):
    # Each with buffers and workspaces of its own, in flight at the same time.
    blocks = [Block(torch.float16, 2400, 4, s) for s in (31, 32)]
    want = []
    for i, b in enumerate(blocks):
        b.fill([[201, 1029, 6, 900], [1, 2000, 77, 301]][i], [0, 1, -1, 2], 40 + i)
        b.out.fill_(0.0)  # rows behind the last sequence stay so
        b.run(eng)
        torch.cuda.synchronize()
        want.append(b.out.clone())
    streams, graphs = [torch.cuda.Stream() for _ in blocks], []
    for b in blocks:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.run(eng, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for turn in range(4):
        for b in blocks:
            b.out.fill_(0.0)
        torch.cuda.synchronize()
        for b, s, g in zip(blocks, streams, graphs):
            with torch.cuda.stream(s):
                if turn % 2:
                    g.replay()
                else:
                    b.run(eng, s.cuda_stream)
        torch.cuda.synchronize()
        for b, w in zip(blocks, want):
            assert torch.equal(b.out, w), turn


def test_on_engine_regions_and_the_engines_stream(eng):
    # A program without device memory of its own: regions, their addresses and
    # the engine's stream.
    rng = np.random.default_rng(3)
    rows, heads, dim = 50, 3, 64
    x = rng.normal(size=(rows, heads * dim)).astype(np.float16)
    angle = rng.random((rows, dim // 2)) * 6.28
    r = [eng.weight(a) for a in (x, np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32),
                                 np.arange(rows, dtype=np.int32))]
    out = eng.allocate(x.nbytes)
    call = packed.Rotation(type=packed.F16, rows=rows, heads=heads, head_dim=dim, rotated=dim, places=rows, x=eng.address(r[0]),
                           out=eng.address(out), x_stride=heads * dim, out_stride=heads * dim, cos=eng.address(r[1]),
                           sin=eng.address(r[2]), index=eng.address(r[3]))
    assert eng.stream != 0
    eng.packed_rotate(call, eng.stream)
    eng.reserve_readback(x.nbytes)
    got = eng.read(out, np.float16, (rows, heads, dim)).astype(np.float64)
    v = x.astype(np.float64).reshape(rows, heads, 2, dim // 2)
    c, s = np.cos(angle).astype(np.float32).astype(np.float64)[:, None], np.sin(angle).astype(np.float32).astype(np.float64)[:, None]
    want = np.stack([v[:, :, 0] * c - v[:, :, 1] * s, v[:, :, 1] * c + v[:, :, 0] * s], 2).reshape(rows, heads, dim)
    assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * np.abs(x).max() + 2.0 ** -25).all()
    with pytest.raises(d.DINOv3Error, match="unknown buffer"):
        eng.address(d.Region(10 ** 6, 0, 4))


def test_rows_far_apart(eng):
    # Rows 8 MiB apart: offsets pass 32 bits (in bytes behind 512 rows, in
    # elements behind 1024).
    stride, lk, heads, dim = 1 << 22, 1100, 2, 64
    g = gen(5)
    far = torch.empty(lk * stride, dtype=torch.float16, device="cuda").view(lk, stride)
    k, v = (far[:, i * heads * dim:(i + 1) * heads * dim].unflatten(1, (heads, dim)) for i in range(2))
    k.copy_(normal(g, torch.float16, lk, heads, dim))
    v.copy_(normal(g, torch.float16, lk, heads, dim))
    for lq in (1, 1100):
        q = normal(g, torch.float16, lq, heads, dim)
        out = torch.empty_like(q)
        run_attention(eng, q, k, v, out, ints([0, lq]), ints([0, lk]), 1, dim ** -0.5, hints=(lq, lk))
        torch.cuda.synchronize()
        want, room, _, _ = attention_want(q, k, v, 1, dim ** -0.5)
        within(out, want, room, torch.float16)
    x, y = far[:, 512:512 + 128], far[:, 1024:1024 + 64]
    x.copy_(normal(g, torch.float16, lk, 128))
    w, a, b = normal(g, torch.float16, 64, 128), normal(g, torch.float16, 1, 8, 128), normal(g, torch.float16, 1, 64, 8)
    for rows in (40, lk):
        run_linear(eng, x[:rows], w, None, a, b, torch.ones(1, device="cuda"), y, ints([0, rows]), ints([0]))
        torch.cuda.synchronize()
        want, bound = linear_want(x[:rows], w, None, a, b, torch.ones(1, device="cuda"), [(0, rows, 0)])
        within(y[:rows], want, bound, torch.float16)
    turned = far[:, 2048:2048 + 128]
    angle = torch.rand(lk, 32, generator=g, device="cuda")
    run_rotation(eng, k.flatten(1), turned, ints(range(lk)), angle.cos(), angle.sin(), heads, dim, dim, 0)
    torch.cuda.synchronize()
    near = torch.empty(lk, 128, dtype=torch.float16, device="cuda")
    run_rotation(eng, k.flatten(1).contiguous(), near, ints(range(lk)), angle.cos(), angle.sin(), heads, dim, dim, 0)
    torch.cuda.synchronize()
    assert torch.equal(turned, near)


@pytest.mark.parametrize("starts", [[0, -7, 30, 2 ** 31 - 1], [60, 20, 5, 0], [10, 10, 10, 10], [-5, -4, -3, -1], [50, 2 ** 30, 0, 64]])
def test_starts_of_any_kind_stay_inside(eng, starts):
    # Starts that decrease or lie outside: nothing outside the rows is touched.
    g = gen(2)
    rows, heads, dim = 64, 4, 64
    q, k, v = (normal(g, torch.float16, rows, heads, dim) for _ in range(3))
    guard = torch.full((rows + 200, heads, dim), 7.0, device="cuda").half()
    lse = torch.full((rows + 200, heads), 7.0, device="cuda")
    for hints in ((64, 64), (1, 4000), (0, 0)):
        run_attention(eng, q, k, v, guard[100:100 + rows], ints(starts), ints(starts[::-1]), 1, dim ** -0.5,
                      lse=lse[100:100 + rows], hints=hints)
    w, a, b = normal(g, torch.float16, 256, 256), normal(g, torch.float16, 2, 8, 256), normal(g, torch.float16, 2, 256, 8)
    y = torch.full((rows + 200, 256), 7.0, device="cuda").half()
    run_linear(eng, q.flatten(1), w, None, a, b, torch.ones(2, device="cuda"), y[100:100 + rows], ints(starts), ints([0, 1, 9]))
    torch.cuda.synchronize()
    for t in (guard, lse, y):
        assert (t[:100] == 7.0).all() and (t[100 + rows:] == 7.0).all()


def test_refusals_change_nothing_and_failures_poison(gpu):
    e = d.Engine(0)
    x = torch.ones(4, 64, device="cuda").half()
    out = torch.full_like(x, 7.0)
    table, index = torch.ones(4, 32, device="cuda"), ints([0, 1, 2, 3])
    run = lambda rotated: run_rotation(e, x, out, index, table, table, 1, 64, rotated, 0)  # noqa: E731
    with pytest.raises(d.DINOv3Error, match="rotated must be"):
        run(24)
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    run(64)
    torch.cuda.synchronize()
    assert (out[:, :32] == 0.0).all() and (out[:, 32:] == 2.0).all()
    assert d._lib.dhx_test_fail_next_call(e._h) == 0
    with pytest.raises(d.DINOv3Error):
        run(64)
    with pytest.raises(d.DINOv3Error, match="session is unusable after a GPU failure"):
        run(64)
    e.close()
