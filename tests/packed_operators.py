"""The operators on packed batches against their definitions in float64 (on
the GPU, by PyTorch), where they can go wrong: lengths of 0 and 1, ragged and
odd sizes, rows of no sequence, masks that leave a row empty, strides,
values that are not finite outside a sequence, streams and graphs.

Tolerances are bounds from the arithmetic. u is half a step of the type
(finfo.eps / 2), f = 2^-24 that of float32. A sum of n float32 products of
exact factors is off by at most (n + 1) f times the sum of their absolute
values, whatever its order; an output is rounded once, by u of itself (and at
most half the type's smallest number where it is subnormal)."""
import math

import pytest

torch = pytest.importorskip("torch")

import dinov3_hrx as d  # noqa: E402
from dinov3_hrx import packed  # noqa: E402

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
TYPES = {"f16": (packed.F16, torch.float16), "bf16": (packed.BF16, torch.bfloat16)}


@pytest.fixture(scope="module")
def eng(gpu):
    e = d.Engine(0)
    yield e
    e.close()


def half_step(t):
    return torch.finfo(t).eps / 2


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(lengths, first=0):
    out = [first]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def normal(g, t, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, bound, t):
    """got equals want to bound plus one rounding to t."""
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    room = bound + half_step(t) * want.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    worst = (off - room).max().item() if off.numel() else -1.0
    assert not math.isnan(worst) and worst <= 0, f"off by {off.max().item():.3g}, {worst:.3g} past the bound"


# --- rotation ----------------------------------------------------------------

def run_rotation(e, x, out, index, cos, sin, heads, dim, rotated, neighbours, stream=0):
    kind = packed.F16 if x.dtype == torch.float16 else packed.BF16
    e.packed_rotate(packed.Rotation(
        type=kind, neighbours=neighbours, rows=x.shape[0], heads=heads, head_dim=dim, rotated=rotated, places=cos.shape[0],
        x=x.data_ptr(), out=out.data_ptr(), x_stride=x.stride(0), out_stride=out.stride(0), cos=cos.data_ptr(),
        sin=sin.data_ptr(), index=index.data_ptr()), stream)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("neighbours", [0, 1])
@pytest.mark.parametrize("rows,heads,dim,rotated,extra", [(1, 1, 16, 16, 0), (201, 12, 64, 64, 384), (37, 3, 80, 80, 8),
                                                          (130, 5, 128, 64, 0), (64, 40, 96, 32, 96), (3, 200, 64, 64, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rotation(eng, t, neighbours, rows, heads, dim, rotated, extra, in_place):
    dt = TYPES[t][1]
    g = gen(rows + dim)
    x = normal(g, dt, rows, heads * dim + extra)
    places = 50
    angle = torch.rand(places, rotated // 2, generator=g, device="cuda") * 6.28
    cos, sin = angle.cos(), angle.sin()
    index = torch.randint(-2, places + 2, (rows,), generator=g, device="cuda", dtype=torch.int32)
    before = x.clone()
    out = x if in_place else torch.full((rows, heads * dim + 16), 7.0, device="cuda").to(dt)
    run_rotation(eng, x, out, index, cos, sin, heads, dim, rotated, neighbours)
    torch.cuda.synchronize()
    v = before[:, :heads * dim].double().view(rows, heads, dim)
    at = index.long()
    there = (at >= 0) & (at < places)
    c = torch.where(there[:, None], cos.double()[at.clamp(0, places - 1)], 1.0)[:, None]
    s = torch.where(there[:, None], sin.double()[at.clamp(0, places - 1)], 0.0)[:, None]
    want = v.clone()
    one = slice(0, rotated, 2) if neighbours else slice(0, rotated // 2)
    two = slice(1, rotated, 2) if neighbours else slice(rotated // 2, rotated)
    want[..., one] = v[..., one] * c - v[..., two] * s
    want[..., two] = v[..., two] * c + v[..., one] * s
    bound = torch.zeros_like(want)  # two products and a sum
    bound[..., one] = 3 * F * ((v[..., one] * c).abs() + (v[..., two] * s).abs())
    bound[..., two] = 3 * F * ((v[..., two] * c).abs() + (v[..., one] * s).abs())
    got = out[:, :heads * dim].reshape(rows, heads, dim)
    within(got, want, bound, dt)
    copied = ~there
    assert torch.equal(got[copied], before[:, :heads * dim].view(rows, heads, dim)[copied])
    assert torch.equal(got[..., rotated:], before[:, :heads * dim].view(rows, heads, dim)[..., rotated:])
    rest = out[:, heads * dim:]
    assert torch.equal(rest, before[:, heads * dim:] if in_place else torch.full_like(rest, 7.0))


def test_rotation_of_more_rows_than_workgroups(eng):
    # More than 2^21 workgroups of one row each: workgroups take a second row.
    rows, heads, dim = (1 << 21) + 700, 129, 16
    x = torch.zeros(rows, heads * dim, dtype=torch.float16, device="cuda")
    some = torch.cat([torch.arange(64, device="cuda"), torch.arange(rows - 764, rows, device="cuda")])
    x[some] = normal(gen(9), torch.float16, some.numel(), heads * dim)
    angle = torch.rand(50, dim // 2, generator=gen(10), device="cuda")
    index = (torch.arange(rows, device="cuda") % 50).int()
    want = torch.empty(some.numel(), heads * dim, dtype=torch.float16, device="cuda")
    run_rotation(eng, x[some], want, index[some], angle.cos(), angle.sin(), heads, dim, dim, 0)
    run_rotation(eng, x, x, index, angle.cos(), angle.sin(), heads, dim, dim, 0)
    torch.cuda.synchronize()
    assert torch.equal(x[some], want) and not x[64:4096].any()


# --- projection with adapters ------------------------------------------------

def run_linear(e, x, w, bias, a, b, scale, y, starts, ids, rows=None, stream=0, workspace=None):
    kind = packed.F16 if x.dtype == torch.float16 else packed.BF16
    call = packed.Linear(
        type=kind, sequences=ids.numel(), rows=x.shape[0] if rows is None else rows, inputs=w.shape[1], outputs=w.shape[0],
        rank=a.shape[1], adapters=a.shape[0], x=x.data_ptr(), w=w.data_ptr(), bias=0 if bias is None else bias.data_ptr(),
        a=a.data_ptr(), b=b.data_ptr(), scale=scale.data_ptr(), y=y.data_ptr(), x_stride=x.stride(0), w_stride=w.stride(0),
        y_stride=y.stride(0), starts=starts.data_ptr(), adapter=ids.data_ptr())
    need = e.packed_linear_workspace(call)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda") if workspace is None else workspace
    call.workspace, call.workspace_bytes = ws.data_ptr(), need
    e.packed_linear(call, stream)
    return ws


def linear_want(x, w, bias, a, b, scale, spans):
    """(want, bound) of the rows in spans (first, last + 1, adapter)."""
    x64, w64 = x.double(), w.double()
    want = x64 @ w64.t().contiguous()
    size = x64.abs() @ w64.abs().t().contiguous()
    k, r = w.shape[1], a.shape[1]
    bound = (k + r + 2) * F * size
    if bias is not None:
        want += bias.double()
        bound += 2 * F * (bias.double().abs() + size)
    u = half_step(x.dtype)
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    for lo, hi, i in spans:
        if i < 0 or lo == hi:
            continue
        s = scale[i].double()
        inner, many = s * (x64[lo:hi] @ a[i].double().t().contiguous()), s.abs() * (x64[lo:hi].abs() @ a[i].double().abs().t().contiguous())
        bt = b[i].double().t().contiguous()
        want[lo:hi] += inner @ bt
        off = (u * inner.abs() + (k + 2) * F * many * (1 + u) + tiny) @ bt.abs()  # u rounded to the type
        bound[lo:hi] += off + (k + r + 2) * F * ((inner.abs() + u * many) @ bt.abs())
    return want, bound


SHAPES = [(64, 64, 8), (384, 1152, 16), (40, 72, 24), (1536, 384, 8), (136, 200, 64), (72, 1000, 256)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lengths", [[1], [5, 0, 17, 1], [1] * 40, [201, 201, 33], [127, 2, 300, 0, 0, 131], [640]])
@pytest.mark.parametrize("inputs,outputs,rank", SHAPES)
def test_linear(eng, t, lengths, inputs, outputs, rank):
    dt = TYPES[t][1]
    g = gen(sum(lengths) + inputs + rank)
    rows, adapters = sum(lengths), 5
    x = normal(g, dt, rows, inputs + 16)[:, :inputs]
    w = normal(g, dt, outputs, inputs + 8, scale=inputs ** -0.5)[:, :inputs]
    a, b = normal(g, dt, adapters, rank, inputs, scale=inputs ** -0.5), normal(g, dt, adapters, outputs, rank, scale=rank ** -0.5)
    scale = torch.rand(adapters, generator=g, device="cuda") * 3 - 1
    bias = torch.randn(outputs, generator=g, device="cuda") if rank != 24 else None
    ids = [(s * 3 + 1) % (adapters + 2) - 1 for s in range(len(lengths))]  # -1 .. adapters: both ends mean none
    st = starts_of(lengths)
    y = torch.full((rows, outputs + 8), 7.0, device="cuda").to(dt)
    run_linear(eng, x, w, bias, a, b, scale, y, ints(st), ints(ids))
    torch.cuda.synchronize()
    spans = [(st[s], st[s + 1], i if i < adapters else -1) for s, i in enumerate(ids)]
    want, bound = linear_want(x, w, bias, a, b, scale, spans)
    within(y[:, :outputs], want, bound, dt)
    assert (y[:, outputs:] == 7.0).all()


# One launch on each route: the few-rows kernel with 1, 2 and 4 row blocks, and
# each tile (256 x 256, 128 x 128, 128 x 64, 64 x 64 in two stages and in four),
# with whole and ragged last tiles and steps, runs that end inside tiles and a
# request per row.
ROUTES = [(16, 264, 640), (32, 264, 640), (50, 264, 640), (3700, 136, 3848), (2500, 584, 1928), (2500, 584, 1304),
          (1500, 520, 1400), (700, 1032, 520), (8300, 72, 264), (8200, 520, 264)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", ["ragged", "single"])
@pytest.mark.parametrize("rows,inputs,outputs", ROUTES)
def test_linear_routes(eng, t, kind, rows, inputs, outputs):
    dt = TYPES[t][1]
    g = gen(rows + outputs)
    if kind == "ragged":
        lengths = [n for i in range(rows) for n in [(37 * i * i + 11) % 300]]
        st = [s for s in starts_of(lengths) if s < rows] + [rows]
    else:
        st = list(range(rows + 1))
    adapters, rank = 7, 24
    x, w = normal(g, dt, rows, inputs), normal(g, dt, outputs, inputs, scale=inputs ** -0.5)
    a, b = normal(g, dt, adapters, rank, inputs, scale=inputs ** -0.5), normal(g, dt, adapters, outputs, rank, scale=rank ** -0.5)
    scale = torch.rand(adapters, generator=g, device="cuda") + 0.5
    bias = torch.randn(outputs, generator=g, device="cuda")
    ids = [(s * 3) % (adapters + 1) - 1 for s in range(len(st) - 1)]
    y = torch.full((rows, outputs), 7.0, device="cuda").to(dt)
    run_linear(eng, x, w, bias, a, b, scale, y, ints(st), ints(ids))
    torch.cuda.synchronize()
    # Rows of one adapter together, so that the 64-bit form takes a few products.
    row_ids = torch.repeat_interleave(torch.tensor(ids), torch.tensor(st).diff()).cuda()
    order = torch.argsort(row_ids, stable=True)
    counts = [int((row_ids == i).sum()) for i in range(-1, adapters)]
    at = starts_of(counts)
    spans = [(at[i], at[i + 1], i - 1) for i in range(adapters + 1)]
    want, bound = linear_want(x[order], w, bias, a, b, scale, spans)
    within(y[order], want, bound, dt)
    again = torch.full_like(y, 3.0)
    run_linear(eng, x, w, bias, a, b, scale, again, ints(st), ints(ids))
    torch.cuda.synchronize()
    assert torch.equal(y, again)  # the same bits from launch to launch


# The few-rows kernel over several blocks of 64 rows (the last one not whole),
# and the first sizes behind it: more rows, more workgroups, fewer columns.
ROUTES_OF_SOME_ROWS = [(65, 1032, 264), (128, 2056, 520), (200, 4096, 1024), (511, 1536, 384), (512, 1024, 8), (513, 1536, 384),
                       (130, 1024, 1376), (400, 1016, 264)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rank", [8, 40])
@pytest.mark.parametrize("kind", ["ragged", "single"])
@pytest.mark.parametrize("rows,inputs,outputs", ROUTES_OF_SOME_ROWS)
def test_linear_of_some_rows(eng, t, rank, kind, rows, inputs, outputs):
    dt = TYPES[t][1]
    g = gen(rows + outputs)
    st = list(range(rows + 1)) if kind == "single" else [0, 0, 3, 60, 70, 127, 131][:4 if rows < 131 else 7] + [rows - 1]
    adapters = 5
    x, w = normal(g, dt, rows, inputs), normal(g, dt, outputs, inputs, scale=inputs ** -0.5)
    a, b = normal(g, dt, adapters, rank, inputs, scale=inputs ** -0.5), normal(g, dt, adapters, outputs, rank, scale=rank ** -0.5)
    scale = torch.rand(adapters, generator=g, device="cuda") + 0.5
    bias = torch.randn(outputs, generator=g, device="cuda")
    ids = [(s * 3) % (adapters + 1) - 1 for s in range(len(st) - 1)]
    y = torch.full((rows, outputs), 7.0, device="cuda").to(dt)
    run_linear(eng, x, w, bias, a, b, scale, y, ints(st), ints(ids))
    torch.cuda.synchronize()
    want, bound = linear_want(x, w, bias, a, b, scale, [(st[s], st[s + 1], i) for s, i in enumerate(ids)])
    within(y[:st[-1]], want[:st[-1]], bound[:st[-1]], dt)
    assert (y[st[-1]:] == 7.0).all()  # of no sequence


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("first,lengths,behind", [(0, [7, 30], 91), (13, [40, 1, 100], 5), (3, [0], 60), (130, [1, 1, 1], 130)])
def test_linear_leaves_rows_of_no_sequence(eng, t, first, lengths, behind):
    dt = TYPES[t][1]
    g = gen(5)
    rows = first + sum(lengths) + behind
    x = normal(g, dt, rows, 128)
    st = starts_of(lengths, first)
    x[:first] = math.nan  # what lies outside the sequences has no effect
    x[st[-1]:] = math.inf
    w, a, b = normal(g, dt, 256, 128), normal(g, dt, 2, 16, 128), normal(g, dt, 2, 256, 16)
    scale = torch.ones(2, device="cuda")
    y = torch.full((rows, 256), 7.0, device="cuda").to(dt)
    ids = [s % 2 for s in range(len(lengths))]
    run_linear(eng, x, w, None, a, b, scale, y, ints(st), ints(ids))
    torch.cuda.synchronize()
    assert (y[:first] == 7.0).all() and (y[st[-1]:] == 7.0).all()
    inside = slice(first, st[-1])
    spans = [(st[s] - first, st[s + 1] - first, i) for s, i in enumerate(ids)]
    want, bound = linear_want(x[inside], w, None, a, b, scale, spans)
    within(y[inside], want, bound, dt)


def test_linear_starts_outside_the_rows(eng):
    # Whatever starts holds, rows outside 0 .. rows-1 are not touched.
    g = gen(9)
    x, w = normal(g, torch.float16, 50, 64), normal(g, torch.float16, 64, 64)
    a, b, scale = normal(g, torch.float16, 1, 8, 64), normal(g, torch.float16, 1, 64, 8), torch.ones(1, device="cuda")
    y = torch.full((70, 64), 7.0, device="cuda").half()
    run_linear(eng, x, w, None, a, b, scale, y, ints([-5, 20, 2 ** 31 - 1]), ints([0, -1]), rows=50)
    torch.cuda.synchronize()
    want, bound = linear_want(x, w, None, a, b, scale, [(0, 20, 0), (20, 50, -1)])
    within(y[:50], want, bound, torch.float16)
    assert (y[50:] == 7.0).all()


# --- attention ---------------------------------------------------------------

def run_attention(e, q, k, v, out, q_starts, k_starts, causal, scale, lse=None, hints=None, stream=0, workspace=None):
    """q, k, v, out: [rows][heads][dim] views of any strides."""
    kind = packed.F16 if q.dtype == torch.float16 else packed.BF16
    call = packed.Attention(
        type=kind, causal=causal, sequences=q_starts.numel() - 1, heads=q.shape[1], kv_heads=k.shape[1], head_dim=q.shape[2],
        q_rows=q.shape[0], k_rows=k.shape[0], scale=scale, q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
        q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0), out_stride=out.stride(0),
        q_head_stride=q.stride(1), k_head_stride=k.stride(1), v_head_stride=v.stride(1), out_head_stride=out.stride(1),
        lse=0 if lse is None else lse.data_ptr(), q_starts=q_starts.data_ptr(), k_starts=k_starts.data_ptr())
    if hints:
        call.longest_q, call.longest_k = hints
    need = e.packed_attention_workspace(call)
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda") if workspace is None else workspace
    call.workspace, call.workspace_bytes = ws.data_ptr(), need
    e.packed_attention(call, stream)
    return ws


def attention_want(q, k, v, causal, scale):
    """(out, bound, lse, its bound) of one sequence, [rows][heads][dim].

    A score is a sum of dim products, off by (dim + 1) f sum|q k|, and its
    exponent carries two more roundings of numbers up to the largest score; a
    weight is then off by that much of itself and 4 f of v_exp_f32 (1 ulp) and
    its argument's sum, P by u more; the sums of weights and of products add
    n f."""
    lq, heads, dim = q.shape
    lk, group = k.shape[0], heads // k.shape[1]
    out, room = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((lq, heads), -math.inf, dtype=torch.float64, device="cuda")
    lse_room = torch.zeros(lq, heads, dtype=torch.float64, device="cuda")
    u = half_step(q.dtype)
    if lk == 0 or lq == 0:
        return out, room, lse, lse_room
    sees = torch.ones(lq, lk, dtype=torch.bool, device="cuda")
    if causal:
        sees = torch.arange(lk, device="cuda") <= torch.arange(lq, device="cuda")[:, None] + (lk - lq)
    some = sees.any(1)
    for h in range(heads):
        qh, kh, vh = q[:, h].double(), k[:, h // group].double(), v[:, h // group].double()
        s = scale * (qh @ kh.t().contiguous())
        size = scale * (qh.abs() @ kh.abs().t().contiguous())
        off = ((dim + 1) * F * size + 4 * F * (s.abs() + s.abs().max())).masked_fill(~sees, 0).amax(1, keepdim=True)
        s = s.masked_fill(~sees, -math.inf)
        top = s.amax(1, keepdim=True).clamp_min(-1e300)
        w = torch.exp(s - top)
        total = w.sum(1, keepdim=True).clamp_min(1e-300)
        out[:, h] = torch.where(some[:, None], (w @ vh.nan_to_num(0, 0, 0)) / total, 0.0)
        rel = 2 * torch.expm1(off) + u + (2 * lk + 16) * F
        # A weight that falls below float32's or the type's normal numbers
        # against the running maximum (at most e^8 under it) is off by 2^-24.
        room[:, h] = torch.where(some[:, None], rel * (w @ vh.abs().nan_to_num(0, 0, 0)) / total + F * vh.abs().nan_to_num(0, 0, 0).sum(0) / total, 0.0)
        lse[:, h] = torch.where(some, (top + total.log())[:, 0], -math.inf)
        lse_room[:, h] = (off + (lk + 16) * F)[:, 0] + 8 * F * lse[:, h].abs().nan_to_num(0, 0, 0)
    return out, room, lse, lse_room


def check_attention(e, dt, ql, kl, heads, kv, dim, causal, *, seed=0, spread=2.0, first=(0, 0), behind=(0, 0), views=None,
                    hints=None, scale=None):
    g = gen(seed + sum(ql) + sum(kl) + dim)
    qs, ks = starts_of(ql, first[0]), starts_of(kl, first[1])
    nq, nk = qs[-1] + behind[0], ks[-1] + behind[1]
    q, k, v = normal(g, dt, nq, heads, dim, scale=spread), normal(g, dt, nk, kv, dim), normal(g, dt, nk, kv, dim)
    # What lies outside the sequences has no effect.
    q[:qs[0]], q[qs[-1]:], k[:ks[0]], k[ks[-1]:], v[:ks[0]], v[ks[-1]:] = [math.nan, math.inf] * 3
    out = torch.full((nq, heads, dim), 7.0, device="cuda").to(dt)
    if views:
        q, k, v, out = views(q, k, v, out)
    lse = torch.full((nq, heads), 7.0, device="cuda")
    scale = dim ** -0.5 if scale is None else scale
    run_attention(e, q, k, v, out, ints(qs), ints(ks), causal, scale, lse, hints)
    torch.cuda.synchronize()
    for s in range(len(ql)):
        a, b, c, f = qs[s], qs[s + 1], ks[s], ks[s + 1]
        want, room, want_lse, lse_room = attention_want(q[a:b], k[c:f], v[c:f], causal, scale)
        within(out[a:b], want, room, dt)
        got = lse[a:b].double()
        empty = want_lse == -math.inf
        assert torch.equal(got == -math.inf, empty)
        assert ((got - want_lse).abs() <= lse_room)[~empty].all()
    for lo, hi in ((0, qs[0]), (qs[-1], nq)):
        assert (out[lo:hi] == 7.0).all() and (lse[lo:hi] == 7.0).all()
    return out


LENGTHS = [[(7 * i) % 50 for i in range(130)], [1] * 63 + [300], [1], [201], [5, 0, 17, 1], [31, 32, 33], [63, 64, 65, 127, 128, 129], [300, 1, 1, 0, 77], [1029]]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("heads,kv,dim", [(6, 6, 64), (8, 2, 128), (3, 1, 32), (5, 5, 80), (4, 4, 96), (16, 2, 8), (14, 2, 120)])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_attention(eng, t, causal, heads, kv, dim, lengths):
    check_attention(eng, TYPES[t][1], lengths, lengths, heads, kv, dim, causal)


# Numbers of queries and keys that differ: single tokens, pooling queries, a
# prompt's next part, keys missing, more queries than keys (rows without keys).
APART = [([1], [1]), ([1], [777]), ([1] * 9, [1, 2, 31, 32, 33, 0, 500, 1000, 64]), ([4] * 5, [201, 0, 3, 64, 700]),
         ([70, 3, 200], [300, 1000, 200]), ([50, 129, 33], [20, 0, 32]), ([260], [100]), ([1, 64, 2], [4000, 4000, 4000]),
         ([i % 3 for i in range(150)], [(i * i) % 90 for i in range(150)])]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (6, 6, 64), (12, 1, 80), (24, 3, 64)])
@pytest.mark.parametrize("ql,kl", APART)
def test_attention_apart(eng, t, causal, heads, kv, dim, ql, kl):
    check_attention(eng, TYPES[t][1], ql, kl, heads, kv, dim, causal, hints=(max(ql), max(kl)))


# One launch on each route: 128-row tiles with one, two and four groups of waves
# (by the number of tiles and the keys), the few-rows kernel with four waves and
# with two, in parts or not.
ROUTES_ATTENTION = [([700] * 8, [700] * 8, 16, 16), ([1500], [1500], 16, 8), ([4200], [4200], 6, 6), ([201], [201], 6, 6),
                    ([1] * 40, [500] * 40, 8, 4), ([1] * 4, [9000, 0, 1, 5000], 8, 1), ([8] * 3, [1000] * 3, 4, 4)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 88, 128])
@pytest.mark.parametrize("ql,kl,heads,kv", ROUTES_ATTENTION)
def test_attention_routes(eng, t, dim, ql, kl, heads, kv):
    causal = dim != 64
    first = check_attention(eng, TYPES[t][1], ql, kl, heads, kv, dim, causal, hints=(max(ql), max(kl)))
    again = check_attention(eng, TYPES[t][1], ql, kl, heads, kv, dim, causal, hints=(max(ql), max(kl)))
    assert torch.equal(first, again)  # the same bits from launch to launch


# Half tiles with four groups (wide heads) and eight (narrow ones, many keys),
# two groups on 128 rows, and the few-rows kernel beside them.
ROUTES_FEW_TILES = [([500], [500], 16, 8), ([300], [3300], 32, 8), ([150, 0, 77, 260], [3500, 10, 0, 3301], 16, 4),
                    ([700] * 3, [700] * 3, 16, 16), ([581], [581], 6, 6), ([64], [4100], 8, 2), ([1400], [1399], 6, 6)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("dim", [32, 64, 80, 128])
@pytest.mark.parametrize("ql,kl,heads,kv", ROUTES_FEW_TILES)
def test_attention_routes_of_few_tiles(eng, t, causal, dim, ql, kl, heads, kv):
    args = eng, TYPES[t][1], ql, kl, heads, kv, dim, causal
    first = check_attention(*args, hints=(max(ql), max(kl)))
    assert torch.equal(first, check_attention(*args, hints=(max(ql), max(kl))))  # the same bits from launch to launch


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal", [0, 1])
def test_attention_rows_of_no_sequence(eng, t, causal):
    check_attention(eng, TYPES[t][1], [40, 1, 90], [40, 64, 100], 4, 2, 64, causal, first=(13, 5), behind=(200, 100))
    check_attention(eng, TYPES[t][1], [1, 1], [40, 300], 4, 2, 128, causal, first=(3, 50), behind=(20, 10), hints=(1, 300))


@pytest.mark.parametrize("t", TYPES)
def test_attention_wrong_hints_cost_time_only(eng, t):
    for hints in ((0, 0), (1, 1), (1, 1 << 31), (1 << 31, 1), (100, 7)):
        check_attention(eng, TYPES[t][1], [100, 1, 30], [100, 700, 30], 4, 2, 64, 1, hints=hints)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("spread,scale", [(30.0, None), (0.01, None), (8.0, 1.0), (100.0, 1.0)])
def test_attention_scores_of_any_size(eng, t, spread, scale):
    check_attention(eng, TYPES[t][1], [150, 1], [150, 900], 4, 2, 64, 1, spread=spread, scale=scale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("lq,lk", [(300, 300), (1, 300), (4, 77), (1500, 1500)])
def test_attention_values_not_finite(eng, t, dim, lq, lk):
    # A key or value that is not finite has no effect on queries that do not see
    # it, and makes those that do not finite, a value in its channel alone.
    dt = TYPES[t][1]
    g = gen(dim + lq)
    heads, kv = 4, 2
    q, k, v = normal(g, dt, lq, heads, dim), normal(g, dt, lk, kv, dim), normal(g, dt, lk, kv, dim)
    want, room, _, _ = attention_want(q, k, v, 1, dim ** -0.5)
    at = {lk * 2 // 3: (math.inf, 3), lk * 2 // 3 + 1: (-math.inf, 7), lk * 3 // 4: (math.nan, 9), lk - 1: (-math.inf, 3)}
    for key, (value, channel) in at.items():
        v[key, :, channel] = value
    out = torch.empty(lq, heads, dim, dtype=dt, device="cuda")
    run_attention(eng, q, k, v, out, ints([0, lq]), ints([0, lk]), 1, dim ** -0.5, hints=(lq, lk))
    torch.cuda.synchronize()
    odd = torch.zeros(lq, dim, dtype=torch.float64, device="cuda")
    for key, (value, channel) in at.items():
        odd[max(0, key - (lk - lq)):, channel] += value
    plain = (odd == 0)[:, None].expand(lq, heads, dim)
    within(out[plain], want[plain], room[plain], dt)
    # Not finite, be it an infinity or no number: a weight under the type's least
    # number (2^-24 of f16) is a zero in the product, and zero times infinity is
    # none.
    assert not out[~plain].isfinite().any()
    # A key that is not a number, seen by the last query only.
    v = normal(g, dt, lk, kv, dim)
    want, room, _, _ = attention_want(q, k, v, 1, dim ** -0.5)
    k[lk - 1] = math.nan
    run_attention(eng, q, k, v, out, ints([0, lq]), ints([0, lk]), 1, dim ** -0.5, hints=(lq, lk))
    torch.cuda.synchronize()
    assert out[lq - 1].isnan().all()
    within(out[:lq - 1], want[:lq - 1], room[:lq - 1], dt)


@pytest.mark.parametrize("t", TYPES)
def test_attention_strides(eng, t):
    dt = TYPES[t][1]

    def in_one_row(q, k, v, out):  # q, k and v as columns of one matrix, out in rows of its own distance
        rows = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1), q.flatten(1)[:, :8]], 1)
        a, b, c = q[0].numel(), k[0].numel(), v[0].numel()
        wide = torch.full((out.shape[0], out[0].numel() + 24), 7.0, device="cuda").to(dt)
        return (rows[:, :a].unflatten(1, q.shape[1:]), rows[:, a:a + b].unflatten(1, k.shape[1:]),
                rows[:, a + b:a + b + c].unflatten(1, v.shape[1:]), wide[:, :out[0].numel()].unflatten(1, out.shape[1:]))

    def by_heads(q, k, v, out):  # [heads][rows][dim]
        return tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, out))

    for views in (in_one_row, by_heads):
        check_attention(eng, dt, [70, 0, 201], [70, 0, 201], 6, 3, 64, 1, views=views)
        check_attention(eng, dt, [100, 513], [100, 513], 8, 2, 128, 0, views=views)
    check_attention(eng, dt, [1, 2], [100, 513], 8, 2, 128, 0, views=by_heads, hints=(2, 513))
