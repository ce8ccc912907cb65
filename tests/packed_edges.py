"""The operators on packed batches at edges of their definitions, against
float64: rotations of heads' first channels where 16-byte pieces do not fit;
adapters that are not finite; rows of attention that are not a number, keys that
weigh nothing, starts that decrease, many sequences. Tolerances as in packed_operators.py."""
import math

import pytest

torch = pytest.importorskip("torch")

import dinov3_hrx as d  # noqa: E402

from packed_operators import (F, TYPES, attention_want, gen, half_step, ints, linear_want, normal, run_attention,  # noqa: E402
                              run_linear, run_rotation, starts_of, within)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(gpu):
    e = d.Engine(0)
    yield e
    e.close()


# --- rotation ----------------------------------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("neighbours", [0, 1])
@pytest.mark.parametrize("rows,heads,dim,rotated,extra", [(1, 1, 8, 8, 0), (57, 2, 16, 8, 8), (201, 12, 80, 40, 960), (130, 5, 40, 40, 0),
                                                          (64, 3, 112, 56, 16), (3, 200, 24, 24, 0), (1029, 1, 80, 40, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rotation_of_an_odd_number_of_eights(eng, t, neighbours, rows, heads, dim, rotated, extra, in_place):
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
    v = before[:, :heads * dim].reshape(rows, heads, dim)
    at = index.long()
    there = (at >= 0) & (at < places)
    c = torch.where(there[:, None], cos.double()[at.clamp(0, places - 1)], 1.0)[:, None]
    s = torch.where(there[:, None], sin.double()[at.clamp(0, places - 1)], 0.0)[:, None]
    one, two = (slice(0, rotated, 2), slice(1, rotated, 2)) if neighbours else (slice(0, rotated // 2), slice(rotated // 2, rotated))
    x1, x2 = v[..., one].double(), v[..., two].double()
    want, bound = v.double().clone(), torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    want[..., one], want[..., two] = x1 * c - x2 * s, x2 * c + x1 * s
    bound[..., one] = 3 * F * ((x1 * c).abs() + (x2 * s).abs())  # two products and a sum
    bound[..., two] = 3 * F * ((x2 * c).abs() + (x1 * s).abs())
    got = out[:, :heads * dim].reshape(rows, heads, dim)
    within(got, want, bound, dt)
    assert torch.equal(got[~there], v[~there])
    assert torch.equal(got[..., rotated:], v[..., rotated:])
    rest = out[:, heads * dim:]
    assert torch.equal(rest, before[:, heads * dim:] if in_place else torch.full_like(rest, 7.0))


# --- projection: an adapter that is not finite ---------------------------------

# A launch on each route: few rows (one, two and four row blocks; columns in
# parts), and each tile.
B_ROUTES = [(12, 264, 136), (30, 264, 136), (60, 264, 136), (60, 2056, 136), (130, 1032, 264), (700, 136, 520), (2500, 136, 1928),
            (2500, 136, 1304), (1500, 136, 1400), (8300, 136, 264), (8200, 136, 264), (3700, 136, 3848)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", ["ragged", "single"])
@pytest.mark.parametrize("rank", [8, 40])
@pytest.mark.parametrize("rows,inputs,outputs", B_ROUTES)
def test_an_adapter_that_is_not_finite_stays_with_its_rows(eng, t, kind, rank, rows, inputs, outputs):
    # Infinities and NaN in B of two adapters: rows of other adapters and rows
    # without one keep every bit; rows of the two are not finite in those columns,
    # an infinity of the right sign where a single infinity meets a nonzero u, and
    # keep every bit in the others.
    dt = TYPES[t][1]
    g = gen(rows + outputs + rank)
    adapters = 5
    if kind == "single":
        st = list(range(rows + 1))
    else:
        st = [s for s in starts_of([(37 * i * i + 11) % 90 for i in range(rows)]) if s < rows - 1] + [rows - 1]  # the last row in none
    ids = [(s * 5 + 2) % (adapters + 1) - 1 for s in range(len(st) - 1)]
    x, w = normal(g, dt, rows, inputs), normal(g, dt, outputs, inputs, scale=inputs ** -0.5)
    a, b = normal(g, dt, adapters, rank, inputs, scale=inputs ** -0.5), normal(g, dt, adapters, outputs, rank, scale=rank ** -0.5)
    scale = torch.rand(adapters, generator=g, device="cuda") + 0.5
    bias = torch.randn(outputs, generator=g, device="cuda")

    def run(b):
        y = torch.full((rows, outputs), 7.0, device="cuda").to(dt)
        run_linear(eng, x, w, bias, a, b, scale, y, ints(st), ints(ids))
        torch.cuda.synchronize()
        return y

    plain = run(b)
    bad = b.clone()
    # [adapter][column][rank column]; adapter 3's column 5 has both infinities.
    places = {(1, 0, 1): math.inf, (1, outputs - 1, rank - 1): math.nan, (3, 5, 0): math.inf, (3, 5, 2): -math.inf, (3, 64, 7): -math.inf}
    for at, value in places.items():
        bad[at] = value
    y = run(bad)
    row_ids = torch.repeat_interleave(torch.tensor(ids), torch.tensor(st).diff()).cuda()
    n = row_ids.numel()
    hit = torch.zeros(rows, outputs, dtype=torch.bool, device="cuda")
    for adapter, column, _ in places:
        hit[:n, column] |= row_ids == adapter
    assert hit.any() and torch.equal(y[~hit], plain[~hit])
    assert not y[hit].isfinite().any()
    # The sum of the infinities times u = scale a x, where u is far enough from
    # zero to have its sign.
    for adapter, column in {p[:2] for p in places}:
        rows_of = (row_ids == adapter).nonzero()[:, 0]
        u = x[rows_of].double() @ a[adapter].double().t().contiguous()
        want = sum(u[:, r] * value for (i, c, r), value in places.items() if (i, c) == (adapter, column))
        clear = (u.abs() > 1e-2).all(1)
        assert torch.equal(y[rows_of, column][clear].double().nan_to_num(9.0), want[clear].nan_to_num(9.0))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [10, 300, 4000])
def test_an_adapter_without_a_finite_value(eng, t, rows):
    # All of B, and rows of one adapter alone in their tiles.
    dt = TYPES[t][1]
    g = gen(rows)
    x, w = normal(g, dt, rows, 128), normal(g, dt, 256, 128)
    a, b = normal(g, dt, 3, 16, 128), normal(g, dt, 3, 256, 16)
    scale = torch.ones(3, device="cuda")
    st, ids = [0, rows // 3, rows // 2, rows], [0, 1, 2]
    ys = []
    for b1 in (b[1], torch.full_like(b[1], math.nan)):
        b[1] = b1
        ys.append(torch.empty(rows, 256, dtype=dt, device="cuda"))
        run_linear(eng, x, w, None, a, b, scale, ys[-1], ints(st), ints(ids))
    torch.cuda.synchronize()
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
    inside[st[1]:st[2]] = True
    assert torch.equal(ys[0][~inside], ys[1][~inside]) and ys[1][inside].isnan().all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("odd", [1, 100])
@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("rows,inputs,outputs", [r for r in B_ROUTES if r[0] > 100])
def test_rows_that_are_not_finite_beside_an_adapter_that_is_not(eng, t, odd, bad, rows, inputs, outputs):
    # Rows of x that are not a number (a few, or whole blocks of the tile), with
    # and without such values in B: the other rows keep every bit.
    dt = TYPES[t][1]
    g = gen(rows + outputs + odd)
    x, w = normal(g, dt, rows, inputs), normal(g, dt, outputs, inputs, scale=inputs ** -0.5)
    a, b = normal(g, dt, 3, 16, inputs, scale=inputs ** -0.5), normal(g, dt, 3, outputs, 16, scale=0.25)
    scale = torch.ones(3, device="cuda")
    st, ids = list(range(0, rows, 10)) + [rows], [s % 3 for s in range((rows + 9) // 10)]
    row_ids = torch.repeat_interleave(torch.tensor(ids), torch.tensor(st).diff()).cuda()
    ys = []
    for _ in range(2):
        ys.append(torch.empty(rows, outputs, dtype=dt, device="cuda"))
        run_linear(eng, x, w, None, a, b, scale, ys[-1], ints(st), ints(ids))
        torch.cuda.synchronize()
        x[20:20 + odd] = math.nan
        if bad:
            b[1, 9, 3] = math.nan
    hit = torch.zeros(rows, outputs, dtype=torch.bool, device="cuda")
    hit[20:20 + odd] = True
    if bad:
        hit[:, 9] |= row_ids == 1
    assert torch.equal(ys[0][~hit], ys[1][~hit]) and ys[1][hit].isnan().all()


# --- projection: sequences without rows ----------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [40, 300, 2500])
def test_linear_with_many_sequences_without_rows(eng, t, rows):
    # Up to 199 empty sequences between two that are not: a tile's rows belong to
    # sequences further apart than the 64 that a wave looks at together.
    dt = TYPES[t][1]
    g = gen(rows)
    lengths, left = [], rows
    while left:
        lengths += [0] * (len(lengths) * 7 % 200) + [min(left, 1 + len(lengths) % 9)]
        left -= lengths[-1]
    st, adapters = starts_of(lengths), 5
    ids = [(s * 5 + 2) % (adapters + 1) - 1 for s in range(len(lengths))]
    x, w = normal(g, dt, rows, 136), normal(g, dt, 200, 136, scale=136 ** -0.5)
    a, b = normal(g, dt, adapters, 8, 136, scale=136 ** -0.5), normal(g, dt, adapters, 200, 8, scale=8 ** -0.5)
    scale = torch.rand(adapters, generator=g, device="cuda") + 0.5
    y = torch.full((rows, 200), 7.0, device="cuda").to(dt)
    run_linear(eng, x, w, None, a, b, scale, y, ints(st), ints(ids))
    torch.cuda.synchronize()
    want, bound = linear_want(x, w, None, a, b, scale, [(st[s], st[s + 1], i) for s, i in enumerate(ids)])
    within(y, want, bound, dt)


# --- attention: rows that are not a number -------------------------------------

# The few-rows kernel with two waves, with four, and in parts of the keys; tiles
# with several groups of waves and with one.
NAN_ROUTES = [(1, 300, 4, 2), (4, 77, 4, 2), (300, 300, 4, 2), (2, 9000, 8, 2), (1500, 1500, 4, 2), (2500, 2500, 32, 16)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("product", [math.nan, math.inf])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("lq,lk,heads,kv", NAN_ROUTES)
def test_log_sum_of_a_row_that_is_not_a_number(eng, t, product, dim, lq, lk, heads, kv):
    # A product that is infinity or not a number, with a key that the last query
    # alone sees: its outputs and its log-sums are not numbers on every route; the
    # other rows keep every bit.
    dt = TYPES[t][1]
    g = gen(dim + lq)
    q, k, v = normal(g, dt, lq, heads, dim), normal(g, dt, lk, kv, dim), normal(g, dt, lk, kv, dim)
    q[..., 0] = 1
    outs, sums = [], []
    for _ in range(2):
        outs.append(torch.empty(lq, heads, dim, dtype=dt, device="cuda"))
        sums.append(torch.zeros(lq, heads, device="cuda"))
        run_attention(eng, q, k, v, outs[-1], ints([0, lq]), ints([0, lk]), 1, dim ** -0.5, sums[-1], hints=(lq, lk))
        torch.cuda.synchronize()
        k[lk - 1] = 0
        k[lk - 1, :, 0] = product
    assert outs[0].isfinite().all() and sums[0].isfinite().all()
    assert torch.equal(outs[0][:-1], outs[1][:-1]) and torch.equal(sums[0][:-1], sums[1][:-1])
    assert outs[1][-1].isnan().all() and sums[1][-1].isnan().all()


# --- attention: keys of no weight ----------------------------------------------

@pytest.mark.parametrize("t,product", [("f16", -math.inf), ("bf16", -math.inf), ("bf16", -3e30)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lq,lk,heads,kv", [(1, 9000, 8, 2), (8, 5000, 4, 4), (1, 300, 4, 2), (300, 900, 4, 2), (1500, 1500, 4, 2)])
@pytest.mark.parametrize("where", ["front", "middle", "back"])
def test_keys_of_no_weight(eng, t, product, dim, lq, lk, heads, kv, where):
    # Products below -1e30 over whole parts of the keys: the result is that of
    # the other keys, whichever part they lie in.
    dt = TYPES[t][1]
    g = gen(dim + lq)
    q, k, v = normal(g, dt, lq, heads, dim), normal(g, dt, lk, kv, dim), normal(g, dt, lk, kv, dim)
    q[..., 0] = 1
    at = {"front": slice(0, lk // 3), "middle": slice(lk // 4, lk * 3 // 4), "back": slice(lk // 2, lk)}[where]
    kept = torch.ones(lk, dtype=torch.bool, device="cuda")
    kept[at] = False
    want, room, want_lse, lse_room = attention_want(q, k[kept], v[kept], 0, dim ** -0.5)
    k[at] = 0
    k[at, :, 0] = product
    out, lse = torch.empty_like(q), torch.zeros(lq, heads, device="cuda")
    run_attention(eng, q, k, v, out, ints([0, lq]), ints([0, lk]), 0, dim ** -0.5, lse, hints=(lq, lk))
    torch.cuda.synchronize()
    within(out, want, room, dt)
    assert ((lse.double() - want_lse).abs() <= lse_room).all()


# --- attention: starts that decrease -------------------------------------------

def test_starts_that_decrease_end(eng):
    # 2^15 sequences of 2^22 rows each in an array of 2^22 rows: 2^32 tiles of 32
    # rows, where sequences in order have 2^17 + 2^16 at most. The call ends, and
    # writes nothing outside the rows.
    rows, sequences, dim = 1 << 22, 1 << 16, 8
    g = gen(1)
    q = normal(g, torch.float16, rows, 1, dim)
    k, v = normal(g, torch.float16, 64, 1, dim), normal(g, torch.float16, 64, 1, dim)
    guard = torch.full((rows + 200, 1, dim), 7.0, dtype=torch.float16, device="cuda")
    turns = torch.arange(sequences + 1, device="cuda") % 2
    run_attention(eng, q, k, v, guard[100:100 + rows], (turns * rows).int(), (turns * 64).int(), 0, dim ** -0.5, hints=(1, 64))
    torch.cuda.synchronize()
    assert (guard[:100] == 7.0).all() and (guard[100 + rows:] == 7.0).all()


# --- attention: many sequences -------------------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (1, 1, 128)])
@pytest.mark.parametrize("sequences", [64, 65, 2100, 9000])
def test_more_sequences_than_workgroups(eng, t, heads, kv, dim, sequences):
    # Single tokens (some sequences without one) with 0 to 6 keys each, then one
    # with many: a workgroup's items lie in windows of 64 sequences far apart.
    dt = TYPES[t][1]
    g = gen(sequences)
    ql = [1 if s % 5 else 0 for s in range(sequences - 1)] + [3]
    kl = [s * s % 7 for s in range(sequences - 1)] + [700]
    qs, ks = starts_of(ql), starts_of(kl)
    q, k, v = normal(g, dt, qs[-1], heads, dim), normal(g, dt, ks[-1], kv, dim), normal(g, dt, ks[-1], kv, dim)
    out, lse = torch.full_like(q, 7.0), torch.full((qs[-1], heads), 7.0, device="cuda")
    run_attention(eng, q, k, v, out, ints(qs), ints(ks), 1, dim ** -0.5, lse, hints=(3, 700))
    torch.cuda.synchronize()
    # Sequences of one query, all at once: each query's keys padded to 6.
    one = torch.tensor([s for s in range(sequences - 1) if ql[s]], device="cuda")
    at = torch.tensor(ks, device="cuda")[one][:, None] + torch.arange(6, device="cuda")
    there = torch.arange(6, device="cuda") < torch.tensor(kl, device="cuda")[one][:, None]
    at = at.clamp_max(ks[-1] - 1)
    q64 = q[:one.numel()].double().view(one.numel(), kv, heads // kv, dim)
    k64, v64 = k[at].double(), v[at].double()  # [query][6][kv][dim]
    s = (q64[:, None] * k64[:, :, :, None]).sum(-1) * dim ** -0.5  # [query][6][kv][group]
    size = (q64[:, None] * k64[:, :, :, None]).abs().sum(-1) * dim ** -0.5
    s = s.masked_fill(~there[:, :, None, None], -math.inf)
    top = s.amax(1, keepdim=True).clamp_min(-1e300)
    w = torch.exp(s - top)
    total = w.sum(1).clamp_min(1e-300)[..., None]
    want = (w[..., None] * v64[:, :, :, None]).sum(1) / total
    mean = (w[..., None] * v64[:, :, :, None].abs()).sum(1) / total
    # As attention_want: a score's error, P's rounding, the sums of 6.
    off = ((dim + 1) * F * size + 4 * F * (s.abs() + s.abs().nan_to_num(0, 0, 0).amax(1, keepdim=True))).masked_fill(~there[:, :, None, None], 0)
    rel = 2 * torch.expm1(off.amax(1)) + half_step(dt) + 28 * F
    floor = F * (v64.abs() * there[:, :, None, None]).sum(1)[:, :, None] / total
    within(out[:one.numel()], want.flatten(1, 2), (rel[..., None] * mean + floor).flatten(1, 2), dt)
    empty = ~there.any(1)
    assert empty.any() and (out[:one.numel()][empty] == 0).all() and (lse[:one.numel()][empty] == -math.inf).all()
    assert lse[:one.numel()][~empty].isfinite().all()
    want, room, want_lse, lse_room = attention_want(q[-3:], k[-700:], v[-700:], 1, dim ** -0.5)
    within(out[-3:], want, room, dt)
    assert ((lse[-3:].double() - want_lse).abs() <= lse_room).all()
