"""The operators of the feed-forward half of a packed block (norms around the
residual step, rows to 4 bits and back, products with 4-bit weights, the gated
projections) against their definitions in float64, where they can go wrong: rows
of no sequence, empty and single-row sequences, odd sizes, strides, in place,
values that are not finite, subnormal and huge blocks, every activation and tile.

Tolerances are bounds from the arithmetic, as in packed_operators.py: F = 2^-24
for each float32 operation, (n + 1) F of the sum of magnitudes for a sum of n
products, half a step of the type for the one rounding of an output; errors are
carried through each formula to first order, with a tenth more for the rest."""
import math

import pytest

torch = pytest.importorskip("torch")

import dinov3_hrx as d  # noqa: E402
from dinov3_hrx import packed  # noqa: E402

from packed_operators import F, TYPES, gen, half_step, ints, normal, starts_of, within  # noqa: E402

pytestmark = pytest.mark.gpu

KIND = {torch.float16: packed.F16, torch.bfloat16: packed.BF16, torch.float32: packed.F32}
NORMS = {"none": packed.NONE, "rms": packed.RMS, "layer": packed.LAYER}
ACTIVATIONS = {"silu": packed.SILU, "gelu": packed.GELU, "gelu_tanh": packed.GELU_TANH, "relu": packed.RELU, "sigmoid": packed.SIGMOID}


@pytest.fixture(scope="module")
def eng(gpu):
    e = d.Engine(0)
    yield e
    e.close()


def at(t):
    return 0 if t is None else t.data_ptr()


# --- norms -------------------------------------------------------------------

def run_norm(e, x, y, x_out, h, post="none", pre="none", post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, scale=None,
             gate=None, starts=None, eps=(1e-5, 1e-6), channels=None, stream=0):
    other = y if y is not None else h
    e.packed_norm(packed.Norm(
        type=KIND[other.dtype], stream_type=KIND[x.dtype], post=NORMS[post], pre=NORMS[pre], rows=x.shape[0],
        channels=channels or x.shape[1], sequences=0 if starts is None else starts.numel() - 1, post_eps=eps[0], pre_eps=eps[1], x=at(x),
        y=at(y), x_out=at(x_out), h=at(h), post_weight=at(post_weight), post_bias=at(post_bias), pre_weight=at(pre_weight),
        pre_bias=at(pre_bias), scale=at(scale), gate=at(gate), x_stride=x.stride(0), y_stride=0 if y is None else y.stride(0),
        x_out_stride=0 if x_out is None else x_out.stride(0), h_stride=0 if h is None else h.stride(0),
        gate_stride=0 if gate is None else gate.stride(0), starts=at(starts)), stream)


def norm_want(v, ev, kind, eps, weight, bias):
    """(norm of v, its error) for float64 rows v that the kernel holds to within ev."""
    if kind == "none":
        return v, ev
    n = v.shape[1]
    if kind == "layer":
        mean = v.mean(1, keepdim=True)
        em = ev.mean(1, keepdim=True) + (n + 2) * F * v.abs().mean(1, keepdim=True)
        v = v - mean
        ev = ev + em + F * v.abs()
    var = (v * v).mean(1, keepdim=True)
    evar = (2 * v.abs() * ev + ev * ev).mean(1, keepdim=True) + (n + 3) * F * var
    r = torch.rsqrt(var + eps)
    off = 1.1 * (0.5 * evar / (var + eps) + 4 * F)  # relative, of r: its argument's, the addition's and its own
    out, eo = v * r, ev * r * (1 + off) + v.abs() * r * (off + F)
    if weight is not None:
        out, eo = out * weight.double(), 1.1 * eo * weight.double().abs() + F * (out * weight.double()).abs()
    if bias is not None:
        out = out + bias.double()
        eo = eo + F * (out.abs() + eo)
    return out, eo


def step_want(x, y, post, pre, vectors, gate_rows, eps=(1e-5, 1e-6)):
    """((x', error), (h, error))."""
    new, e = x.double(), torch.zeros_like(x, dtype=torch.float64)
    if y is not None:
        z, ez = norm_want(y.double(), torch.zeros_like(new), post, eps[0], vectors.get("post_weight"), vectors.get("post_bias"))
        for by in (vectors.get("scale"), gate_rows):
            if by is not None:
                z, ez = z * by.double(), 1.1 * ez * by.double().abs() + F * (z * by.double()).abs()
        new = new + z
        e = ez + F * (new.abs() + ez)
    return (new, e), norm_want(new, e, pre, eps[1], vectors.get("pre_weight"), vectors.get("pre_bias"))


def vectors_of(g, channels, post, pre, which):
    out = {}
    for i, name in enumerate(("post_weight", "post_bias", "pre_weight", "pre_bias", "scale")):
        if which >> i & 1 and not (name.startswith("post") and post == "none") and not (name.startswith("pre") and pre == "none"):
            out[name] = torch.randn(channels, generator=g, device="cuda")
    return out


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("post,pre", [("none", "layer"), ("rms", "rms"), ("layer", "none"), ("layer", "layer"), ("none", "none"), ("rms", "none")])
@pytest.mark.parametrize("lengths,channels,which", [([1], 8, 31), ([5, 0, 17, 1], 384, 31), ([3, 130], 72, 5), ([40], 1000, 26),
                                                    ([2, 9, 0], 2056, 31), ([7], 4096, 0), ([2, 1], 8192, 31), ([3], 32768, 21)])
def test_norm(eng, t, wide, post, pre, lengths, channels, which):
    dt = TYPES[t][1]
    st = torch.float32 if wide else dt
    g = gen(channels + len(lengths))
    rows, spare = sum(lengths), 6
    x = (normal(g, torch.float32, rows + spare, channels + 16, scale=3.0) + 0.5).to(st)[:, :channels]
    y = normal(g, dt, rows + spare, channels + 8)[:, :channels]
    gate = torch.randn(len(lengths), channels + 8, generator=g, device="cuda")[:, :channels] if which & 1 else None
    vectors = vectors_of(g, channels, post, pre, which)
    first = 2
    starts = starts_of(lengths, first)
    x_out, h = (torch.full((rows + spare, channels + 8), 7.0, device="cuda").to(k) for k in (st, dt))
    run_norm(eng, x, y, x_out[:, :channels], h[:, :channels] if pre != "none" else None, post, pre, gate=gate, starts=ints(starts), **vectors)
    torch.cuda.synchronize()
    mine = slice(first, first + rows)
    by = None
    if gate is not None:
        by = torch.cat([gate[s].expand(n, channels) for s, n in enumerate(lengths)])
    (want, e), (want_h, eh) = step_want(x[mine], y[mine], post, pre, vectors, by)
    within(x_out[mine, :channels], want, e, st)
    if pre != "none":
        within(h[mine, :channels], want_h, eh, dt)
    for out in (x_out,) if pre == "none" else (x_out, h):  # rows of no sequence, and what lies between rows
        assert (out[:first] == 7.0).all() and (out[first + rows:] == 7.0).all() and (out[:, channels:] == 7.0).all()


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("channels", [64, 384, 5000])
def test_norm_in_place_and_in_front_of_the_first_block(eng, dt, channels):
    g = gen(channels)
    x, y = normal(g, dt, 33, channels), normal(g, dt, 33, channels)
    w = torch.randn(channels, generator=g, device="cuda")
    out, h = torch.empty_like(x), torch.empty_like(y)
    run_norm(eng, x, y, out, h, "rms", "layer", pre_weight=w)
    a, b = x.clone(), y.clone()
    run_norm(eng, a, b, a, b, "rms", "layer", pre_weight=w)
    torch.cuda.synchronize()
    assert torch.equal(a, out) and torch.equal(b, h)
    run_norm(eng, x, None, None, h, "none", "layer", pre_weight=w)
    torch.cuda.synchronize()
    _, (want, e) = step_want(x, None, "none", "layer", {"pre_weight": w}, None)
    within(h, want, e, dt)


def test_norm_of_many_sequences(eng):
    # More sequences than a wave has lanes, many of them empty, a gate each.
    g = gen(4)
    lengths = [(s * 7) % 5 if s % 3 else 0 for s in range(700)]
    for channels in (40, 384, 1024, 4096):
        rows = sum(lengths)
        x, y = normal(g, torch.bfloat16, rows, channels), normal(g, torch.bfloat16, rows, channels)
        gate = torch.randn(len(lengths), channels, generator=g, device="cuda")
        out = torch.empty_like(x)
        run_norm(eng, x, y, out, None, gate=gate, starts=ints(starts_of(lengths)))
        torch.cuda.synchronize()
        by = torch.repeat_interleave(gate, torch.tensor(lengths, device="cuda"), 0)
        (want, e), _ = step_want(x, y, "none", "none", {}, by)
        within(out, want, e, torch.bfloat16)


def test_norm_values_that_are_not_finite_stay_in_their_row(eng):
    g = gen(8)
    for channels in (64, 384, 2048, 4096):
        x, y = normal(g, torch.float16, 20, channels), normal(g, torch.float16, 20, channels)
        out, h = torch.empty_like(x), torch.empty_like(x)
        run_norm(eng, x, y, out, h, "layer", "rms")
        a, b = x.clone(), y.clone()
        a[3, 5], b[7, 9], b[11, 0] = math.inf, math.nan, -math.inf
        out2, h2 = torch.empty_like(x), torch.empty_like(x)
        run_norm(eng, a, b, out2, h2, "layer", "rms")
        torch.cuda.synchronize()
        same = [r for r in range(20) if r not in (3, 7, 11)]
        assert torch.equal(out[same], out2[same]) and torch.equal(h[same], h2[same])
        assert out2[3, 5] == math.inf and h2[3, 5].isnan() and (h2[3, :5] == 0).all()
        for r in (7, 11):
            assert out2[r].isnan().all() and h2[r].isnan().all()


def test_norm_of_large_means(eng):
    # A mean far above the deviations: the deviations are summed, not the squares.
    g = gen(6)
    x = (normal(g, torch.float32, 50, 384) + 1000.0).float()
    h = torch.empty(50, 384, dtype=torch.float16, device="cuda")
    run_norm(eng, x, None, None, h, "none", "layer")
    torch.cuda.synchronize()
    want = torch.nn.functional.layer_norm(x.double(), (384,), eps=1e-6)
    # the mean of 1000 passes at most 8 sums in a lane, 6 across lanes and two roundings
    # (of 1 / 384 and the product), each under F 1001
    within(h, want, 17 * F * 1001 * 1.2 + 17 * F * want.abs(), torch.float16)


def test_norm_of_rows_past_the_range_and_of_zeros(eng):
    # As the header says: squares past float32's range, and 0 / 0 with eps 0; their
    # neighbours are untouched.
    for channels in (64, 384, 4096):
        x = torch.ones(4, channels, dtype=torch.bfloat16, device="cuda")
        x[1] = 1e30
        x[2] = 0.0
        h = torch.empty_like(x)
        run_norm(eng, x, None, None, h, "none", "rms", eps=(0.0, 0.0))
        torch.cuda.synchronize()
        assert (h[0] == 1).all() and (h[3] == 1).all() and (h[1] == 0).all() and h[2].isnan().all()
        run_norm(eng, x, None, None, h, "none", "layer", eps=(0.0, 1e-5))
        torch.cuda.synchronize()
        assert (h[[0, 2, 3]] == 0).all()


# --- 4 bits ------------------------------------------------------------------

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def pad16(columns):
    return ((columns + 31) // 32 + 15) // 16 * 16


def quantised_want(x):
    """(codes, scale bytes) of the rows of x by the definition, on the CPU."""
    rows, columns = x.shape
    v = torch.nn.functional.pad(x.cpu().double(), (0, -columns % 32)).view(rows, -1, 32)
    top = v.abs().amax(2)
    finite = v.isfinite().all(2)
    exponent = torch.where(top > 0, torch.frexp(top)[1] - 1, torch.full_like(top, -1000, dtype=torch.int32)) - 2
    exponent = exponent.clamp(-127, 127)
    size = v.abs() / torch.ldexp(torch.ones_like(top), exponent)[:, :, None]
    distance = (size.clamp_max(6.0)[..., None] - torch.tensor(GRID, dtype=torch.float64)).abs()
    near = distance == distance.amin(3, keepdim=True)  # two of them in a tie: the even one
    index = torch.arange(8)
    codes = torch.where(near & (index % 2 == 0), index, -1).amax(3)
    odd = torch.where(near, index, -1).amax(3)
    codes = torch.where(codes >= 0, codes, odd) + 8 * torch.signbit(v)
    codes = torch.where(finite[:, :, None], codes, 0).to(torch.uint8).view(rows, -1)
    scales = torch.where(finite, exponent + 127, 255).to(torch.uint8)
    return codes[:, 0::2] + 16 * codes[:, 1::2], torch.nn.functional.pad(scales, (0, -scales.shape[1] % 16))


def values(codes, scales, columns):
    """What codes and scale bytes stand for, in float64."""
    table = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device=codes.device)
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], 2).flatten(1)
    n = v.shape[1] // 32
    # Powers of two from the host: on the GPU ldexp is a product with a rounded pow.
    steps = torch.tensor([2.0 ** (b - 127) for b in range(255)] + [math.nan], dtype=torch.float64).to(codes.device)
    by = steps[scales[:, :n].long()]
    return (v.view(-1, n, 32) * by[:, :, None]).flatten(1)[:, :columns]


def four(x, codes=None, scales=None):
    rows, columns = x.shape
    codes = torch.full((rows, (columns + 31) // 32 * 16), 0xee, dtype=torch.uint8, device="cuda") if codes is None else codes
    scales = torch.full((rows, pad16(columns)), 0xee, dtype=torch.uint8, device="cuda") if scales is None else scales
    return codes, scales


def quantisation(x, codes, scales, starts=None):
    return packed.Quantisation(type=KIND[x.dtype], sequences=0 if starts is None else starts.numel() - 1, rows=x.shape[0], columns=x.shape[1],
                               x=at(x), x_stride=x.stride(0), codes=at(codes), codes_stride=codes.stride(0), scales=at(scales),
                               scales_stride=scales.stride(0), starts=at(starts))


def quantised(e, x):
    codes, scales = four(x)
    e.packed_quantise(quantisation(x, codes, scales))
    return codes, scales


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,columns", [(1, 8), (1, 32), (7, 40), (33, 384), (5, 1000), (300, 512), (2, 4104), (64, 24)])
def test_quantise(eng, t, rows, columns):
    dt = TYPES[t][1]
    g = gen(rows + columns)
    x = normal(g, torch.float32, rows, columns + 8) * torch.exp2(torch.randint(-8, 9, (rows, columns + 8), generator=g, device="cuda"))
    x = x.to(dt)[:, :columns]
    codes, scales = (torch.full((rows, n + 32), 0xee, dtype=torch.uint8, device="cuda") for n in ((columns + 31) // 32 * 16, pad16(columns)))
    n_codes, n_scales = codes.shape[1] - 32, scales.shape[1] - 32
    eng.packed_quantise(quantisation(x, codes, scales))
    back = torch.full((rows, columns + 8), 7.0, device="cuda").to(dt)
    eng.packed_dequantise(quantisation(back[:, :columns], codes, scales))
    torch.cuda.synchronize()
    want_codes, want_scales = quantised_want(x)
    assert torch.equal(scales[:, :n_scales].cpu(), want_scales)
    assert torch.equal(codes[:, :n_codes].cpu(), want_codes)
    assert (codes[:, n_codes:] == 0xee).all() and (scales[:, n_scales:] == 0xee).all() and (back[:, columns:] == 7.0).all()
    assert torch.equal(back[:, :columns].double().cpu(), values(want_codes, want_scales, columns))


@pytest.mark.parametrize("t", TYPES)
def test_quantise_every_value(eng, t):
    # Every finite value of the type as a block's largest, with fractions of it that
    # lie on, next to and between the borders of the codes.
    dt = TYPES[t][1]
    top = torch.arange(0x7c00 if t == "f16" else 0x7f80, dtype=torch.int32).to(torch.int16).view(dt).double()
    exponent = torch.floor(torch.log2(top.clamp_min(1e-300))) - 2
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    borders = torch.cat([borders, borders * (1 - 2.0 ** -7), borders * (1 + 2.0 ** -7), borders + 0.1])
    x = torch.zeros(top.numel(), 32, dtype=torch.float64)
    x[:, 3] = top
    x[:, 4:] = torch.minimum(borders * torch.exp2(exponent)[:, None], top[:, None])
    x[:, 5::2] *= -1
    x = x.to(dt).cuda()
    codes, scales = quantised(eng, x)
    back = torch.empty_like(x)
    eng.packed_dequantise(quantisation(back, codes, scales))
    torch.cuda.synchronize()
    want_codes, want_scales = quantised_want(x)
    assert torch.equal(scales.cpu(), want_scales) and torch.equal(codes.cpu(), want_codes)
    assert torch.equal(back.double().cpu(), values(want_codes, want_scales, 32))


def test_quantise_blocks_that_are_not_finite(eng):
    g = gen(3)
    for dt in KIND:
        if dt == torch.float32:
            continue
        x = normal(g, dt, 6, 136)
        x[1, 40], x[2, 0], x[2, 135], x[4, 64] = math.nan, math.inf, -math.inf, math.nan
        codes, scales = quantised(eng, x)
        back = torch.empty_like(x)
        eng.packed_dequantise(quantisation(back, codes, scales))
        torch.cuda.synchronize()
        want_codes, want_scales = quantised_want(x)
        assert torch.equal(scales.cpu(), want_scales) and torch.equal(codes.cpu(), want_codes)
        bad = want_scales[:, :5].repeat_interleave(32, 1)[:, :136] == 255
        assert torch.equal(back.isnan().cpu(), bad) and int(bad.sum()) == 32 * 3 + 8


def test_quantise_rows_of_no_sequence(eng):
    x = normal(gen(1), torch.float16, 40, 96)
    codes, scales = four(x)
    starts = ints([5, 5, 9, 30])
    eng.packed_quantise(quantisation(x, codes, scales, starts))
    all_codes, all_scales = quantised(eng, x)
    back = torch.full_like(x, 7.0)
    eng.packed_dequantise(quantisation(back, all_codes, all_scales, starts))
    torch.cuda.synchronize()
    for got, want in ((codes, all_codes), (scales, all_scales)):
        assert torch.equal(got[5:30], want[5:30]) and (got[:5] == 0xee).all() and (got[30:] == 0xee).all()
    assert (back[:5] == 7.0).all() and (back[30:] == 7.0).all()
    assert torch.equal(back[5:30].double(), values(all_codes, all_scales, 96)[5:30])


# --- products ----------------------------------------------------------------

def product_want(x, w, bias):
    """(x w^T + bias, its error) of float64 matrices whose products float32 holds."""
    want = x @ w.t().contiguous()
    size = x.abs() @ w.abs().t().contiguous()
    e = (x.shape[1] + 2) * F * size
    if bias is not None:
        want = want + bias.double()
        e = e + F * (want.abs() + e)
    return want, e


def run_linear4(e, x, codes, scales, bias, y, starts=None, workspace=None, stream=0):
    call = packed.QuantisedLinear(
        type=KIND[x.dtype], sequences=0 if starts is None else starts.numel() - 1, rows=x.shape[0], inputs=x.shape[1], outputs=codes.shape[0],
        x=at(x), w=at(codes), w_scales=at(scales), bias=at(bias), y=at(y), x_stride=x.stride(0), y_stride=y.stride(0),
        w_stride=codes.stride(0), scales_stride=scales.stride(0), starts=at(starts))
    need = e.packed_quantised_linear_workspace(call)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda") if workspace is None else workspace
    call.workspace, call.workspace_bytes = at(ws), need
    e.packed_quantised_linear(call, stream)
    return ws


def run_gated(e, x, gate, up, gate_bias, up_bias, out, activation, scales=None, starts=None, workspace=None, stream=0):
    call = packed.Gated(
        type=KIND[x.dtype], activation=ACTIVATIONS[activation], rows=x.shape[0], inputs=x.shape[1], outputs=gate.shape[0],
        sequences=0 if starts is None else starts.numel() - 1, x=at(x), gate=at(gate), up=at(up),
        gate_scales=at(scales and scales[0]), up_scales=at(scales and scales[1]), gate_bias=at(gate_bias), up_bias=at(up_bias), out=at(out),
        x_stride=x.stride(0), out_stride=out.stride(0), w_stride=gate.stride(0), scales_stride=scales[0].stride(0) if scales else 0,
        starts=at(starts))
    need = e.packed_gated_workspace(call)
    assert scales or not need
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda") if workspace is None else workspace
    call.workspace, call.workspace_bytes = at(ws), need
    e.packed_gated(call, stream)
    return ws


def weights4(e, g, outputs, inputs, dt):
    """(codes, scales, values) of a random matrix; the bytes that fill its scales up are not a number."""
    codes, scales = quantised(e, normal(g, dt, outputs, inputs, scale=inputs ** -0.5))
    scales[:, (inputs + 31) // 32:] = 255
    return codes, scales, values(codes, scales, inputs)


SIZES = [(8, 8), (64, 72), (384, 1152), (136, 200), (1000, 328), (1536, 384), (40, 1000), (512, 64), (4104, 136)]
LENGTHS = [[1], [5, 0, 17, 1], [9], [201, 33], [64], [640, 3]]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("inputs,outputs", SIZES)
def test_quantised_linear(eng, t, lengths, inputs, outputs):
    dt = TYPES[t][1]
    g = gen(sum(lengths) + inputs)
    rows, first = sum(lengths), 3
    x = normal(g, dt, rows + 5, inputs + 8)[:, :inputs]
    codes, scales, w = weights4(eng, g, outputs, inputs, dt)
    bias = torch.randn(outputs, generator=g, device="cuda") if inputs != 64 else None
    y = torch.full((rows + 5, outputs + 8), 7.0, device="cuda").to(dt)
    run_linear4(eng, x, codes, scales, bias, y, ints(starts_of(lengths, first)))
    torch.cuda.synchronize()
    mine = slice(first, first + rows)
    xq = values(*(t.cuda() for t in quantised_want(x[mine])), inputs)
    want, e = product_want(xq, w, bias)
    within(y[mine, :outputs], want, e, dt)
    assert (y[:first] == 7.0).all() and (y[first + rows:] == 7.0).all() and (y[:, outputs:] == 7.0).all()


def activation_want(name, g, e):
    """(act(g), its error) for sums g that are within e."""
    size = g.abs()
    if name == "relu":
        return g.clamp_min(0), e
    if name == "sigmoid":
        out = torch.sigmoid(g)  # e^-g: its argument's two roundings and its own; the sum; the reciprocal
        return out, 0.25 * e + 1.1 * out * (2 * size + 8) * F
    if name == "silu":
        out = g * torch.sigmoid(g)
        return out, 1.1 * e + 1.1 * out.abs() * (2 * size + 9) * F
    if name == "gelu":
        # erf within 4 steps of 1, its argument's rounding (at most 0.5 F), the sum
        return torch.nn.functional.gelu(g), 1.13 * e + 0.5 * size * 12 * F
    inner = 2 * math.sqrt(2 / math.pi) * (size + 0.044715 * size ** 3)
    out = torch.nn.functional.gelu(g, approximate="tanh")
    return out, 1.13 * e + 1.1 * out.abs() * (6 * inner + 9) * F + 1e-37


def gated_want(name, x, gate, up, gate_bias, up_bias):
    (g, eg), (u, eu) = product_want(x, gate, gate_bias), product_want(x, up, up_bias)
    a, ea = activation_want(name, g, eg)
    want = a * u
    e = ea * u.abs() + a.abs() * eu + ea * eu
    return want, e + F * (want.abs() + e)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("inputs,outputs", SIZES)
def test_gated(eng, t, bits, lengths, inputs, outputs):
    dt = TYPES[t][1]
    g = gen(sum(lengths) + inputs + bits)
    rows, first = sum(lengths), 2
    activation = list(ACTIVATIONS)[(inputs // 8 + len(lengths)) % 5]
    x = normal(g, dt, rows + 4, inputs + 8)[:, :inputs]
    bias = torch.randn(2, outputs, generator=g, device="cuda") if inputs != 64 else (None, None)
    out = torch.full((rows + 4, outputs + 8), 7.0, device="cuda").to(dt)
    mine = slice(first, first + rows)
    if bits == 4:
        (gate, gs, gw), (up, us, uw) = (weights4(eng, g, outputs, inputs, dt) for _ in range(2))
        scales, xs = (gs, us), values(*(t.cuda() for t in quantised_want(x[mine])), inputs)
    else:  # the halves of one matrix
        both = normal(g, dt, 2 * outputs, inputs + 8, scale=inputs ** -0.5)[:, :inputs]
        gate, up, scales, xs = both[:outputs], both[outputs:], None, x[mine].double()
        gw, uw = gate.double(), up.double()
    run_gated(eng, x, gate, up, bias[0], bias[1], out, activation, scales, ints(starts_of(lengths, first)))
    torch.cuda.synchronize()
    want, e = gated_want(activation, xs, gw, uw, bias[0], bias[1])
    within(out[mine, :outputs], want, e, dt)
    assert (out[:first] == 7.0).all() and (out[first + rows:] == 7.0).all() and (out[:, outputs:] == 7.0).all()


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_activations_over_their_range(eng, activation, dt):
    # One input column: the sums are x times the weight, -200 to 200.
    x = torch.zeros(401, 8, device="cuda")
    x[:, 0] = torch.linspace(-1, 1, 401)
    x = x.to(dt)
    w = torch.zeros(2, 64, 8, device="cuda")
    w[0, :, 0] = torch.logspace(-3, 2.3, 64)
    w[1, :, 1] = 1.0
    w = w.to(dt)
    ones = torch.ones(64, device="cuda")
    out = torch.empty(401, 64, dtype=dt, device="cuda")
    run_gated(eng, x, w[0], w[1], None, ones, out, activation)
    torch.cuda.synchronize()
    want, e = gated_want(activation, x.double(), w[0].double(), w[1].double(), None, ones)
    within(out, want, e, dt)


def test_products_with_values_that_are_not_finite(eng):
    # They stay in their row of x and in their column of the weights.
    g = gen(12)
    for rows in (3, 70, 300):
        for bits in (16, 4):
            x = normal(g, torch.bfloat16, rows, 160)
            w = normal(g, torch.bfloat16, 2, 96, 160, scale=0.1)
            x2, w2 = x.clone(), w.clone()
            x2[1, 5], x2[rows - 1, 159], w2[0, 7, 33], w2[1, 90, 159] = math.nan, math.inf, math.inf, math.nan
            outs = []
            for a, b in ((x, w), (x2, w2)):
                out = torch.empty(rows, 96, dtype=torch.bfloat16, device="cuda")
                if bits == 4:
                    (gate, gs), (up, us) = quantised(eng, b[0]), quantised(eng, b[1])
                    run_gated(eng, a, gate, up, None, None, out, "silu", (gs, us))
                    y = torch.empty_like(out)
                    run_linear4(eng, a, gate, gs, None, y)
                else:
                    run_gated(eng, a, b[0], b[1], None, None, out, "silu")
                    y = None
                outs.append((out, y))
            torch.cuda.synchronize()
            same = torch.ones(rows, 96, dtype=torch.bool, device="cuda")
            same[1], same[rows - 1], same[:, 7], same[:, 90] = False, False, False, False
            assert torch.equal(outs[0][0][same], outs[1][0][same])
            assert outs[1][0][1].isnan().all()
            if bits == 4:
                assert outs[1][0][~same].isnan().all()
                same[:, 90] = True
                same[1], same[rows - 1] = False, False
                assert torch.equal(outs[0][1][same], outs[1][1][same]) and outs[1][1][~same].isnan().all()


def test_quantised_product_of_extreme_scales(eng):
    # Blocks near both ends of the type's range: their scales cancel in the product.
    g = gen(14)
    x = normal(g, torch.bfloat16, 70, 256) * 2.0 ** 100
    w = normal(g, torch.bfloat16, 96, 256) * 2.0 ** -110
    x[:, 64:128] *= 2.0 ** -220
    codes, scales = quantised(eng, w)
    y = torch.empty(70, 96, dtype=torch.bfloat16, device="cuda")
    run_linear4(eng, x, codes, scales, None, y)
    torch.cuda.synchronize()
    want, e = product_want(values(*(t.cuda() for t in quantised_want(x)), 256), values(codes, scales, 256), None)
    within(y, want, e, torch.bfloat16)
