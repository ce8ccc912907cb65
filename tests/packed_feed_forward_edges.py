"""The operators of the feed-forward half of a packed block at edges of their
definitions: float32 rows of one value, outputs in the place of inputs, activations
far from zero, forms of the kernels that few sizes take. Tolerances as in
packed_feed_forward.py."""
import math

import pytest

torch = pytest.importorskip("torch")

import dinov3_hrx as d  # noqa: E402

import packed_block  # noqa: E402
import packed_feed_forward  # noqa: E402
from packed_feed_forward import ACTIVATIONS, activation_want, norm_want, run_gated, run_norm  # noqa: E402
from packed_operators import F, TYPES, gen, normal, within  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(gpu):
    e = d.Engine(0)
    yield e
    e.close()


# --- norms -------------------------------------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("channels", [8, 72, 136, 384, 1000, 4096, 8200, 20000])
def test_layer_norm_of_a_row_of_one_value(eng, t, channels):
    # The mean is that value, whatever it is, so that nothing is left of the row: its
    # norm is the bias, and without an eps 0 / 0.
    dt = TYPES[t][1]
    g = gen(channels)
    value = torch.randn(200, 1, generator=g, device="cuda") * torch.exp2(torch.randint(-8, 12, (200, 1), generator=g, device="cuda"))
    value[:3, 0] = torch.tensor([0.3, 1000.1, -1.1])
    rows, more = value.shape[0], torch.randn(channels, generator=g, device="cuda")
    x = value.expand(rows, channels).contiguous()
    h = torch.empty(rows, channels, dtype=dt, device="cuda")
    for bias in (None, more):
        run_norm(eng, x, None, None, h, "none", "layer", pre_weight=more, pre_bias=bias, eps=(0.0, 1e-6))
        torch.cuda.synchronize()
        assert (h == (0.0 if bias is None else bias.to(dt))).all()
    run_norm(eng, x, None, None, h, "none", "layer", eps=(0.0, 0.0))
    torch.cuda.synchronize()
    assert h.isnan().all()
    # Behind the residual step, which is not rounded in front of the norm, and in y.
    y, out = value.flip(0).to(dt).expand(rows, channels).contiguous(), torch.empty_like(x)
    scale = torch.full((channels,), 0.3, device="cuda")
    run_norm(eng, x, y, out, h, "none", "layer", scale=scale, pre_bias=more, eps=(0.0, 1e-6))
    torch.cuda.synchronize()
    assert (h == more.to(dt)).all()
    run_norm(eng, x, y, out, h, "layer", "layer", post_bias=scale, pre_bias=more, eps=(1e-6, 1e-6))
    torch.cuda.synchronize()
    assert torch.equal(out, x + scale) and (h == more.to(dt)).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("channels", [8, 72, 136, 384, 1000, 4096, 8200, 20000])
def test_layer_norm_of_a_row_of_nearly_one_value(eng, t, channels):
    # A few steps of float32 around a value: deviations from the mean, from the first of
    # them and their sum are whole numbers of steps, so exact; their mean is rounded once
    # and so is what it is taken from.
    dt = TYPES[t][1]
    g = gen(channels)
    value = torch.tensor([0.3, 1000.1, -1.1, 7.0e4, -3.0e-5], device="cuda")[:, None]
    steps = torch.randint(-3, 4, (5, channels), generator=g, device="cuda")
    steps[:, :2] = torch.tensor([1, -2], device="cuda")
    x = (value.view(torch.int32) + steps.int()).view(torch.float32)
    w, b = (torch.randn(channels, generator=g, device="cuda") for _ in range(2))
    h = torch.empty(5, channels, dtype=dt, device="cuda")
    run_norm(eng, x, None, None, h, "none", "layer", pre_weight=w, pre_bias=b, eps=(0.0, 0.0))
    torch.cuda.synchronize()
    v = x.double() - x.double().mean(1, keepdim=True)
    want, e = norm_want(v, 2 * F * (v.abs() + v[:, :1].abs()), "rms", 0.0, w, b)
    within(h, want, e, dt)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("channels", [8, 72, 136, 384, 1000, 12288])
def test_rows_of_one_value_beside_others(eng, t, channels):
    # Rows that share a wave with them have the same bits as without them.
    dt = TYPES[t][1]
    g = gen(channels)
    x = normal(g, torch.float32, 67, channels, scale=2.0)
    x[5, 0], x[9, channels - 1] = math.inf, math.nan
    with_them, odd = x.clone(), torch.arange(67, device="cuda") % 3 == 1
    with_them[odd] = torch.randn(67, 1, generator=g, device="cuda")[odd].expand(-1, channels)
    alone, h = torch.empty(67, channels, dtype=dt, device="cuda"), torch.empty(67, channels, dtype=dt, device="cuda")
    run_norm(eng, x, None, None, alone, "none", "layer", eps=(0.0, 1e-6))
    run_norm(eng, with_them, None, None, h, "none", "layer", eps=(0.0, 1e-6))
    torch.cuda.synchronize()
    bits = lambda v: v[~odd].view(torch.int16)  # noqa: E731
    assert torch.equal(bits(h), bits(alone)) and (h[odd] == 0).all()
    assert h[5].isnan().all() and h[9].isnan().all()


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("channels", [64, 384, 4096, 12288])
def test_norm_in_place_the_other_way_round(eng, dt, channels):
    # h where x was, x_out where y was.
    g = gen(channels)
    x, y = normal(g, dt, 33, channels), normal(g, dt, 33, channels)
    for post, pre in (("none", "layer"), ("rms", "rms")):
        out, h = torch.empty_like(x), torch.empty_like(x)
        run_norm(eng, x, y, out, h, post, pre)
        a, b = x.clone(), y.clone()
        run_norm(eng, a, b, b, a, post, pre)
        torch.cuda.synchronize()
        assert torch.equal(a, h) and torch.equal(b, out)
    a = x.clone()
    run_norm(eng, x, None, None, h, "none", "rms")
    run_norm(eng, a, None, None, a, "none", "rms")
    torch.cuda.synchronize()
    assert torch.equal(a, h)


# --- activations -------------------------------------------------------------

# Down to where the factor of g still has float32's whole precision (2^-126).
LOWEST = {"silu": -86.0, "gelu": -12.5, "gelu_tanh": -9.9, "relu": -40.0, "sigmoid": -86.0}


def far_activation_want(name, g):
    """(act(g), its error) for exact g, relative to act(g) where g is negative."""
    if name == "gelu_tanh":  # without the cancellation of 1 + tanh
        inner = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        want = g * torch.sigmoid(inner)
        return want, 1.1 * want.abs() * (6 * inner.abs() + 9) * F
    if name != "gelu":
        return activation_want(name, g, torch.zeros_like(g))
    # Half of erfc: the polynomial's 2.6 F near 0, up to 300 times as much (780 F) where erfc
    # is small; its argument 1 / (1 + c |g|) to 3 F, which the polynomial and its factor
    # pass on up to 2.3 times; five steps with their coefficients 5 F; e^(-g^2 / 2) to 2 F
    # and, of the three roundings of its argument, 1.5 g^2 F; two products. Then the last sum.
    less = g.abs() * 0.5 * torch.special.erfc(g.abs() / math.sqrt(2))
    want = g.clamp_min(0) - less
    return want, 1.1 * less * (2.6 * (1 / torch.special.erfc(g.abs() / math.sqrt(2))).clamp_max(300) + 16 + 1.5 * g * g) * F + F * want.abs()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("rows", [3, 300])
def test_activations_far_from_zero(eng, t, activation, bits, rows):
    # Sums of nothing but the bias, with an up projection that brings what is left of
    # a negative g back into the type's range.
    dt = TYPES[t][1]
    outputs, inputs = 1000, 64
    gate_bias = torch.cat([torch.linspace(LOWEST[activation], -0.01, 800, device="cuda"), torch.linspace(0.01, 30, 200, device="cuda")])
    want, e = far_activation_want(activation, gate_bias.double())
    up_bias = (1 / want.clamp_min(1e-30) if activation == "relu" else 1 / want).clamp(-1e37, 1e37).float()
    up_bias[want == 0] = 1.0
    x = normal(gen(rows), dt, rows, inputs)
    out = torch.empty(rows, outputs, dtype=dt, device="cuda")
    if bits == 4:
        codes, scales = (torch.zeros(outputs, n, dtype=torch.uint8, device="cuda") for n in (32, 16))
        run_gated(eng, x, codes, codes, gate_bias, up_bias, out, activation, (scales, scales))
    else:
        none = torch.zeros(outputs, inputs, dtype=dt, device="cuda")
        run_gated(eng, x, none, none, gate_bias, up_bias, out, activation)
    torch.cuda.synchronize()
    e = e * up_bias.double().abs()
    want = want * up_bias.double()
    within(out, want.expand(rows, outputs), (e + F * want.abs()).expand(rows, outputs), dt)


# --- routes ------------------------------------------------------------------

@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("post,pre", [("none", "layer"), ("rms", "rms"), ("layer", "layer"), ("rms", "none")])
@pytest.mark.parametrize("lengths,channels,which", [([5, 0, 2], 8200, 31), ([3], 12288, 5), ([1, 4], 16384, 26), ([3], 16392, 31),
                                                    ([2, 2], 20000, 31), ([3], 32760, 21)])
def test_norm_of_several_pieces_per_lane(eng, t, wide, post, pre, lengths, channels, which):
    # Two and four pieces, the last of which some lanes lack.
    packed_feed_forward.test_norm(eng, t, wide, post, pre, lengths, channels, which)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", ["gated4", "linear4"])
@pytest.mark.parametrize("rows,inputs,outputs", [(100, 1000, 1200), (40, 1504, 3000), (5, 2000, 9000), (3, 4096, 9000)])
def test_few_rows_walk_several_outputs(eng, t, kind, rows, inputs, outputs):
    # Each form of the few-rows kernel whose workgroups take a further block of outputs:
    # 32 rows in steps of 4 and 8 blocks, 16 rows in steps of 8 and 16.
    packed_block.test_routes(eng, t, kind, rows, inputs, outputs)
