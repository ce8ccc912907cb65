"""The operators of the feed-forward half of a packed block at edges of their
definitions: float32 rows of one value. Tolerances as in packed_feed_forward.py."""
import pytest

torch = pytest.importorskip("torch")

import dinov3_hrx as d  # noqa: E402

from packed_feed_forward import norm_want, run_norm  # noqa: E402
from packed_operators import F, TYPES, gen, within  # noqa: E402

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
