"""The operators on packed batches at edges of their definitions, against
float64: rotations of heads' first channels where 16-byte pieces do not fit.
Tolerances as in packed_operators.py."""
import pytest

torch = pytest.importorskip("torch")

import dinov3_hrx as d  # noqa: E402

from packed_operators import F, TYPES, gen, normal, run_rotation, within  # noqa: E402

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
