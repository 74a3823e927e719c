"""GPU tests of the row operators of compact rows where every workgroup takes several rounds of rows, the last one ragged.

All numbers are whole (the rows', the vectors', the weights'; gaussian family) and their sums stay below 2^53: every order of
a sum gives the same double, so results are equal to the last bit.  The logistic link is compared to 1e-12, the rounding of
its 64-bit formula."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    return torch


# Rows past three rounds of the largest grid that any operator takes on 256 CUs.  2 to 64 lanes of a wave; 128, 256 and 512
# threads with one piece (for operators without column sums: 2, 3 and 5 waves); two and three pieces; two passes.
SHAPES = [(270001, 5), (280003, 50), (140001, 100), (70001, 200), (35003, 400), (17003, 900), (17011, 1030), (11003, 2049),
          (7001, 5003), (2501, 8200), (2503, 16400), (16501, 20400)]


@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_row_operators_in_several_rounds(n, d, fmt):
    torch = _torch()
    import vittles_amd as va
    from vittles_amd import rows
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    whole = lambda low, high, *size: torch.randint(low, high, size, generator=gen, device="cuda").to(torch.float64)
    # magnitudes that E2M1 and E4M3 both hold, times 1, 2, 4 or 8 by row
    table = torch.tensor([0.0, 0.0, 1.0, -1.0, 2.0, -2.0, 3.0, -3.0, 4.0, -4.0, 6.0, -6.0], dtype=torch.float64, device="cuda")
    x = table[torch.randint(0, 12, (n, d), generator=gen, device="cuda")] * 2.0 ** whole(0, 4, n, 1)
    X = va.compact.quantise(x, fmt)
    assert torch.equal(X.dequantise(torch.float64), x)
    v, u1, u2, w, y = whole(-3, 4, d), whole(-3, 4, n), whole(-2, 3, n), whole(0, 4, n), whole(-5, 6, n)
    prior, off = whole(1, 5, d), whole(-9, 10, n)
    xt = x.t()

    def down(c):                  # whole numbers: exact, and so are the sums of their magnitudes that bound every partial sum
        assert float((xt.abs() @ c.abs()).max()) < 2.0 ** 53
        return xt @ c

    z = x @ v
    assert torch.equal(rows.gemv(X, v), z)
    assert torch.equal(rows.gemv_t(X, u1), down(u1))
    assert torch.equal(rows.gemv_t2(X, u1, u2), down(u1 * u2))
    assert torch.equal(rows.glm_hvp(X, w, v, prior=prior), down(w * z) + prior * v)
    obj = va.WeightedGLMObjective(X, y, family="gaussian", offset=off)
    l1 = z + off - y
    got_z, r, dd = rows.glm_link(obj, v, w, want_z=True)
    assert torch.equal(got_z, z + off) and torch.equal(r, l1) and torch.equal(dd, w)
    g, r, dd = rows.glm_grad(obj, v, w, prior=prior)
    assert torch.equal(g, down(w * l1) + prior * v) and torch.equal(r, l1) and torch.equal(dd, w)
    loss = w * l1 * l1                # halved: a multiple of 1/2
    assert float(loss.sum()) < 2.0 ** 52
    assert rows.glm_value(obj, v, w) == 0.5 * float(loss.sum())
    theta = v / (8.0 * d ** 0.5)
    z = x @ theta
    obj = va.WeightedGLMObjective(X, (y > 0).to(torch.float64), family="logistic")
    _, r, dd = rows.glm_link(obj, theta, w)
    p = torch.sigmoid(z)
    assert float((r - (p - obj.y)).abs().max()) < 1e-12
    assert float((dd - w * p * torch.sigmoid(-z)).abs().max()) < 1e-12
