"""GPU tests of compact rows at the largest sizes: more rows or columns than the threads of one launch."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    return torch


@pytest.mark.parametrize("side", ["rows of A", "rows of B"])
def test_gemm_nt_more_rows_than_a_launch_holds(side):
    """2^28 + 21 rows against three: one block of 32 columns each.  The codes stand for whole numbers whose sums stay
    below 2^24: products are exact in float, and the bfloat16 result is their one rounding."""
    torch = _torch()
    from vittles_amd import compact, rows
    many, few, d = (1 << 28) + 21, 3, 32
    gen = torch.Generator(device="cuda").manual_seed(5)
    # an even E2M1 index is 0, 1, 2 or 4: whole numbers in both halves of a byte
    codes = torch.randint(0, 256, (many, 16), generator=gen, dtype=torch.uint8, device="cuda").bitwise_and_(0xEE)
    scales = torch.randint(126, 130, (many, 1), generator=gen, dtype=torch.uint8, device="cuda").add_(1)
    long = compact.CompactRows(codes, scales, d, "mxfp4")
    short = compact.CompactRows(codes[7:7 + few].clone(), scales[7:7 + few].clone(), d, "mxfp4")
    short_values = short.dequantise(torch.float64)
    if side == "rows of B":
        bias = (torch.arange(many, device="cuda") % 251).to(torch.float32)
        out = torch.full((few, many), float("nan"), dtype=torch.bfloat16, device="cuda")
        rows.gemm_nt(short, long, bias=bias, out=out)
    else:
        bias = torch.tensor([1.0, -2.0, 5.0], device="cuda")
        out = torch.full((many, few), float("nan"), dtype=torch.bfloat16, device="cuda")
        rows.gemm_nt(long, short, bias=bias, out=out)
    # the rows around every border of the launches, and a stretch of the others
    for lo in (0, (1 << 27) - 40, (1 << 28) - 40, 3 << 26, many - 60):
        part = slice(lo, min(many, lo + 100))
        x = compact.CompactRows(codes[part], scales[part], d, "mxfp4").dequantise(torch.float64)
        if side == "rows of B":
            want, got = short_values @ x.t().contiguous() + bias[part].double(), out[:, part]
        else:
            want, got = x @ short_values.t().contiguous() + bias.double(), out[part]
        assert float(want.abs().max()) < 1 << 24
        assert torch.equal(got, want.to(torch.bfloat16)), lo
    assert not bool(torch.isnan(out).any())


def test_row_operators_more_columns_than_a_launch_holds():
    """Two rows of 2^27 + 37 columns: whole numbers, exact sums."""
    torch = _torch()
    from vittles_amd import compact, rows
    n, d = 2, (1 << 27) + 37
    nb = (d + 31) // 32
    gen = torch.Generator(device="cuda").manual_seed(6)
    codes = torch.randint(0, 256, (n, nb * 16), generator=gen, dtype=torch.uint8, device="cuda").bitwise_and_(0xEE)
    codes[:, (d - 1) // 2 + 1:] = 0                       # the columns behind the last one
    codes[:, (d - 1) // 2] &= 0x0F
    scales = torch.randint(127, 131, (n, nb), generator=gen, dtype=torch.uint8, device="cuda")
    X = compact.CompactRows(codes, scales, d, "mxfp4")
    x = X.dequantise(torch.float64)
    u = torch.tensor([3.0, -2.0], dtype=torch.float64, device="cuda")
    assert torch.equal(rows.gemv_t(X, u), 3.0 * x[0] - 2.0 * x[1])
    v = torch.randint(-2, 3, (d,), generator=gen, device="cuda").to(torch.float64)
    z = torch.stack([(x[0] * v).sum(), (x[1] * v).sum()])
    assert torch.equal(rows.gemv(X, v), z)
    prior = torch.randint(1, 4, (d,), generator=gen, device="cuda").to(torch.float64)
    assert torch.equal(rows.glm_hvp(X, u, v, prior=prior), x[0] * (3.0 * z[0]) + x[1] * (-2.0 * z[1]) + prior * v)


@pytest.mark.parametrize("fmt,border,below", [("mxfp8", 1.9375, 1.875), ("mxfp4", 1.75, 1.5)])
def test_numbers_that_round_to_the_first_power_past_float(fmt, border, below):
    """The largest numbers of float: those below the border keep a value, the others have a code that stands for 2^128 and
    read as infinities of their sign; the rest of the block is as it was."""
    import numpy as np
    torch = _torch()
    from vittles_amd import compact, rows
    p = 2.0 ** 127
    last = float(np.nextafter(np.float32(border * p), np.float32(0)))
    x = torch.tensor([[last, -last, 2.0 ** 125], [border * p, -border * p, 2.0 ** 125]], dtype=torch.float64, device="cuda")
    inf = float("inf")
    want = torch.tensor([[below * p, -below * p, 2.0 ** 125], [inf, -inf, 2.0 ** 125]], dtype=torch.float64, device="cuda")
    for dtype in (torch.float64, torch.float32):
        X = compact.quantise(x.to(dtype), fmt)
        assert torch.equal(X.dequantise(torch.float64), want) and torch.equal(X.dequantise(), want.float())
        assert torch.equal(rows.gemv(X, torch.tensor([1.0, 0.0, 0.0], dtype=torch.float64, device="cuda"))[:1], want[:1, 0])
