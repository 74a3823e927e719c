"""GPU tests of compact rows with row pitches up to and past what 32-bit offsets inside a tile allow: the kernels' last
pitch, the first one that takes the other way, and the refusals.

Whole numbers, exact sums.  What lies between the rows is not written: it is whatever the memory held."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    return torch


def _whole(n, d, fmt, seed):
    torch = _torch()
    from vittles_amd import compact
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table = torch.tensor([0.0, 1.0, -1.0, 2.0, -2.0, 3.0, -3.0, 4.0, -4.0, 6.0, -6.0], dtype=torch.float64, device="cuda")
    x = table[torch.randint(0, 11, (n, d), generator=gen, device="cuda")]
    X = compact.quantise(x, fmt)
    assert torch.equal(X.dequantise(torch.float64), x)
    return X, x


def _pitched(t, pitch, first=0):
    """``t`` as a view of rows ``pitch`` elements apart."""
    torch = _torch()
    wide = torch.empty((t.shape[0] * pitch + first,), dtype=t.dtype, device="cuda")
    view = wide[first:].as_strided(t.shape, (pitch, 1))
    view.copy_(t)
    return view


def _rows(X, ldc, lds):
    from vittles_amd import compact
    Y = compact.CompactRows(_pitched(X.codes, ldc), _pitched(X.scales, lds), X.D, X.format)
    assert Y.codes.stride(0) == ldc and Y.scales.stride(0) == lds
    return Y


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("n,d", [(300, 5), (70, 900), (50, 5003), (20, 16400)])
@pytest.mark.parametrize("ldc,lds", [((1 << 22) - 16, (1 << 22) - 1), (1 << 22, 600), (4200000 // 16 * 16, 1 << 22), (1 << 26, 600)])
def test_row_operators(n, d, fmt, ldc, lds):
    torch = _torch()
    from vittles_amd import rows
    X, x = _whole(n, d, fmt, n + d)
    X = _rows(X, ldc, lds)
    whole = lambda m: torch.randint(-3, 4, (m,), device="cuda").to(torch.float64)
    v, u = whole(d), whole(n)
    assert torch.equal(X.dequantise(torch.float64), x)
    assert torch.equal(rows.gemv(X, v), x @ v)
    assert torch.equal(rows.gemv_t(X, u), x.t() @ u)
    assert torch.equal(rows.glm_hvp(X, u, v), x.t() @ (u * (x @ v)))


# the last pitches that tiles take and the first ones past them: codes, scales, result
@pytest.mark.parametrize("ldc,lds,out", [((1 << 23) - 16, (1 << 23) - 4, 0), ((1 << 23) - 16, (1 << 23) - 3, 0), (2064, 1 << 23, 0),
                                         (1 << 23, 68, 0), (2064, 68, (1 << 24) - 64), (2064, 68, (1 << 24) - 1), (2064, 68, 1 << 24)])
def test_gemm_nt(ldc, lds, out):
    torch = _torch()
    from vittles_amd import rows
    m, n, k = 600, 1300, 2050
    A, a = _whole(m, k, "mxfp4", 1)
    B, b = _whole(n, k, "mxfp4", 2)
    A = _rows(A, ldc, lds)
    ref = a @ b.t()
    for dtype in (torch.float32, torch.bfloat16):
        C = _pitched(torch.zeros((m, n), dtype=dtype, device="cuda"), out or n)
        rows.gemm_nt(A, B, out=C)
        assert torch.equal(C, ref.to(dtype))
    # the other side
    if not out:
        assert torch.equal(rows.gemm_nt(B, A), ref.t().float())


# 128 x 64 and 256 x 256 tiles (up to 87 GB of address range, of which the rows are touched)
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("n,da,db", [(70, 300, 65), (2600, 1200, 301)])
@pytest.mark.parametrize("which", ["codes", "scales", "B", "out"])
def test_gemm_tn(n, da, db, fmt, which):
    torch = _torch()
    from vittles_amd import rows
    from vittles_amd._lib import VittlesHipError
    X, x = _whole(n, da, fmt, 3)
    for kind in (torch.bfloat16, torch.float16, torch.float32):
        g = torch.randint(-200, 201, (n, db), device="cuda").to(kind)
        ref = (x.t() @ g.double()).float()
        for limit in (False, True):
            Y, h, C = X, g, torch.zeros((da, db), device="cuda")
            if which == "codes":
                Y = _rows(X, (1 << 25) - (0 if limit else 16), X.scales.shape[1])
            elif which == "scales":
                Y = _rows(X, X.codes.shape[1], (1 << 25) - (0 if limit else 1))
            elif which == "B":
                h = _pitched(g, (1 << 23) - (0 if limit else 1), first=1)
            else:
                C = _pitched(C, (1 << 24) - (0 if limit else 1))
            if limit:
                with pytest.raises(VittlesHipError, match="not supported"):
                    rows.gemm_tn(Y, h, out=C)
            else:
                assert torch.equal(rows.gemm_tn(Y, h, out=C), ref)
            del Y, h, C
