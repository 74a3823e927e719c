"""GPU tests of the products of compact rows: every tile and split of them, with operands and results at any offset and pitch.

The reference is the fp64 product of the stored values.  A sum of L exact products in float32 is off by at most L roundings
of 2^-24 of the sum of their magnitudes; the matrix instruction may add in any order and cut instead of round, which doubles
the bound: L 2^-23 sum |a b|; the result's own rounding adds 2^-24 (float32) or 2^-8 (bfloat16) of it."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    return torch


def _rows(n, d, fmt, seed, shifted):
    """Compact rows and their values in fp64; ``shifted``: views into wider codes and scales, scales at an odd address."""
    torch = _torch()
    from vittles_amd import compact
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, d), generator=g, device="cuda") * torch.exp(torch.randn((n, 1), generator=g, device="cuda"))
    x[::5, : d // 2] = 0.0
    X = compact.quantise(x, fmt)
    if shifted:
        nb, width = X.scales.shape[1], X.codes.shape[1]
        codes = torch.full((n, width + 48), 0x77, dtype=torch.uint8, device="cuda")
        scales = torch.full((n, nb + 4), 255, dtype=torch.uint8, device="cuda")       # NaN around what is read
        codes[:, 16:16 + width] = X.codes
        scales[:, 1:1 + nb] = X.scales
        X = compact.CompactRows(codes[:, 16:16 + width], scales[:, 1:1 + nb], d, fmt)
        assert X.codes.data_ptr() == codes.data_ptr() + 16 and X.scales.data_ptr() == scales.data_ptr() + 1
    return X, X.dequantise(torch.float64)


# few rows in several blocks, 128 x 128 tiles, 256 x 256 tiles, a split axis
@pytest.mark.parametrize("m,n,k", [(70, 65, 33), (151, 219, 563), (1100, 1201, 1056), (4000, 4090, 130), (512, 500, 8190)])
@pytest.mark.parametrize("shifted", [False, True])
def test_gemm_nt_tiles(m, n, k, shifted):
    torch = _torch()
    from vittles_amd import rows
    A, a = _rows(m, k, "mxfp4", 1, shifted)
    B, b = _rows(n, k, "mxfp4", 2, shifted)
    ref, bound = a @ b.t(), k * 2.0 ** -23 * (a.abs() @ b.abs().t())
    bias = torch.linspace(-1, 1, n, device="cuda")
    # rows of the result on whole lines, or between guards at an odd pitch
    pitch, off = ((n + 63) // 64 * 64, 0) if not shifted else (n + 3, 1)
    for dtype, step in ((torch.float32, 2.0 ** -24), (torch.bfloat16, 2.0 ** -8)):
        buf = torch.full((m + 1, pitch), 7.0, dtype=dtype, device="cuda")
        out = buf[:m, off:off + n]
        rows.gemm_nt(A, B, alpha=0.5, bias=bias, out=out)
        want = 0.5 * ref + bias.double()
        err = (out.double() - want).abs()
        assert bool((err <= 0.5 * bound + (2.0 ** -24 + step) * (want.abs() + bound)).all())
        assert bool((buf[m] == 7).all() and (buf[:, :off] == 7).all() and (buf[:, off + n:] == 7).all())


# 128 x 64, 256 x 128 and 256 x 256 tiles
@pytest.mark.parametrize("n,da,db", [(35, 1156, 217), (16384, 1000, 99), (8200, 500, 301)])
@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shifted", [False, True])
def test_gemm_tn_tiles(n, da, db, kind, shifted):
    torch = _torch()
    from vittles_amd import rows
    for fmt in ("mxfp8", "mxfp4"):
        X, x = _rows(n, da, fmt, 3, shifted)
        wide = torch.full((n, (db + 15) // 8 * 8), float("nan"), dtype=getattr(torch, kind), device="cuda")
        g = wide[:, 1:db + 1] if shifted else wide[:, :db]      # in 16-byte pieces or at the element's own alignment
        g.copy_(torch.randn((n, db), device="cuda"))
        w = torch.rand(n, dtype=torch.float64, device="cuda")
        for scale in (None, w):
            gs = g.double() if scale is None else w[:, None] * g.double()
            ref, bound = x.t() @ gs, (n + 2) * 2.0 ** -23 * (x.abs().t() @ gs.abs()) + 2.0 ** -126 * n
            got = rows.gemm_tn(X, g, rowscale=scale)
            assert bool(((got.double() - ref).abs() <= bound + 2.0 ** -24 * ref.abs()).all())


def test_gemm_tn_single_row_has_no_stride():
    """The pitch of a matrix of one row says nothing: no row behind it is read through it."""
    torch = _torch()
    from vittles_amd import _lib, compact, device as dev
    X = compact.quantise(torch.ones((1, 40), device="cuda"), "mxfp8")
    B = torch.tensor([[1.0, float("inf"), 2.0, 3.0]], device="cuda")
    C, lib = torch.zeros((40, 4), device="cuda"), _lib.load()
    nbytes = lib.vt_mx_gemm_tn_workspace_bytes(1, 40, 4)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    for ldb in (4, 1 << 29, 1 << 30, (1 << 30) + 1, 1 << 40):
        C.zero_()
        _lib.check(lib.vt_mx_gemm_tn(X.c_format(), *X.c_args(), 40, compact.TYPE[B.dtype], B.data_ptr(), ldb, 4, 0, 1, 1.0, 0,
                                     C.data_ptr(), 4, ws.data_ptr(), nbytes, dev.stream_ptr()), "vt_mx_gemm_tn")
        assert torch.equal(C, B.expand(40, 4))


def test_objective_and_panels_take_compact_rows_as_they_are():
    torch = _torch()
    import vittles_amd as va
    from vittles_amd import rows
    X = va.compact.quantise(torch.randn((50, 70), device="cuda"), "mxfp8")
    y = torch.zeros(50, dtype=torch.float64, device="cuda")
    for device in ("cuda", X.device, str(X.device), None):
        assert va.WeightedGLMObjective(X, y, family="gaussian", device=device).X is X
    for device in ("cpu", "cuda:%d" % (X.device.index + 1)):
        with pytest.raises(ValueError):
            va.WeightedGLMObjective(X, y, family="gaussian", device=device)
    g = torch.randn((50, 9), device="cuda")
    assert torch.equal(rows.gemm_tn_tiled(X, g, tile=32), rows.gemm_tn(X, g))


@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("n,da,db,start", [(1000, 64, 33, 1), (1000, 64, 33, 0), (127, 40, 301, 1), (1, 40, 5, 3), (9000, 300, 129, 1)])
def test_gemm_tn_rows_that_share_a_word(kind, n, da, db, start):
    """Odd rows without a gap: what lies before the first row, behind the last one and in the next slab's first row shares
    a word with a row that is read, and must not reach the result, not as 0 * inf either."""
    torch = _torch()
    from vittles_amd import compact, rows
    X = compact.quantise(torch.ones((n, da), device="cuda"), "mxfp8")
    flat = torch.full((n * db + 8,), float("nan"), dtype=getattr(torch, kind), device="cuda")
    g = flat[start:start + n * db].view(n, db)
    g.fill_(1.0)
    for scale in (None, torch.ones(n, dtype=torch.float64, device="cuda")):
        g.fill_(1.0)
        assert torch.equal(rows.gemm_tn(X, g, rowscale=scale), torch.full((da, db), float(n), device="cuda"))
        g[::64, 0] = float("inf")           # the first rows of all slabs among them
        want = torch.full((da, db), float(n), device="cuda")
        want[:, 0] = float("inf")
        assert torch.equal(rows.gemm_tn(X, g, rowscale=scale), want)
