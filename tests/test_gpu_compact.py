"""GPU tests of compact rows (microscaled 8-bit and 4-bit storage) against plain 64-bit implementations.

Tolerances, all derived from the arithmetic:
  * quantisation and reading back are exact: bits and values are equal.
  * row operators carry every sum in fp64: 1e-12 of the largest result, as in the fp32 storage mode's tests.
  * products are sums of L exact products in float32: a sum of L terms is off by at most L roundings of 2^-24 of the sum
    of their magnitudes; the matrix instruction may add in any order and cut instead of round, which doubles the bound:
    L 2^-23 sum |a b|, plus the result's own rounding."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EXACT = 1e-12
FORMATS = ("mxfp8", "mxfp4")


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    return torch


def _data(n, d, seed):
    """Rows of unequal size with outlier columns, empty rows and empty blocks."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, d)) * np.exp(rng.standard_normal(d)) * np.exp(2 * rng.standard_normal((n, 1)))
    x[:, rng.random(d) < 0.02] *= 50
    x[rng.random(n) < 0.1] = 0.0
    if d > 40:
        x[::3, 32:64] = 0.0
    return x


def _compact(x, fmt):
    import vittles_amd as va
    torch = _torch()
    return va.compact.quantise(torch.as_tensor(x, device="cuda"), fmt)


def _codes(X):
    """One code per column, on the host."""
    c = X.codes.cpu().numpy()
    return c if X.format == "mxfp8" else np.stack([c & 15, c >> 4], axis=-1).reshape(c.shape[0], -1)


@pytest.mark.parametrize("n,d", [(1, 1), (3, 31), (5, 32), (7, 33), (2, 100), (300, 257), (1000, 129), (65, 2049), (1, 20000),
                                 (70000, 5)])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kind", ["float64", "float32", "bfloat16", "float16"])
def test_quantise_and_read_back(n, d, fmt, kind):
    torch = _torch()
    from oracle import compact as oc
    # float16: small enough for its range, down into its subnormals
    x = torch.as_tensor(_data(n, d, seed=n + d) * (1e-4 if kind == "float16" else 0.1), device="cuda").to(getattr(torch, kind))
    assert bool(torch.isfinite(x).all())
    X = _compact(x, fmt)
    codes, scales = oc.quantise(x.double().cpu().numpy(), fmt)
    assert X.shape == (n, d) and np.array_equal(X.scales.cpu().numpy(), scales)
    assert np.array_equal(_codes(X), codes)
    v = oc.values(codes, scales, d, fmt)
    assert np.array_equal(X.dequantise().cpu().numpy(), v)
    assert np.array_equal(X.dequantise(torch.float64).cpu().numpy(), v)
    for t in (torch.bfloat16, torch.float16):
        assert torch.equal(X.dequantise(t).cpu(), torch.as_tensor(v).to(t))
    # what was stored reads the same after a second quantisation of the values (they are on the grid)
    assert torch.equal(_compact(X.dequantise(torch.float64), fmt).dequantise(), X.dequantise())


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantise_ties_and_edges(fmt):
    """Every code, every middle between two codes and its neighbours, at three scales, in fp64 (one rounding: a middle plus
    2^-60 is not a tie) and in fp32."""
    torch = _torch()
    from oracle import compact as oc
    grid = np.append(oc.GRID[fmt], oc.NEXT[fmt])
    mid = (grid[1:] + grid[:-1]) / 2
    # another name for the block's largest magnitude, so that it fixes the scale of the other 31
    for dtype, eps in ((torch.float64, 2.0 ** -50), (torch.float32, 2.0 ** -22)):
        pts = np.concatenate([grid[:-1], mid[:-1], mid[:-1] * (1 + eps), mid[:-1] * (1 - eps)])
        pts = np.concatenate([pts, -pts])
        rows = np.zeros((-(-len(pts) // 31), 32))
        rows[:, 0] = grid[-2]
        flat = np.zeros(rows.shape[0] * 31)
        flat[:len(pts)] = pts
        rows[:, 1:] = flat.reshape(-1, 31)
        tops = np.concatenate([mid[-1:] * f for f in (1, 1 + eps, 1 - eps)])
        rows = np.concatenate([rows, np.pad(tops[:, None], ((0, 0), (0, 31)))])
        for p in (0, -40, 90):
            x = torch.as_tensor(np.ldexp(rows, p)).to(dtype).cuda()
            X = _compact(x, fmt)
            codes, scales = oc.quantise(x.double().cpu().numpy(), fmt)
            assert np.array_equal(X.scales.cpu().numpy(), scales)
            assert np.array_equal(_codes(X), codes)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantise_extremes(fmt):
    torch = _torch()
    from oracle import compact as oc
    f = np.float32
    big, tiny = float(np.finfo(f).max), 2.0 ** -149
    rows = np.zeros((12, 70))
    rows[0, :3] = big, -big, 1.0
    rows[1, :3] = tiny, -tiny, 0.0
    rows[2, :2] = 2.0 ** -126, 2.0 ** -130
    rows[3, 40] = np.inf
    rows[4, 5] = np.nan
    rows[5, 69] = -np.inf
    rows[6] = -0.0
    rows[7, :2] = 1.0, -1e-30
    rows[8, 64:] = 3e38
    for dtype in (torch.float32, torch.float64):
        if dtype == torch.float64:
            rows[9, 0] = 1e300                        # beyond float: the block cannot be stored
            rows[10, 0] = oc.FLT_EDGE                 # the first number that rounds past the largest float
            rows[11, :2] = np.nextafter(oc.FLT_EDGE, 0), 5e-324
        x = torch.as_tensor(rows).to(dtype).cuda()
        X = _compact(x, fmt)
        codes, scales = oc.quantise(x.double().cpu().numpy(), fmt)
        assert np.array_equal(X.scales.cpu().numpy(), scales)
        assert np.array_equal(_codes(X), codes)
        with np.errstate(over="ignore"):
            v = oc.values(codes, scales, 70, fmt).astype(f).astype(np.float64)
        assert np.array_equal(X.dequantise(torch.float64).cpu().numpy(), v, equal_nan=True)


def test_quantise_layouts():
    """Column slices, transposed and broadcast inputs, bases off 16 bytes, numpy and CPU tensors."""
    torch = _torch()
    import vittles_amd as va
    base = torch.randn((40, 300), device="cuda")
    for dtype in (torch.float32, torch.bfloat16, torch.float64):
        b = base.to(dtype)
        views = [b[:, 3:200], b[1:, 16:], b[::2, 64:128], b.t(), b[:1].expand(7, 300), b[:, :1], b[5:5], b[:, 8:136]]
        for x in views:
            X = va.compact.quantise(x, "mxfp8")
            Y = va.compact.quantise(x.contiguous().clone(), "mxfp8")
            assert X.shape == tuple(x.shape) and torch.equal(X.codes, Y.codes) and torch.equal(X.scales, Y.scales)
    a = va.compact.quantise(base.double().cpu().numpy(), "mxfp4")
    for other in (base.cpu(), base.double(), base):
        assert torch.equal(va.compact.quantise(other, "mxfp4").codes, a.codes)
    # codes and scales handed in, in layouts that the kernels do not take as they are
    X = va.compact.quantise(base, "mxfp8")
    wide = torch.zeros((40, X.codes.shape[1] + 7), dtype=torch.uint8, device="cuda")
    wide[:, 7:] = X.codes
    Y = va.compact.CompactRows(wide[:, 7:], X.scales.t().contiguous().t(), 300)
    assert torch.equal(Y.dequantise(), X.dequantise())
    Z = va.compact.CompactRows(X.codes[10:20], X.scales[10:20], 300)
    assert torch.equal(Z.dequantise(), X.dequantise()[10:20])
    with pytest.raises(TypeError):
        va.compact.quantise(torch.zeros((2, 2), dtype=torch.int32, device="cuda"))
    for bad in (torch.zeros(3, device="cuda"), torch.zeros((3, 0), device="cuda")):
        with pytest.raises(ValueError):
            va.compact.quantise(bad)
    with pytest.raises(TypeError):
        X.dequantise(torch.int8)


# (rows, columns): widths from one column past every team size, counts around the batches of rows
SHAPES = [(1, 1), (2, 5), (3, 31), (5, 32), (17, 33), (64, 64), (1000, 20), (257, 100), (4099, 128), (500, 129), (301, 255),
          (70, 513), (33, 1000), (129, 1025), (40, 2047), (13, 2049), (9, 4096), (21, 4097), (7, 8191), (11, 8193), (5, 12300),
          (37, 16385), (6, 20000), (3, 20449), (2, 40001), (30011, 7)]


@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_row_operators(n, d, fmt, relerr):
    torch = _torch()
    from oracle import compact as oc, glm
    import vittles_amd as va
    from vittles_amd import rows
    rng = np.random.default_rng(n + 7 * d)
    x = rng.standard_normal((n, d)) * np.exp(0.5 * rng.standard_normal(d))
    xs = oc.store(x, fmt)
    X = _compact(x, fmt)
    v, u1, u2 = rng.standard_normal(d), rng.standard_normal(n), rng.standard_normal(n)
    t = lambda a: torch.as_tensor(a, device="cuda")
    c = lambda a: a.cpu().numpy()
    prior = np.linspace(0.5, 2.0, d)
    dd = rng.random(n)
    dd[::4] = 0.0
    assert relerr(c(rows.gemv(X, t(v))), xs @ v) < EXACT
    assert relerr(c(rows.gemv_t(X, t(u1))), xs.T @ u1) < EXACT
    assert relerr(c(rows.gemv_t2(X, t(u1), t(u2))), xs.T @ (u1 * u2)) < EXACT
    hv = xs.T @ (dd * (xs @ v))
    assert relerr(c(rows.glm_hvp(X, t(dd), t(v))), hv) < EXACT
    assert relerr(c(rows.glm_hvp(X, t(dd), t(v), prior_scalar=2.5)), hv + 2.5 * v) < EXACT
    out = torch.full((d,), float("nan"), dtype=torch.float64, device="cuda")
    assert rows.glm_hvp(X, t(dd), t(v), prior=t(prior), out=out) is out
    assert relerr(c(out), hv + prior * v) < EXACT
    theta = v / np.sqrt(3 * d)
    w = 0.5 + rng.random(n)
    w[::5] = 0.0
    y = (rng.random(n) < 0.5).astype(float)
    for family in ("logistic", "poisson", "gaussian"):
        off = None if family == "poisson" else 0.1 * rng.standard_normal(n)
        obj = va.WeightedGLMObjective(X, y, family=family, prior=prior, scale=1.5, offset=off)
        assert obj.dtype == fmt and (obj.N, obj.D) == (n, d)
        z = glm.linear_predictor(xs, theta, off)
        ell, l1, l2 = glm.link(family, z, y)
        zz, r, d2 = rows.glm_link(obj, theta, w, want_z=True)
        assert relerr(c(zz), z) < EXACT and relerr(c(r), 1.5 * l1) < EXACT and relerr(c(d2), 1.5 * w * l2) < EXACT
        g, r, d2 = rows.glm_grad(obj, theta, w, prior=obj.prior)
        ref = glm.grad(family, xs, y, theta, w, prior, 1.5, off)
        assert relerr(c(g), ref) < EXACT and relerr(c(r), 1.5 * l1) < EXACT and relerr(c(d2), 1.5 * w * l2) < EXACT
        assert relerr(c(obj.grad(theta, w)), ref) < EXACT
        val = glm.value(family, xs, y, theta, w, prior, 1.5, off)
        assert abs(obj.value(theta, w) - val) < EXACT * max(1.0, 1.5 * np.abs(w * ell).sum())


@pytest.mark.parametrize("fmt", FORMATS)
def test_row_operators_repeat_bit_for_bit_and_leave_no_trace(fmt):
    torch = _torch()
    from vittles_amd import rows
    X = _compact(_data(3001, 777, 3), fmt)
    d = torch.rand(3001, dtype=torch.float64, device="cuda")
    v = torch.randn(777, dtype=torch.float64, device="cuda")
    first = rows.glm_hvp(X, d, v)
    junk = rows.glm_hvp(_compact(_data(50, 5000, 4), fmt), d[:50], torch.randn(5000, dtype=torch.float64, device="cuda"))
    assert torch.equal(rows.glm_hvp(X, d, v), first) and bool(torch.isfinite(junk).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_row_operators_nan_stays_in_its_block(fmt):
    """A block that could not be stored poisons its row's dot and its own columns only, as the values say."""
    torch = _torch()
    from oracle import compact as oc
    from vittles_amd import rows
    x = np.random.default_rng(0).standard_normal((20, 100))
    x[7, 40] = np.inf
    X, xs = _compact(x, fmt), oc.store(x, fmt)
    v, u = np.ones(100), np.ones(20)
    z = rows.gemv(X, torch.as_tensor(v, device="cuda")).cpu().numpy()
    assert np.array_equal(np.isnan(z), np.isnan(xs @ v)) and np.isnan(z).sum() == 1
    s = rows.gemv_t(X, torch.as_tensor(u, device="cuda")).cpu().numpy()
    assert np.array_equal(np.isnan(s), np.isnan(xs.T @ u)) and np.isnan(s).sum() == 32


def test_row_operators_empty_and_refusals():
    torch = _torch()
    import vittles_amd as va
    from vittles_amd import rows
    from vittles_amd._lib import VittlesHipError
    X0 = _compact(np.zeros((0, 50)), "mxfp8")
    f = lambda *s: torch.ones(s, dtype=torch.float64, device="cuda")
    prior = 2 * f(50)
    assert X0.shape == (0, 50) and X0.dequantise().shape == (0, 50)
    assert rows.gemv(X0, f(50)).shape == (0,) and not rows.gemv_t(X0, f(0)).any()
    assert torch.equal(rows.glm_hvp(X0, f(0), f(50), prior=prior), prior)
    obj = va.WeightedGLMObjective(X0, np.zeros(0), prior=2.0)
    assert torch.equal(obj.grad(np.ones(50), np.zeros(0)), prior) and obj.value(np.ones(50), np.zeros(0)) == 50.0
    X = _compact(np.ones((10, 50)), "mxfp8")
    obj = va.WeightedGLMObjective(X, np.zeros(10), prior=1.0)
    for call in (lambda: rows.gemv(X, f(49)), lambda: rows.gemv(X, f(50).float()), lambda: rows.gemv(X, f(50).cpu()),
                 lambda: rows.gemv_t(X, f(11)), lambda: rows.glm_hvp(X, f(9), f(50)), lambda: rows.glm_hvp(X, f(10), f(51)),
                 lambda: rows.glm_hvp(X, f(10), f(50), out=f(49)), lambda: rows.glm_hvp(X, f(10), f(50), prior=f(1)),
                 lambda: obj.grad(f(49), f(10)), lambda: obj.value(f(50), f(9)),
                 lambda: va.WeightedGLMObjective(X, np.zeros(10), dtype=torch.float32),
                 lambda: va.WeightedGLMObjective(X, np.zeros(10), dtype="mxfp4"),
                 lambda: va.WeightedGLMObjective(X, np.zeros(9)),
                 lambda: va.WeightedGLMObjective(X, np.zeros(10), offset=np.zeros(3)).grad(f(50), f(10))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: obj.hessian(f(50), f(10)), lambda: obj.fused(f(50), f(10)), lambda: obj.cross_hessian(f(50), f(10)),
                 lambda: rows.glm_hvp_multi(X, f(10), f(2, 50)), lambda: va.optim.newton_glm(obj, f(10)),
                 lambda: va.HyperparameterSensitivityLinearApproximation(obj, f(50), f(10))):
        with pytest.raises(VittlesHipError, match="compact"):
            call()


@pytest.mark.parametrize("fmt", FORMATS)
def test_gradient_against_differences_of_the_value(fmt):
    """The value's central difference along a direction: off by h^2 / 6 of the third derivative (bounded by the sum of
    |x u|^3 w / 10 for the logistic loss, whose third derivative is under 0.1) and the value's rounding over h."""
    _torch()
    from oracle import compact as oc
    import vittles_amd as va
    rng = np.random.default_rng(5)
    n, d, h = 700, 90, 1e-4
    x = rng.standard_normal((n, d))
    y, w = (rng.random(n) < 0.5).astype(float), rng.random(n)
    obj = va.WeightedGLMObjective(x, y, prior=0.7, dtype=fmt)
    theta, u = 0.1 * rng.standard_normal(d), rng.standard_normal(d)
    g = obj.grad(theta, w).cpu().numpy()
    slope = (obj.value(theta + h * u, w) - obj.value(theta - h * u, w)) / (2 * h)
    bound = h * h / 6 * 0.1 * (w * np.abs(oc.store(x, fmt) @ u) ** 3).sum() + 1e-12 * obj.value(theta, w) / h
    assert abs(slope - g @ u) < bound


def _product_bound(a, b, length):
    return length * 2.0 ** -23 * (np.abs(a) @ np.abs(b)) + 1e-300


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 32), (3, 5, 31), (2, 300, 129), (16, 64, 128), (17, 65, 257), (1, 4099, 513),
                                   (33, 127, 1000), (128, 128, 128), (129, 257, 383), (200, 1, 640), (256, 256, 512), (257, 513, 260),
                                   (64, 2000, 4096), (1000, 70, 2049), (5, 33, 20000), (520, 390, 96)])
def test_gemm_nt(m, n, k):
    torch = _torch()
    from oracle import compact as oc
    from vittles_amd import rows
    a, b = _data(m, k, m + k), _data(n, k, n + 2 * k)
    A, B = _compact(a, "mxfp4"), _compact(b, "mxfp4")
    a, b = oc.store(a, "mxfp4"), oc.store(b, "mxfp4")
    ref, bound = a @ b.T, _product_bound(a, b.T, k)
    c = rows.gemm_nt(A, B)
    assert c.dtype == torch.float32 and (np.abs(c.cpu().numpy().astype(float) - ref) <= bound + 2.0 ** -24 * np.abs(ref)).all()
    bias = np.random.default_rng(1).standard_normal(n).astype(np.float32)
    out = torch.full((m, n + 3), 7.0, dtype=torch.bfloat16, device="cuda")[:, :n]
    assert rows.gemm_nt(A, B, alpha=-0.5, bias=torch.as_tensor(bias, device="cuda"), out=out) is out
    ref2 = -0.5 * ref + bias
    # alpha is a power of two; the float sum with the bias and the bfloat16 result round once each
    err = np.abs(out.float().cpu().numpy().astype(float) - ref2)
    assert (err <= 0.5 * bound + (2.0 ** -23 + 2.0 ** -8) * (np.abs(ref2) + bound)).all()


def test_gemm_nt_exact_integers_and_specials():
    """Codes whose products and sums are whole numbers below 2^24 come out exactly; a NaN block poisons its row alone."""
    torch = _torch()
    from vittles_amd import rows
    rng = np.random.default_rng(2)
    a, b = (rng.integers(-4, 5, (m, 1024)).astype(float) for m in (150, 300))
    a[np.abs(a) == 5] = 0
    C = rows.gemm_nt(_compact(a, "mxfp4"), _compact(b, "mxfp4")).cpu().numpy()
    assert np.array_equal(C, a @ b.T)
    a[3, 100], b[7] = np.nan, 0.0
    C = rows.gemm_nt(_compact(a, "mxfp4"), _compact(b, "mxfp4")).cpu().numpy()
    assert np.isnan(C[3]).all() and np.isfinite(np.delete(C, 3, 0)).all() and not np.delete(C, 3, 0)[:, 7].any()
    E = rows.gemm_nt(_compact(a[:0], "mxfp4"), _compact(b, "mxfp4"))
    assert E.shape == (0, 300)
    assert torch.equal(rows.gemm_nt(_compact(a[5:6], "mxfp4"), _compact(b, "mxfp4"))[0].cpu(), torch.as_tensor(C[5]))


def test_gemm_nt_does_not_write_past_its_columns():
    torch = _torch()
    from vittles_amd import rows
    for m, n in ((5, 37), (130, 129), (300, 259)):
        buf = torch.full((m + 2, n + 9), 7.0, device="cuda")
        rows.gemm_nt(_compact(_data(m, 200, 1), "mxfp4"), _compact(_data(n, 200, 2), "mxfp4"), out=buf[1:m + 1, 4:n + 4])
        assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, :4] == 7).all() and (buf[:, n + 4:] == 7).all()


@pytest.mark.parametrize("n,da,db", [(1, 1, 1), (3, 5, 2), (31, 33, 1), (32, 32, 32), (100, 64, 10), (257, 100, 129), (1000, 129, 65),
                                     (5001, 777, 33), (4096, 256, 128), (300, 1025, 300), (20000, 40, 7), (63, 130, 1000), (2049, 2049, 17)])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16"])
def test_gemm_tn(n, da, db, fmt, kind):
    torch = _torch()
    from oracle import compact as oc
    from vittles_amd import rows
    rng = np.random.default_rng(n + da + db)
    x = _data(n, da, n)
    X, xs = _compact(x, fmt), oc.store(x, fmt)
    g = torch.as_tensor(rng.standard_normal((n, db)) * np.exp(rng.standard_normal((n, 1))), device="cuda").to(getattr(torch, kind))
    g[::7] = 0.0
    gs = g.double().cpu().numpy()
    c = rows.gemm_tn(X, g)
    assert c.dtype == torch.float32
    bound = _product_bound(xs.T, gs, n) + 2.0 ** -126 * n
    assert (np.abs(c.cpu().numpy().astype(float) - xs.T @ gs) <= bound + 2.0 ** -24 * np.abs(xs.T @ gs)).all()
    # with data weights: rowscale * g is rounded once to float
    w = rng.random(n)
    w[::3] = 0.0
    bias = rng.standard_normal(db).astype(np.float32)
    out = torch.full((da, db + 5), 7.0, device="cuda")
    got = rows.gemm_tn(X, g, rowscale=torch.as_tensor(w, device="cuda"), alpha=2.0, bias=torch.as_tensor(bias, device="cuda"),
                       out=out[:, 2:db + 2])
    ws = w[:, None] * gs
    ref = 2.0 * (xs.T @ ws) + bias
    bound = 2.0 * _product_bound(xs.T, ws, n + 2) + 2.0 ** -125 * n
    assert (np.abs(got.cpu().numpy().astype(float) - ref) <= bound + 2.0 ** -23 * (np.abs(ref) + bound)).all()
    assert (out[:, :2] == 7).all() and (out[:, db + 2:] == 7).all()


def test_gemm_tn_extremes_and_refusals():
    torch = _torch()
    from vittles_amd import rows
    X = _compact(np.ones((40, 70)), "mxfp8")
    big = torch.full((40, 3), 1e38, device="cuda")
    big[1:] = 0.0
    assert torch.equal(rows.gemm_tn(X, big), torch.full((70, 3), 1e38, device="cuda"))
    mx = torch.zeros((40, 2), device="cuda")
    mx[5, 0] = torch.finfo(torch.float32).max
    assert (rows.gemm_tn(X, mx)[:, 0] == torch.finfo(torch.float32).max).all()
    for v in (float("inf"), float("-inf"), float("nan")):
        g = torch.zeros((40, 5), device="cuda")
        g[17, 2] = v
        c = rows.gemm_tn(X, g)
        assert torch.equal(torch.isfinite(c).all(0).cpu(), torch.tensor([True, True, False, True, True]))
        assert (c[:, 2] == v).all() or v != v and torch.isnan(c[:, 2]).all()
    bad = np.ones((40, 70))
    bad[3, 33] = np.nan
    c = rows.gemm_tn(_compact(bad, "mxfp8"), torch.ones((40, 4), device="cuda", dtype=torch.bfloat16))
    assert torch.isnan(c[32:64]).all() and (c[:32] == 40).all() and (c[64:] == 40).all()
    X0 = _compact(np.zeros((0, 70)), "mxfp8")
    z = rows.gemm_tn(X0, torch.zeros((0, 4), device="cuda"), bias=torch.arange(4.0, device="cuda"))
    assert torch.equal(z, torch.arange(4.0, device="cuda").expand(70, 4))
    g = torch.ones((40, 6), device="cuda")
    # orders and offsets of B
    t = torch.randn((6, 40), device="cuda").t()
    assert torch.equal(rows.gemm_tn(X, t), rows.gemm_tn(X, t.contiguous()))
    o = torch.randn((41, 9), device="cuda").to(torch.bfloat16)
    assert torch.equal(rows.gemm_tn(X, o[1:, 3:]), rows.gemm_tn(X, o[1:, 3:].contiguous()))
    assert torch.equal(rows.gemm_tn(X, o[:1].expand(40, 9)), rows.gemm_tn(X, o[:1].expand(40, 9).contiguous()))
    f64 = torch.ones(40, dtype=torch.float64, device="cuda")
    for call in (lambda: rows.gemm_tn(X, g[:39]), lambda: rows.gemm_tn(X, g[:, :0]), lambda: rows.gemm_tn(X, g, rowscale=f64[:39]),
                 lambda: rows.gemm_tn(X, g, rowscale=f64.float()), lambda: rows.gemm_tn(X, g, bias=f64[:6]),
                 lambda: rows.gemm_tn(X, g, out=torch.empty((70, 5), device="cuda")), lambda: rows.gemm_tn(X, g.cpu()),
                 lambda: rows.gemm_tn(X, g, out=torch.empty((6, 70), device="cuda").t()),
                 lambda: rows.gemm_tn(X, g, out=torch.empty((70, 6), device="cuda", dtype=torch.bfloat16)),
                 lambda: rows.gemm_nt(_compact(np.ones((3, 64)), "mxfp4"), _compact(np.ones((3, 65)), "mxfp4"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        rows.gemm_tn(X, g.double())
    with pytest.raises(TypeError):
        rows.gemm_nt(X, X)


def test_offsets_past_32_bits():
    """Codes of more than 4 GiB: the last rows are read from where they are."""
    torch = _torch()
    import vittles_amd as va
    from vittles_amd import rows
    n, d = 140000, 32768
    codes = torch.zeros((n, d), dtype=torch.uint8, device="cuda")
    scales = torch.full((n, d // 32), 127, dtype=torch.uint8, device="cuda")
    last = _compact(_data(3, d, 1), "mxfp8")
    codes[-3:], scales[-3:] = last.codes, last.scales
    X = va.compact.CompactRows(codes, scales, d)
    assert X.codes.data_ptr() == codes.data_ptr() and X.nbytes > 1 << 32
    v = torch.randn(d, dtype=torch.float64, device="cuda")
    u = torch.randn(n, dtype=torch.float64, device="cuda")
    z = rows.gemv(X, v)
    assert not z[:-3].any()
    torch.testing.assert_close(z[-3:], rows.gemv(last, v), rtol=EXACT, atol=EXACT * float(z.abs().max()))
    s = rows.gemv_t(X, u)
    torch.testing.assert_close(s, rows.gemv_t(last, u[-3:].clone()), rtol=EXACT, atol=EXACT * float(s.abs().max()))
    h = rows.glm_hvp(X, u.abs(), v)
    torch.testing.assert_close(h, rows.glm_hvp(last, u[-3:].abs(), v), rtol=EXACT, atol=EXACT * float(h.abs().max()))
    g = torch.randn((n, 3), device="cuda")
    c = rows.gemm_tn(X, g)
    ref = last.dequantise(torch.float64).t().contiguous() @ g[-3:].double()
    assert ((c - ref).abs() <= 5 * 2.0 ** -23 * (last.dequantise(torch.float64).abs().t() @ g[-3:].double().abs())).all()
    codes4 = codes.view(2 * n, d // 2)
    B = va.compact.CompactRows(codes4[:, :], torch.full((2 * n, d // 32), 127, dtype=torch.uint8, device="cuda"), d, "mxfp4")
    A = va.compact.CompactRows(B.codes[-2:].clone(), B.scales[-2:].clone(), d, "mxfp4")
    C = rows.gemm_nt(A, B)
    full = A.dequantise(torch.float64) @ A.dequantise(torch.float64).t().contiguous()
    assert not C[:, :-6].any() and ((C[:, -2:] - full).abs() <= d * 2.0 ** -23 * A.dequantise(torch.float64).square().sum()).all()


def test_streams_and_captured_graphs():
    """A side stream, and two captured graphs replayed several times in turn with eager work between them."""
    torch = _torch()
    import vittles_amd as va
    from vittles_amd import rows
    x = torch.randn((3000, 700), device="cuda")
    w = torch.rand(3000, dtype=torch.float64, device="cuda")
    v = torch.randn(700, dtype=torch.float64, device="cuda")
    g = torch.randn((3000, 40), device="cuda").to(torch.bfloat16)

    def work():
        X8, X4 = va.compact.quantise(x, "mxfp8"), va.compact.quantise(x, "mxfp4")
        return [rows.glm_hvp(X8, w, v), rows.gemv(X4, v), rows.gemv_t(X8, w), rows.gemm_nt(va.compact.quantise(x[:300], "mxfp4"), X4),
                rows.gemm_tn(X8, g, rowscale=w), X8.dequantise()]

    expect = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work())
        graphs.append(graph)
    for k in range(3):
        x.copy_(torch.randn((3000, 700), device="cuda"))
        w.copy_(torch.rand(3000, dtype=torch.float64, device="cuda"))
        expect = work()
        for graph, out in zip(graphs, outs):
            for t in out:
                t.fill_(float("nan"))
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, expect)), k


def test_used_together(relerr):
    """The whole path: activations stored in 8 bits, a logistic head on them fitted by the gradient, data-weight
    sensitivities of the fit by CG, 4-bit scores of query rows against all stored rows, and the weight gradient of a
    several-output head from the same store."""
    torch = _torch()
    from oracle import compact as oc, glm
    import vittles_amd as va
    from vittles_amd import rows
    from vittles_amd.cg import GLMHessianVectorProduct
    rng = np.random.default_rng(11)
    n, d, k = 1200, 150, 6
    x = rng.standard_normal((n, d))
    xs = oc.store(x, "mxfp8")
    y = (rng.random(n) < 1 / (1 + np.exp(-xs[:, 0]))).astype(float)
    w = 0.5 + rng.random(n)
    obj = va.WeightedGLMObjective(x, y, prior=1.0, dtype="mxfp8")
    theta = np.zeros(d)
    for _ in range(8):                                                   # Newton steps by CG
        hvp = GLMHessianVectorProduct(obj, theta, w)
        solve = va.solver_lib.get_cg_solver(hvp, d, cg_opts={"tol": 1e-13})
        theta = theta - solve(obj.grad(theta, w).cpu().numpy())
    ref = glm.newton_optimum("logistic", xs, y, w, prior=1.0)
    assert relerr(theta, ref) < 1e-9
    _, r, _ = rows.glm_link(obj, theta, w)
    picked = np.arange(0, n, 300)
    cross = xs[picked].T * r.cpu().numpy()[picked]
    S = -va.solver_lib.get_cg_solver(GLMHessianVectorProduct(obj, theta, w), d, cg_opts={"tol": 1e-13})(cross)
    _, _, S_ref = glm.sensitivity("logistic", xs, y, ref, w, prior=1.0)
    assert relerr(S, S_ref[:, picked]) < 1e-9
    scores = rows.gemm_nt(va.compact.quantise(S.T.copy(), "mxfp4"), va.compact.quantise(x, "mxfp4"))
    a, b = oc.store(S.T, "mxfp4"), oc.store(x, "mxfp4")
    assert (np.abs(scores.cpu().numpy() - a @ b.T) <= _product_bound(a, b.T, d) + 2.0 ** -24 * np.abs(a @ b.T)).all()
    dz = torch.as_tensor(rng.standard_normal((n, k)), device="cuda").to(torch.bfloat16)
    dW = rows.gemm_tn(obj.X, dz, rowscale=torch.as_tensor(w, device="cuda"))
    wz = w[:, None] * dz.double().cpu().numpy()
    assert (np.abs(dW.cpu().numpy() - xs.T @ wz) <= _product_bound(xs.T, wz, n + 2) + 2.0 ** -23 * np.abs(xs.T @ wz)).all()
