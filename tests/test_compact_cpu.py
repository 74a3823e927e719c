"""CPU tests (no GPU) of compact rows: the oracle's quantisation against the format's definition, the refusals that run
before any kernel, and the workspace queries."""
import numpy as np
import pytest
import torch

from oracle import compact as oc


@pytest.mark.parametrize("fmt,step", [("mxfp8", 2.0 ** -4), ("mxfp4", 2.0 ** -2)])
def test_oracle_rounds_by_half_a_step_and_never_saturates(fmt, step):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 97)) * np.exp(3 * rng.standard_normal((200, 1)))
    v = oc.store(x, fmt)
    codes, scales = oc.quantise(x, fmt)
    s = np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, axis=1)[:, :97]
    # half a step of the element, or half the smallest step of its block
    smallest = oc.GRID[fmt][1] * s
    assert (np.abs(v - x) <= np.maximum(step * np.abs(x), smallest / 2)).all()
    # the scale is the smallest one: with half of it the largest magnitude has no code
    top = np.abs(np.pad(x, ((0, 0), (0, 31)))).reshape(200, 4, 32).max(-1)
    assert (oc.round_to_code(top / np.ldexp(0.5, scales.astype(int) - 127), fmt) > len(oc.GRID[fmt]) - 1).all()


def test_oracle_edges():
    row = lambda *v: np.array([list(v)])
    assert oc.store(row(464.0), "mxfp8")[0, 0] == 448.0           # the tie past 448 stays with the even code
    assert oc.store(row(465.0), "mxfp8")[0, 0] == 480.0           # the scale doubles: 240 * 2
    assert oc.store(row(7.0), "mxfp4")[0, 0] == 8.0               # 7 is a tie between 6 (odd) and 8: 4 * 2
    assert oc.store(row(6.9), "mxfp4")[0, 0] == 6.0
    assert (oc.store(row(1.0, 2.0 ** -30), "mxfp8")[0] == [1.0, 0.0]).all()
    codes, scales = oc.quantise(np.zeros((1, 40)), "mxfp8")
    assert (codes == 0).all() and (scales == 0).all()
    for bad in (np.inf, -np.inf, np.nan, 2.0 ** 128):
        v = oc.store(row(1.0, bad), "mxfp4")
        assert np.isnan(v).all()
    v = oc.store(np.concatenate([np.full((1, 32), np.nan), np.ones((1, 3))], axis=1), "mxfp8")
    assert np.isnan(v[0, :32]).all() and (v[0, 32:] == 1.0).all()


def test_formats_agree_with_torch_float8():
    codes = np.arange(256, dtype=np.uint8).reshape(8, 32)
    v = oc.values(codes, np.full((8, 1), 127, dtype=np.uint8), 32, "mxfp8")
    t = torch.from_numpy(codes).view(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert np.array_equal(v, t, equal_nan=True)


def test_refusals_before_any_kernel():
    import vittles_amd as va
    from vittles_amd import _lib, rows
    c, s = torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8)
    with pytest.raises(ValueError, match="format"):
        va.compact.CompactRows(c, s, 40, "mxfp6")
    with pytest.raises(ValueError, match="on the GPU"):
        va.compact.CompactRows(c, s, 40)
    for codes, scales, D in ((c[:, :32], s, 40), (c, s[:, :1], 40), (c.to(torch.int8), s, 40), (c, s, 100), (c[0], s, 40)):
        with pytest.raises(ValueError, match="uint8 tensor"):
            va.compact.CompactRows(codes, scales, D)
    with pytest.raises(ValueError, match="at least 1"):
        va.compact.CompactRows(c, s, 0)
    with pytest.raises(TypeError, match="mxfp4"):
        rows.gemm_nt(torch.zeros(2, 2), torch.zeros(2, 2))
    if not torch.cuda.is_available():
        with pytest.raises(_lib.VittlesHipError, match="no CPU fallback"):
            va.compact.quantise(np.zeros((2, 2)))
        with pytest.raises(_lib.VittlesHipError, match="no CPU fallback"):
            va.WeightedGLMObjective(np.zeros((4, 2)), np.zeros(4), dtype="mxfp8")


def test_c_abi_refuses_bad_arguments():
    """Everything here returns before a launch: the addresses are never used."""
    from vittles_amd import _lib
    lib = _lib.load()
    BAD, WS = -1, -3
    A = 1 << 20                                                     # an aligned address
    q = lambda **k: lib.vt_mx_quantise(*{**dict(type=1, X=A, ldx=64, N=2, D=64, format=1, codes=A, ldc=64, scales=A, lds=2,
                                                stream=0), **k}.values())
    for bad in (dict(type=4), dict(type=-1), dict(X=0), dict(ldx=63), dict(N=-1), dict(D=0), dict(D=(1 << 30) + 1), dict(format=2), dict(codes=0),
                dict(codes=A + 8), dict(ldc=48), dict(ldc=72), dict(scales=0), dict(lds=1)):
        assert q(**bad) == BAD, bad
    assert q(N=0) == 0
    dq = lambda **k: lib.vt_mx_dequantise(*{**dict(format=0, codes=A, ldc=32, scales=A, lds=2, N=2, D=64, type=1, out=A,
                                                   ldo=64, stream=0), **k}.values())
    for bad in (dict(format=-1), dict(out=0), dict(ldo=63), dict(type=9), dict(ldc=16)):
        assert dq(**bad) == BAD, bad
    ws = lib.vt_mx_rows_workspace_bytes(100, 64)
    assert ws >= 800 and lib.vt_mx_rows_workspace_bytes(-1, 64) == 0
    hvp = lambda **k: lib.vt_mx_glm_hvp(*{**dict(format=1, codes=A, ldc=64, scales=A, lds=2, d=A, prior=0, ps=0.0, v=A, N=100,
                                                 D=64, out=A, ws=A, wsb=ws, stream=0), **k}.values())
    for bad, rc in ((dict(v=0), BAD), (dict(out=0), BAD), (dict(d=0), BAD), (dict(lds=1), BAD), (dict(ws=0), WS),
                    (dict(wsb=ws - 1), WS)):
        assert hvp(**bad) == rc, bad
    grad = lambda **k: lib.vt_mx_glm_grad(*{**dict(family=0, format=1, codes=A, ldc=64, scales=A, lds=2, theta=A, y=A, w=A,
                                                   off=0, scale=1.0, prior=0, N=100, D=64, g=A, r=0, d=0, ws=A, wsb=ws,
                                                   stream=0), **k}.values())
    for bad, rc in ((dict(family=3), BAD), (dict(theta=0), BAD), (dict(y=0), BAD), (dict(g=0), BAD), (dict(wsb=0), WS)):
        assert grad(**bad) == rc, bad
    nws = lib.vt_mx_gemm_nt_workspace_bytes(4, 4, 64)
    nt = lambda **k: lib.vt_mx_gemm_nt(*{**dict(ca=A, ldca=32, sa=A, ldsa=2, M=4, cb=A, ldcb=32, sb=A, ldsb=2, N=4, K=64,
                                                alpha=1.0, bias=0, type=1, C=A, ldc=4, ws=A, wsb=nws, stream=0), **k}.values())
    for bad in (dict(ca=0), dict(ldcb=16), dict(ldsa=1), dict(type=0), dict(type=3), dict(C=0), dict(ldc=3), dict(K=0), dict(M=-1)):
        assert nt(**bad) == BAD, bad
    assert nt(M=0) == 0 and nt(N=0) == 0
    tws = lib.vt_mx_gemm_tn_workspace_bytes(100, 64, 8)
    tn = lambda **k: lib.vt_mx_gemm_tn(*{**dict(format=1, codes=A, ldc=64, scales=A, lds=2, Da=64, type=2, B=A, ldb=8, Db=8,
                                                rs=0, N=100, alpha=1.0, bias=0, C=A, ldo=8, ws=A, wsb=tws, stream=0), **k}.values())
    for bad, rc in ((dict(type=0), BAD), (dict(B=0), BAD), (dict(ldb=7), BAD), (dict(Db=0), BAD), (dict(C=0), BAD),
                    (dict(ldo=7), BAD), (dict(ws=0), WS), (dict(wsb=tws - 1), WS)):
        assert tn(**bad) == rc, bad
    assert lib.vt_mx_gemm_tn_workspace_bytes(-1, 4, 4) == 0
