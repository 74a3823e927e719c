"""GPU tests of the products of compact rows with whole numbers: every tile, whole and split, compared bit for bit.

The stored values, the other operand, the bias and every sum of magnitudes are whole numbers below 2^24, so each partial sum
is exact in float whatever the order, and a bfloat16 result is the one rounding of it.  Each shape names the kernel that it
is meant for; what ran is read from the kernel profiler."""
import re

import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    return torch


def _kernels(call):
    """The kernels that ``call`` runs, as (name, numbers and truth values among its template's arguments); None without a
    profiler, which gives names as they were written or mangled."""
    torch = _torch()
    from torch.profiler import profile, ProfilerActivity
    call()
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as prof:
        call()
        torch.cuda.synchronize()
    found = set()
    for e in prof.events():
        name = re.search(r"k_mx_(tn_join_few|tn_join|tn|nt_tile|nt_join|nt_few|quantise|dequantise)(?=[<(IE])(.*)", e.name)
        if name is None or not str(getattr(e, "device_type", "")).endswith("CUDA"):
            continue
        if name[2].startswith("<"):
            args = [{"true": 1, "false": 0}.get(s.strip(), s.strip()) for s in name[2][1:name[2].index(">")].split(",")]
            args = [int(s) for s in args if isinstance(s, int) or s.isdigit()]
        else:
            args = [int(s) for s in re.findall(r"L[ib](\d+)E", name[2])]
        found.add((name[1], tuple(args)))
    return found or None


def _placed(X, where):
    """``X`` in scales whose rows begin on 4 bytes ("words"), or in wider codes and scales, off by one byte ("shifted"),
    with codes and NaN scales around what is read."""
    torch = _torch()
    from vittles_amd import compact
    n, nb, width = X.shape[0], X.scales.shape[1], X.codes.shape[1]
    pitch, first = ((nb + 3) // 4 * 4, 0) if where == "words" else (nb + 4, 1)
    lead = 0 if where == "words" else 16
    codes = torch.full((n, width + 2 * lead), 0x77, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, pitch), 255, dtype=torch.uint8, device="cuda")
    codes[:, lead:lead + width] = X.codes
    scales[:, first:first + nb] = X.scales
    return compact.CompactRows(codes[:, lead:lead + width], scales[:, first:first + nb], X.D, X.format)


def _whole_rows(n, d, fmt, seed, largest):
    """Rows of whole numbers that E2M1 and E4M3 hold, times 1 or 2 by row, and their values in fp64."""
    torch = _torch()
    from vittles_amd import compact
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table = torch.tensor([0.0, 1.0, -1.0, 2.0, -2.0, 3.0, -3.0, 4.0, -4.0, 6.0, -6.0], dtype=torch.float64, device="cuda")
    table = table[table.abs() <= largest]
    x = table[torch.randint(0, len(table), (n, d), generator=gen, device="cuda")]
    x *= 2.0 ** torch.randint(0, 2, (n, 1), generator=gen, device="cuda").to(torch.float64)
    X = compact.quantise(x, fmt)
    assert torch.equal(X.dequantise(torch.float64), x)
    return X, x


# few rows; 128 x 128 tiles, whole and split; 256 x 256 tiles: a row's blocks end inside a chunk of eight, with it, after one
@pytest.mark.parametrize("m,n,k,kernel", [(150, 300, 1024, ("nt_few",)), (1100, 1201, 1056, ("nt_tile", 2, 2, 2, 2)),
                                          (512, 500, 8190, ("nt_tile", 2, 2, 2, 2)), (4000, 4090, 2050, ("nt_tile", 4, 2, 2, 4)),
                                          (3900, 4001, 3001, ("nt_tile", 4, 2, 2, 4)), (4096, 4096, 2048, ("nt_tile", 4, 2, 2, 4))])
@pytest.mark.parametrize("where", ["words", "shifted"])
def test_gemm_nt_whole_numbers(m, n, k, kernel, where):
    torch = _torch()
    from vittles_amd import compact, rows
    A, a = _whole_rows(m, k, "mxfp4", 1, 6)
    B, b = _whole_rows(n, k, "mxfp4", 2, 6)
    A, B = _placed(A, where), _placed(B, where)
    # bound of every partial sum of alpha times the product and the bias
    assert 2 * k * 12 * 12 + n < 1 << 24
    ref = a @ b.t()
    bias = torch.arange(n, device="cuda", dtype=torch.float32)
    want = 2.0 * ref + bias.double()
    pitch, first = ((n + 63) // 64 * 64, 0) if where == "words" else (n + 3, 1)
    for dtype in (torch.float32, torch.bfloat16):
        buf = torch.full((m + 1, pitch), 7.0, dtype=dtype, device="cuda")
        out = buf[:m, first:first + n]
        names = _kernels(lambda: rows.gemm_nt(A, B, alpha=2.0, bias=bias, out=out))
        if names is not None:              # in tiles: the scales come by DMA, or through registers
            way = () if kernel[0] == "nt_few" else (int(where == "words"),)
            assert any((s,) + args[:len(kernel) - 1 + len(way)] == kernel + way for s, args in names), names
        assert torch.equal(out, want.to(dtype))
        assert bool((buf[m] == 7).all() and (buf[:, :first] == 7).all() and (buf[:, first + n:] == 7).all())
    assert torch.equal(rows.gemm_nt(A, B), ref.float())
    # scale 255: the row is NaN, whatever the codes; in the first block, inside, in the last row's last block
    nb = A.scales.shape[1]
    A.scales[3, 0] = A.scales[m // 2, nb // 2] = A.scales[m - 1, nb - 1] = B.scales[n - 2, nb - 1] = 255
    A.codes[3] = 0
    ref[3] = ref[m // 2] = ref[m - 1] = ref[:, n - 2] = float("nan")
    for dtype in (torch.float32, torch.bfloat16):
        out = rows.gemm_nt(A, B, out=torch.empty((m, n), dtype=dtype, device="cuda"))
        assert torch.equal(torch.isnan(out), torch.isnan(ref)) and torch.equal(torch.nan_to_num(out), torch.nan_to_num(ref).to(dtype))


# 128 x 64, 256 x 128 and 256 x 256 tiles; one slab, a few (joined a thread an element), many
@pytest.mark.parametrize("n,da,db,kernel,split", [(120, 300, 65, (2, 1, 2, 2), False), (5001, 300, 33, (2, 1, 2, 2), True),
                                                  (300, 66000, 100, (4, 2, 2, 2), False), (16384, 1000, 99, (4, 2, 2, 2), True),
                                                  (700, 4090, 2301, (4, 2, 2, 4), False), (2000, 2560, 2550, (4, 2, 2, 4), True),
                                                  (8200, 500, 301, (4, 2, 2, 4), True)])
@pytest.mark.parametrize("kind,bits", [("bfloat16", 8), ("float16", 11), ("float32", 24), ("float32", 17)])
@pytest.mark.parametrize("weighted", [False, True])
def test_gemm_tn_whole_numbers(n, da, db, kernel, split, kind, bits, weighted):
    """Numbers of all the bits that the type holds: none of the bfloat16 parts they are cut into may be lost."""
    torch = _torch()
    from vittles_amd import compact, rows
    gen = torch.Generator(device="cuda").manual_seed(n + db + bits)
    fmt = "mxfp8" if (n + bits) % 2 else "mxfp4"
    bits -= 2 if weighted and bits == 24 else 0
    g = torch.randint(-(1 << bits) + 1, 1 << bits, (n, db), generator=gen, device="cuda").to(torch.float64)
    w = torch.randint(0, 4, (n,), generator=gen, device="cuda").to(torch.float64)
    gs = w[:, None] * g if weighted else g
    # as many rows of A as the sums have room for: every row in some column, 1 or -1
    room = max(1, min(n, (1 << 24) // (int(gs.abs().max()) + 1)))
    x = torch.zeros((n, da), dtype=torch.float64, device="cuda")
    pick = (torch.arange(da, device="cuda")[None, :] * 7 + torch.arange(room, device="cuda")[:, None] * (n // room)) % n
    sign = 1.0 - 2.0 * torch.randint(0, 2, (room, da), generator=gen, device="cuda").to(torch.float64)
    x.scatter_(0, pick, sign)
    X = compact.quantise(x, fmt)
    B = g.to(getattr(torch, kind))
    assert torch.equal(B.double(), g) and float((x.abs().t() @ gs.abs()).max()) < 1 << 24
    ref = x.t() @ gs
    names = _kernels(lambda: rows.gemm_tn(X, B, rowscale=w if weighted else None))
    if names is not None:                  # (format, weighted,) the tile, B's rows in words, split
        assert any(s == "tn" and args[-6:-2] == kernel and args[-1] == int(split) for s, args in names), names
    assert torch.equal(rows.gemm_tn(X, B, rowscale=w if weighted else None), ref.float())
    # alpha (a power of two), a bias whose infinity stays in its column, a result between guards at an odd pitch
    bias = torch.zeros(db, device="cuda")
    bias[db // 2] = float("inf")
    buf = torch.full((da + 1, db + 3), 7.0, device="cuda")
    rows.gemm_tn(X, B, rowscale=w if weighted else None, alpha=-2.0, bias=bias, out=buf[:da, 1:db + 1])
    assert torch.equal(buf[:da, 1:db + 1], (-2.0 * ref + bias.double()).float())
    assert bool((buf[da] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, db + 1:] == 7).all())


def test_gemm_tn_smallest_numbers():
    """A is taken to the nearest multiple of 2^-133 (ties to even), a float of B cut to one; larger numbers are exact."""
    torch = _torch()
    from vittles_amd import compact, rows
    step = 2.0 ** -133
    for fmt, width in (("mxfp8", 256), ("mxfp4", 128)):
        # a row for each scale byte 0 .. 7, all bytes as codes but the NaN of E4M3
        codes = (torch.arange(width, device="cuda") * (256 // width) + (fmt == "mxfp4")).to(torch.uint8).expand(8, width).clone()
        if fmt == "mxfp8":
            codes[:, [0x7F, 0xFF]] = 0x7E
        d = width * (1 if fmt == "mxfp8" else 2)
        scales = torch.arange(8, dtype=torch.uint8, device="cuda")[:, None].expand(8, d // 32).clone()
        X = compact.CompactRows(codes, scales, d, fmt)
        x = X.dequantise(torch.float64)
        near = torch.round(x / step) * step
        assert torch.equal(near[3:], x[3:]) and (fmt == "mxfp8") != torch.equal(near[:3], x[:3])
        for kind in (torch.bfloat16, torch.float32):
            g = (2.0 ** 100 * torch.eye(8, device="cuda")).to(kind)
            for w in (None, torch.ones(8, dtype=torch.float64, device="cuda")):
                assert torch.equal(rows.gemm_tn(X, g, rowscale=w).double(), near.t() * 2.0 ** 100)
    gen = torch.Generator(device="cuda").manual_seed(8)
    X = compact.quantise(torch.full((1, 40), 2.0 ** 20, device="cuda"), "mxfp8")
    b = (1.0 + torch.rand(900, generator=gen, device="cuda")) * torch.sign(torch.randn(900, generator=gen, device="cuda"))
    b = torch.ldexp(b.double(), torch.arange(900, device="cuda") % 50 - 149).float()[None, :]
    cut = torch.trunc(b.double() / step) * step
    large = b.abs() >= 2.0 ** -110
    assert torch.equal(cut[large], b.double()[large]) and bool(large.any())
    for w in (None, torch.ones(1, dtype=torch.float64, device="cuda")):
        assert torch.equal(rows.gemm_tn(X, b, rowscale=w).double(), (cut * 2.0 ** 20).expand(40, 900))
