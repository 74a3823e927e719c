"""Cases of the compact-row operators: rows kept in microscaled 4-bit or 8-bit floating point, and what reads them.

    store      rows are quantised (``compact.quantise``) and read back
    product    scores of query rows against stored 4-bit rows: the queries are quantised within the call, ``rows.gemm_nt``
    weights    gradient of a linear layer's weights from its 8-bit activations, ``rows.gemm_tn``
    gradient   forward and backward pass of a weighted GLM over compact rows, ``rows.glm_grad``
    hvp        Hessian-vector product of that GLM, one product of a CG solve, ``rows.glm_hvp``

A block is 32 columns of a row: one scale byte (a power of two, 2^(byte - 127)) and 32 codes, E2M1 ("mxfp4", two in a byte, the
even column in the low half) or E4M3 ("mxfp8").  The scale is the smallest one with which the block's largest magnitude, rounded,
is still a finite code; columns behind the row's end hold code 0.
"""
import math

import torch

own = False

BLOCK = 32
CODE_BYTES = {"mxfp4": 16, "mxfp8": 32}          # of a block
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token's activations written to a 4-bit store and read back: latency
        {"name": "store 4-bit, one row", "op": "store", "format": "mxfp4", "type": "bf16", "n": 1, "d": 4096},
        # a batch's activations kept in 8 bits until the backward pass
        {"name": "store 8-bit, batch", "op": "store", "format": "mxfp8", "type": "bf16", "n": 16384, "d": 4096},
        # one query against the stored rows: each stored byte is read once
        {"name": "product, one query", "op": "product", "type": "bf16", "m": 1, "n": 4096, "k": 4096},
        # a few queries, nothing a multiple of anything
        {"name": "product, ragged", "op": "product", "type": "fp32", "m": 37, "n": 5003, "k": 1111},
        # an ordinary batch of queries
        {"name": "product, batch", "op": "product", "type": "bf16", "m": 2048, "n": 4096, "k": 4096},
        # all rows of one store against all of another: the largest product
        {"name": "product, all pairs", "op": "product", "type": "bf16", "m": 8192, "n": 8192, "k": 8192},
        # a layer of 1000 outputs, gradients in bfloat16
        {"name": "weights, bf16", "op": "weights", "type": "bf16", "n": 16384, "d": 4096, "k": 1000, "weighted": False},
        # a small odd layer, float gradients, data weights on the rows
        {"name": "weights, fp32 weighted", "op": "weights", "type": "fp32", "n": 5001, "d": 777, "k": 33, "weighted": True},
        # the framework's N = 10^6, D = 100 logistic regression, rows in 8 bits
        {"name": "gradient, D = 100", "op": "gradient", "format": "mxfp8", "family": "logistic", "n": 1000000, "d": 100},
        # wide odd rows in 4 bits
        {"name": "gradient, wide 4-bit", "op": "gradient", "format": "mxfp4", "family": "poisson", "n": 20011, "d": 5003},
        # the framework's D = 20 000 matrix-free solve, rows in 8 bits: one product of its CG iteration
        {"name": "hvp, D = 20000", "op": "hvp", "format": "mxfp8", "n": 100000, "d": 20000},
        # a small solve: latency
        {"name": "hvp, small", "op": "hvp", "format": "mxfp8", "n": 1001, "d": 333},
    ]


def _size(rng, low, high):
    """A size between low and high, even over the logarithm; every second one odd."""
    s = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return min(high, s | 1 if rng.random() < 0.5 else s)


def draw(rng):
    op = rng.choice(["store", "product", "weights", "gradient", "hvp"])
    if op == "store":
        d = _size(rng, 1, 20000)
        return {"op": op, "format": rng.choice(["mxfp4", "mxfp8"]), "type": rng.choice(["bf16", "fp16", "fp32"]),
                "n": _size(rng, 1, max(1, min(200000, 60000000 // d))), "d": d}
    if op == "product":
        return {"op": op, "type": rng.choice(["bf16", "fp16", "fp32"]), "m": _size(rng, 1, 8192), "n": _size(rng, 16, 8192),
                "k": _size(rng, 16, 8192)}
    if op == "weights":
        return {"op": op, "type": rng.choice(["bf16", "fp16", "fp32"]), "n": _size(rng, 1, 16384), "d": _size(rng, 16, 4096),
                "k": _size(rng, 1, 1000), "weighted": rng.random() < 0.5}
    d = _size(rng, 4, 20000)
    case = {"op": op, "format": rng.choice(["mxfp4", "mxfp8", "mxfp8"]), "n": _size(rng, 16, min(1000000, 400000000 // d)), "d": d}
    if op == "gradient":
        case["family"] = rng.choice(["logistic", "poisson", "gaussian"])
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------

def _activations(n, d, gen, dtype):
    """Rows as a network's layer gives them: normal, columns of unequal scale and a few large ones, some rows that are padding."""
    column = torch.exp(0.5 * torch.randn(d, generator=gen, device="cuda"))
    column = torch.where(torch.rand(d, generator=gen, device="cuda") < 0.01, 20 * column, column)
    row = (torch.rand(n, generator=gen, device="cuda") >= 0.02).to(torch.float32)
    return torch.randn((n, d), generator=gen, device="cuda").mul_(column).mul_(row[:, None]).to(dtype)


def _stored(n, d, fmt, gen):
    """Codes and scales of n rows, as a program holds them."""
    codes = torch.empty((n, -(-d // BLOCK) * CODE_BYTES[fmt]), dtype=torch.uint8, device="cuda")
    scales = torch.empty((n, -(-d // BLOCK)), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // d)
    for i in range(0, n, step):
        codes[i:i + step], scales[i:i + step] = _quantise(_activations(min(step, n - i), d, gen, torch.float32), fmt)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    op = case["op"]
    if op == "store":
        s["x"] = _activations(case["n"], case["d"], gen, TYPES[case["type"]])
    elif op == "product":
        s["x"] = _activations(case["m"], case["k"], gen, TYPES[case["type"]])
        s["codes"], s["scales"] = _stored(case["n"], case["k"], "mxfp4", gen)
    elif op == "weights":
        s["codes"], s["scales"] = _stored(case["n"], case["d"], "mxfp8", gen)
        g = 1e-3 * torch.randn((case["n"], case["k"]), generator=gen, device="cuda")
        s["g"] = g.to(TYPES[case["type"]])
        s["rowscale"] = 0.5 + torch.rand(case["n"], generator=gen, device="cuda", dtype=torch.float64) if case["weighted"] else None
    else:
        n, d = case["n"], case["d"]
        s["codes"], s["scales"] = _stored(n, d, case["format"], gen)
        w = 0.5 + torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        w[torch.rand(n, generator=gen, device="cuda") < 0.05] = 0.0          # rows left out of the fit
        s["prior"] = 0.5 + torch.rand(d, generator=gen, device="cuda", dtype=torch.float64)
        s["v"] = 0.3 * torch.randn(d, generator=gen, device="cuda", dtype=torch.float64) / d ** 0.5
        if op == "hvp":
            s["dd"] = 0.25 * w
        else:
            s["w"] = w
            s["y"] = (torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) < 0.5).to(torch.float64)
            if own:       # the objective holds the rows for as long as the program runs
                import vittles_amd as va
                s["objective"] = va.WeightedGLMObjective(_compact(s, d), s["y"], family=case["family"], prior=s["prior"])
    return s


# ---- the framework's operators ------------------------------------------------------------------------------------

def _compact(s, d):
    from vittles_amd import compact
    return compact.CompactRows(s["codes"], s["scales"], d, s.get("format") or ("mxfp4" if s["op"] == "product" else "mxfp8"))


def _run_own(s):
    from vittles_amd import compact, rows
    op = s["op"]
    if op == "store":
        return compact.quantise(s["x"], s["format"]).dequantise()
    if op == "product":
        return rows.gemm_nt(compact.quantise(s["x"], "mxfp4"), _compact(s, s["k"]))
    if op == "weights":
        return rows.gemm_tn(_compact(s, s["d"]), s["g"], rowscale=s["rowscale"])
    if op == "gradient":
        return rows.glm_grad(s["objective"], s["v"], s["w"], prior=s["prior"])
    return rows.glm_hvp(_compact(s, s["d"]), s["dd"], s["v"], prior=s["prior"])


# ---- the plain form -----------------------------------------------------------------------------------------------

def _quantise(x, fmt):
    """Codes and scales of float rows.  Scaling by a power of two is exact in 32 bits, so only the code is rounded."""
    n, d = x.shape
    nb = -(-d // BLOCK)
    x = torch.nn.functional.pad(x.to(torch.float32), (0, nb * BLOCK - d)).view(n, nb, BLOCK)
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m == 0, -127, e - 1 - (8 if fmt == "mxfp8" else 2) + (m > 0.90625 if fmt == "mxfp8" else m >= 0.875).to(e.dtype))
    e = e.clamp(-127, 126)
    x = x * ((127 - e) << 23).view(torch.float32).unsqueeze(-1)
    if fmt == "mxfp8":
        codes = x.to(torch.float8_e4m3fn).view(torch.uint8).view(n, nb * BLOCK)
    else:
        a = x.abs()
        c = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
        c = (c + 8 * (x < 0)).to(torch.uint8).view(n, nb * BLOCK // 2, 2)
        codes = c[:, :, 0] + 16 * c[:, :, 1]
    return codes, (e + 127).to(torch.uint8)


def _values(codes, scales, d, fmt, dtype=torch.float32):
    """The values that codes and scales stand for."""
    n, nb = scales.shape
    if fmt == "mxfp8":
        v = codes.view(torch.float8_e4m3fn).to(dtype)
    else:
        table = torch.tensor(FP4 + tuple(-f for f in FP4), dtype=dtype, device="cuda")
        v = table[torch.stack((codes & 15, codes >> 4), dim=-1).to(torch.int32)]
    scale = ((scales.to(torch.int64) + 896) << 52).view(torch.float64).to(dtype)
    return (v.view(n, nb, BLOCK) * scale.unsqueeze(-1)).view(n, nb * BLOCK)[:, :d]


def _link(family, z, y):
    if family == "logistic":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p - y, p * (1.0 - p)
    if family == "poisson":
        e = torch.exp(z)
        return e - y, e
    return z - y, torch.ones_like(z)


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "store":
        return _values(*_quantise(s["x"], s["format"]), s["d"], s["format"])
    if op == "product":
        a = _values(*_quantise(s["x"], "mxfp4"), s["k"], "mxfp4")
        return a @ _values(s["codes"], s["scales"], s["k"], "mxfp4").t()
    if op == "weights":
        g = s["g"].to(torch.float32)
        if s["rowscale"] is not None:
            g = (s["rowscale"][:, None] * g).to(torch.float32)
        return _values(s["codes"], s["scales"], s["d"], "mxfp8").t() @ g
    x = _values(s["codes"], s["scales"], s["d"], s["format"], torch.float64)     # the framework's vectors are 64-bit
    if op == "gradient":
        l1, l2 = _link(s["family"], x @ s["v"], s["y"])
        return x.t() @ (s["w"] * l1) + s["prior"] * s["v"], l1, s["w"] * l2
    return x.t() @ (s["dd"] * (x @ s["v"])) + s["prior"] * s["v"]


# ---- work and exact values ----------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "store":
        elements = case["n"] * case["d"]
        return {"bytes": elements * ((4 if case["type"] == "fp32" else 2) + 4), "flops": 3 * elements}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * (4 if case["type"] == "fp32" else 2) + n * -(-k // BLOCK) * 17 + 4 * m * n, "flops": 2 * m * n * k}
    if op == "weights":
        n, d, k = case["n"], case["d"], case["k"]
        return {"bytes": n * -(-d // BLOCK) * 33 + n * k * (4 if case["type"] == "fp32" else 2) + 4 * d * k + (8 * n if case["weighted"] else 0),
                "flops": 2 * n * d * k}
    n, d = case["n"], case["d"]
    stored = n * -(-d // BLOCK) * (1 + CODE_BYTES[case["format"]])
    return {"bytes": stored + (32 * n if op == "gradient" else 8 * n) + 24 * d, "flops": 4 * n * d}


def _grid(fmt):
    """All magnitudes of a format, from its definition."""
    if fmt == "mxfp4":
        return [0.0, 0.5] + [(1 + f / 2) * 2.0 ** e for e in range(3) for f in range(2)]
    return [f * 2.0 ** -9 for f in range(8)] + [(1 + f / 8) * 2.0 ** e for e in range(-6, 9) for f in range(8)][:-1]


def _power(e):
    """2^e in 64 bits, for whole e."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_store(x, fmt):
    """The values of quantised rows in 64 bits, by the definition: the smallest scale whose largest magnitude still rounds to a
    code, each element to the nearest code, ties to the code whose last bit is 0 (every second magnitude)."""
    n, d = x.shape
    grid = torch.tensor(_grid(fmt), dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    last = 2 * grid[-1] - grid[-2] if fmt == "mxfp8" else grid[-1] + 2.0       # the step that would follow the largest code
    border = (grid[-1] + last) / 2
    ties_up = (len(grid) - 1) % 2 == 1                                          # at the border an odd code rounds away
    out = torch.empty((n, d), dtype=torch.float64, device=x.device)
    for i in range(0, n, max(1, (1 << 24) // d)):
        part = x[i:i + max(1, (1 << 24) // d)].to(torch.float64)
        nb = -(-d // BLOCK)
        p = torch.zeros((part.shape[0], nb * BLOCK), dtype=torch.float64, device=x.device)
        p[:, :d] = part
        p = p.view(-1, nb, BLOCK)
        top = p.abs().amax(-1)
        e = torch.floor(torch.log2(torch.clamp(top / border, min=2.0 ** -140))).to(torch.int64) - 1
        for _ in range(3):                                                      # up to the first scale that holds it
            q = top * _power(-e)
            e = torch.where((q >= border) if ties_up else (q > border), e + 1, e)
        e = e.clamp(-127, 127)
        q = p * _power(-e).unsqueeze(-1)
        a = q.abs()
        k = torch.bucketize(a, middle)                                          # a tie stays with the lower code ...
        tie = (k < len(middle)) & (a == middle[k.clamp(max=len(middle) - 1)])
        k = k + (tie & (k % 2 == 1))                                            # ... unless that one is odd
        v = grid[k] * torch.sign(q) * _power(e).unsqueeze(-1)
        out[i:i + part.shape[0]] = v.view(-1, nb * BLOCK)[:, :d]
    return out


def _exact_values(codes, scales, d, fmt):
    """Codes to values in 64 bits, bit by bit."""
    out = torch.empty((codes.shape[0], d), dtype=torch.float64, device=codes.device)
    step = max(1, (1 << 25) // d)
    for i in range(0, codes.shape[0], step):
        c = codes[i:i + step].to(torch.int16)
        if fmt == "mxfp4":
            c = torch.stack((c % 16, c // 16), dim=-1).reshape(c.shape[0], -1)
            sign, ex, mant, bias, width = c // 8, c // 2 % 4, c % 2, 1, 2.0
        else:
            sign, ex, mant, bias, width = c // 128, c // 8 % 16, c % 8, 7, 8.0
        mant = mant.to(torch.float64)
        v = torch.where(ex == 0, mant / width * 2.0 ** (1 - bias), (1 + mant / width) * _power(ex - bias))
        v = torch.where(sign == 1, -v, v).view(c.shape[0], -1, BLOCK)
        v = v * _power(scales[i:i + step].to(torch.int16) - 127).unsqueeze(-1)
        out[i:i + step] = v.view(c.shape[0], -1)[:, :d]
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "store":
        return _exact_store(s["x"], case["format"])
    if op == "product":
        return _exact_store(s["x"], "mxfp4") @ _exact_values(s["codes"], s["scales"], case["k"], "mxfp4").t().contiguous()
    if op == "weights":
        g = s["g"].to(torch.float64)
        if case["weighted"]:
            g = g * s["rowscale"][:, None]
        return _exact_values(s["codes"], s["scales"], case["d"], "mxfp8").t().contiguous() @ g
    d = case["d"]
    z = torch.empty(case["n"], dtype=torch.float64, device="cuda")
    total = torch.zeros(d, dtype=torch.float64, device="cuda")
    l1, l2 = torch.empty_like(z), torch.empty_like(z)
    step = max(1, (1 << 27) // d)
    for i in range(0, case["n"], step):
        x = _exact_values(s["codes"][i:i + step], s["scales"][i:i + step], d, case["format"])
        z = (x * s["v"]).sum(-1)
        if op == "hvp":
            total += (x * (s["dd"][i:i + step] * z)[:, None]).sum(0)
            continue
        y, w = s["y"][i:i + step], s["w"][i:i + step]
        if case["family"] == "logistic":
            p = torch.sigmoid(z)
            a, b = p - y, p * torch.sigmoid(-z)
        elif case["family"] == "poisson":
            a, b = torch.exp(z) - y, torch.exp(z)
        else:
            a, b = z - y, torch.ones_like(z)
        l1[i:i + step], l2[i:i + step] = a, w * b
        total += (x * (w * a)[:, None]).sum(0)
    total = total + s["prior"] * s["v"]
    return total if op == "hvp" else (total, l1, l2)
