"""Cases for timing the optimiser-state operators: rows kept in 8 bits, sparse Adam on such rows, and
orthogonalised updates of matrices.  ``run`` computes the plain form in elementary 32-bit torch operations, or
calls the package's operators where ``own`` is true; ``exact`` is the same from the definition in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
COEF = (3.4445, -4.7750, 2.0315)
EPS_NORM = 1e-7
B1, B2, EPS_ADAM = 0.9, 0.999, 1e-15
BETA, DECAY = 0.95, 0.01
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # first moments or features of the Gaussians one camera sees, stored into a 2M scene's 8-bit rows
        dict(name="write_visible_sh", op="write", kind="e4m3", N=2_000_000, D=45, group=128, n=150_001, dtype="f32",
             dither=True),
        # a handful of feature rows written and read back: latency
        dict(name="write_few_int8", op="write", kind="int8", N=4096, D=128, group=64, n=37, dtype="bf16",
             dither=False),
        # a whole store decoded, as before a checkpoint
        dict(name="read_all_sh", op="read", kind="e4m3", N=1_000_000, D=48, group=48, n=0, dtype="bf16"),
        # listed rows of odd width in odd groups
        dict(name="read_rows_odd", op="read", kind="int8", N=300_000, D=201, group=67, n=99_991, dtype="f16"),
        # the step of the SH coefficients of an 8M scene for the Gaussians one batch sees
        dict(name="adam_rows_city", op="adam_rows", N=8_000_000, M=45, group=128, n=320_003),
        # dense gradients with a visibility mask, a million Gaussians
        dict(name="adam_dense_mid", op="adam_dense", N=1_000_000, M=45, group=128, n=0),
        # a small scene's step: latency
        dict(name="adam_rows_small", op="adam_rows", N=5000, M=12, group=128, n=1001),
        # one small colour matrix per Gaussian or image
        dict(name="orth_small_batch", op="orth", B=200_000, rows=15, cols=3, dtype="f32"),
        # a square weight of a decoder
        dict(name="orth_square", op="orth", B=1, rows=1024, cols=1024, dtype="bf16"),
        # a tall ragged weight
        dict(name="orth_ragged", op="orth", B=1, rows=777, cols=201, dtype="f16"),
        # the layers of a small network in one call
        dict(name="update_layers", op="update", B=24, rows=128, cols=256, dtype="f32", nesterov=True),
        # a wide weight
        dict(name="update_large", op="update", B=1, rows=4096, cols=2048, dtype="bf16", nesterov=True),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "read", "adam_rows", "adam_dense", "orth", "orth", "update", "update"))
    if op in ("write", "read"):
        D = _between(rng, 1, 300)
        N = _between(rng, 500, min(2_000_000, 40_000_000 // D))
        c = dict(op=op, kind=rng.choice(("int8", "e4m3")), N=N, D=D, group=rng.choice((16, 45, 64, 128, 256)),
                 n=_between(rng, 1, N), dtype=rng.choice(("f32", "bf16", "f16")))
        if op == "write":
            c["n"] = min(c["n"], 6_000_000 // D + 1)
            c["dither"] = rng.random() < 0.5
        return c
    if op.startswith("adam"):
        M = rng.choice((1, 3, 4, 12, 45, 48, rng.randrange(5, 200)))
        N = _between(rng, 300, 40_000_000 // M if op == "adam_rows" else 20_000_000 // M)
        n = _between(rng, 1, max(1, min(N, 12_000_000 // M))) if op == "adam_rows" else 0
        return dict(op=op, N=N, M=M, group=rng.choice((45, 64, 128)), n=n)
    form = rng.choice(("tiny", "mid", "large"))
    if form == "tiny":
        r, c, B = rng.randrange(1, 17), rng.randrange(1, 17), _between(rng, 1, 50_000)
    elif form == "mid":
        r, c, B = _between(rng, 17, 384), _between(rng, 17, 384), _between(rng, 1, 16)
    else:
        r, c, B = _between(rng, 256, 2048), _between(rng, 256, 2048), 1
    if op == "orth":
        # 16-bit where the matrices are large: the direction is then rounded once to that type
        return dict(op=op, B=B, rows=r, cols=c, dtype="f32" if form == "tiny" else rng.choice(("bf16", "f16")))
    return dict(op=op, B=B, rows=r, cols=c, dtype=rng.choice(("f32", "bf16")), nesterov=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _rows_of(g, N, n):
    return torch.randperm(N, generator=g, device=DEV)[:n].sort().values


def _gradient(g, *shape):
    """Gradients as the rows see them: every row of its own magnitude, over several decades."""
    scale = torch.exp(2.0 * torch.randn(shape[0], 1, generator=g, device=DEV)) * 1e-4
    return torch.randn(shape, generator=g, device=DEV) * scale


def _matrices(g, B, r, c):
    """Gradients of matrices: a few strong directions over a floor of noise."""
    k = max(1, min(r, c) // 16)
    low = torch.randn(B, r, k, generator=g, device=DEV) @ torch.randn(B, k, c, generator=g, device=DEV)
    return (low / math.sqrt(k) + 0.3 * torch.randn(B, r, c, generator=g, device=DEV)) * 1e-3


def _stored(x, kind, group):
    """A store (codes, scales) holding about x, made without the operators under test."""
    N, D = x.shape
    G = -(-D // group)
    pad = torch.nn.functional.pad(x, (0, G * group - D)).view(N, G, group)
    amax = pad.abs().amax(-1)
    if kind == "int8":
        s = amax / 127.0
        q = torch.round(pad / torch.where(s > 0, s, torch.ones_like(s)).unsqueeze(-1)).clamp_(-127, 127)
        return q.view(N, -1)[:, :D].to(torch.int8).contiguous(), s
    s = _pow2_scale(amax)
    q = pad * _inverse(s).unsqueeze(-1)
    return q.view(N, -1)[:, :D].to(torch.float8_e4m3fn).contiguous(), s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    st = dict(case)
    st["seed"] = seed * 7919 + 13
    op = case["op"]
    if op in ("write", "read"):
        N, D, group = case["N"], case["D"], case["group"]
        st["codes"], st["scales"] = _stored(_gradient(g, N, D), case["kind"], group)
        st["rows"] = _rows_of(g, N, case["n"]) if case["n"] else None
        if op == "write":
            st["values"] = _gradient(g, case["n"], D).to(DTYPES[case["dtype"]])
    elif op.startswith("adam"):
        N, M, group = case["N"], case["M"], case["group"]
        st["param"] = torch.randn(N, M, generator=g, device=DEV)
        st["m"] = _stored(0.3 * _gradient(g, N, M), "e4m3", group)
        # the second moment's root is never zero where a gradient was seen
        st["r"] = _stored(_gradient(g, N, M).abs() + 1e-9, "e4m3", group)
        st["r"][0].view(torch.uint8).clamp_(min=1)
        if op == "adam_rows":
            st["rows"] = _rows_of(g, N, case["n"])
            st["grad"] = _gradient(g, case["n"], M)
        else:
            st["visible"] = torch.rand(N, generator=g, device=DEV) < 0.4
            st["grad"] = _gradient(g, N, M)
    else:
        B, r, c = case["B"], case["rows"], case["cols"]
        st["g"] = _matrices(g, B, r, c).to(DTYPES[case["dtype"]])
        if op == "update":
            st["momentum"] = 0.5 * _matrices(g, B, r, c)
            st["param"] = torch.randn(B, r, c, generator=g, device=DEV) / math.sqrt(c)
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _mask32(h):
    return h & 0xFFFFFFFF


def _uniform(seed, rows, D):
    """20 random bits in [0, 1) for each value of the rows: a hash of (seed, row, column)."""
    k = _mask32((seed & 0xFFFFFFFF) * 0x9E3779B1 + _mask32(rows) * 0x85EBCA77)
    k = _mask32((k ^ (k >> 16)) * 0x7FEB352D)
    k = _mask32((k ^ (k >> 15)) * 0x846CA68B)
    k = k ^ (k >> 16)
    h = _mask32(k.unsqueeze(1) + _mask32(torch.arange(D, device=rows.device) * 0x9E3779B1).unsqueeze(0))
    h = _mask32((h ^ (h >> 15)) * 0x2C1B3C6D)
    h = h ^ (h >> 12)
    return (h >> 12).to(torch.float32) * 2.0 ** -20


def _pow2_scale(amax):
    """The smallest power of two s (at least 2^-126) with amax / s <= 448; 0 for 0."""
    bits = amax.view(torch.int32)
    e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)
    return torch.where(amax > 0, (e.clamp(min=1) << 23).view(torch.float32), torch.zeros_like(amax))


def _inverse(s):
    """1 / s of powers of two, 0 for 0."""
    return torch.where(s > 0, ((254 << 23) - s.view(torch.int32)).view(torch.float32), torch.zeros_like(s))


def _e4m3(y, u):
    """y rounded to e4m3's values, to nearest even or (u given) down after adding u steps."""
    mag = y.abs()
    step = (mag.view(torch.int32) & 0x7F800000).clamp(min=121 << 23).view(torch.float32) * 0.125
    z = mag / step
    q = torch.round(z) if u is None else torch.floor(z + u)
    return torch.copysign(q * step, y)


def _grouped(x, group):
    n, D = x.shape
    G = -(-D // group)
    return torch.nn.functional.pad(x, (0, G * group - D)).view(n, G, group)


def _quantise(x, kind, group, u, never_zero=False):
    """Values [n, D] in 32 bits -> (codes as numbers [n, D], scales [n, G])."""
    n, D = x.shape
    p = _grouped(x, group)
    up = None if u is None else _grouped(u, group)
    amax = p.abs().amax(-1)
    if kind == "int8":
        s = amax / 127.0
        y = p / torch.where(s > 0, s, torch.ones_like(s)).unsqueeze(-1)
        y = torch.where((s > 0).unsqueeze(-1), y, torch.zeros_like(y))
        q = torch.round(y) if u is None else torch.floor(y + up)
        q = q.clamp(-127, 127)
    else:
        s = _pow2_scale(amax)
        q = _e4m3(p * _inverse(s).unsqueeze(-1), up)
        if never_zero:
            q = torch.where(p > 0, q.clamp(min=2.0 ** -9), q)
    return q.view(n, -1)[:, :D], s


def _dequantise(codes, scales, group):
    n, D = codes.shape
    return (_grouped(codes.to(torch.float32), group) * scales.unsqueeze(-1)).view(n, -1)[:, :D]


def _adam_plain(p, g, m, r, seed, rows, group, lr):
    D = p.shape[1]
    m = m * B1 + g * (1.0 - B1)
    v = (r * r) * B2 + (g * g) * (1.0 - B2)
    r = torch.sqrt(v)
    p = p - (m * lr) / (r + EPS_ADAM)
    qm = _quantise(m, "e4m3", group, _uniform(seed, rows, D))
    qr = _quantise(r, "e4m3", group, _uniform(seed ^ 0x5BF03635, rows, D), never_zero=True)
    return p, qm, qr


def _step(X):
    a, b, c = COEF
    A = X @ X.mT
    return a * X + (b * A + c * (A @ A)) @ X


def _orthogonal(u):
    X = u.mT if u.shape[-2] > u.shape[-1] else u
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + EPS_NORM)
    X = _step(_step(_step(_step(_step(X)))))
    return X.mT if u.shape[-2] > u.shape[-1] else X


LR_ADAM, LR_ORTH = 1e-4, 0.01


def run(st):
    op = st["op"]
    if own:
        return _run_own(st)
    if op == "write":
        x, rows, group = st["values"].to(torch.float32), st["rows"], st["group"]
        u = _uniform(st["seed"], rows, st["D"]) if st["dither"] else None
        q, s = _quantise(x, st["kind"], group, u)
        st["codes"][rows] = q.to(KINDS[st["kind"]])
        st["scales"][rows] = s
        if st["kind"] == "int8":
            back = _dequantise(st["codes"][rows], st["scales"][rows], group)
            return back.to(torch.bfloat16), st["scales"]
        return st["codes"], st["scales"]
    if op == "read":
        c, s = st["codes"], st["scales"]
        if st["rows"] is not None:
            c, s = c.view(torch.uint8)[st["rows"]].view(c.dtype), s[st["rows"]]
        return _dequantise(c, s, st["group"]).to(DTYPES[st["dtype"]])
    if op.startswith("adam"):
        group, (mc, ms), (rc, rs) = st["group"], st["m"], st["r"]
        if op == "adam_rows":
            rows, g = st["rows"], st["grad"]
        else:
            rows = torch.nonzero(st["visible"]).flatten()
            g = st["grad"][rows]
        m = _dequantise(mc.view(torch.uint8)[rows].view(mc.dtype), ms[rows], group)
        r = _dequantise(rc.view(torch.uint8)[rows].view(rc.dtype), rs[rows], group)
        p, (qm, sm), (qr, sr) = _adam_plain(st["param"][rows], g, m, r, st["seed"], rows, group, LR_ADAM)
        st["param"][rows] = p
        mc.view(torch.uint8)[rows] = qm.to(torch.float8_e4m3fn).view(torch.uint8)
        rc.view(torch.uint8)[rows] = qr.to(torch.float8_e4m3fn).view(torch.uint8)
        ms[rows], rs[rows] = sm, sr
        return st["param"], mc, ms, rc, rs
    g = st["g"].to(torch.float32)
    if op == "orth":
        return _orthogonal(g).to(st["g"].dtype)
    M = st["momentum"]
    M.mul_(BETA).add_(g, alpha=1.0 - BETA)
    u = g * (1.0 - BETA) + M * BETA if st["nesterov"] else M
    s = math.sqrt(max(1.0, st["rows"] / st["cols"]))
    st["param"].mul_(1.0 - LR_ORTH * DECAY).sub_(_orthogonal(u), alpha=LR_ORTH * s)
    return st["param"], M


def _run_own(st):
    from blitzgs_b200 import ops
    op = st["op"]
    if op == "write":
        ops.quant_rows_write(st["values"], st["codes"], st["scales"], st["rows"], group=st["group"],
                             seed=st["seed"] if st["dither"] else None)
        if st["kind"] == "int8":
            back = ops.quant_rows_read(st["codes"], st["scales"], st["rows"], group=st["group"], dtype=torch.bfloat16)
            return back, st["scales"]
        return st["codes"], st["scales"]
    if op == "read":
        return ops.quant_rows_read(st["codes"], st["scales"], st["rows"], group=st["group"], dtype=DTYPES[st["dtype"]])
    if op == "adam_rows":
        ops.adam8_update_rows(st["param"], st["grad"], *st["m"], *st["r"], st["rows"], LR_ADAM, B1, B2, EPS_ADAM,
                              st["N"], st["M"], group=st["group"], seed=st["seed"])
        return (st["param"], *st["m"], *st["r"])
    if op == "adam_dense":
        ops.adam8_update(st["param"], st["grad"], *st["m"], *st["r"], st["visible"], LR_ADAM, B1, B2, EPS_ADAM,
                         st["N"], st["M"], group=st["group"], seed=st["seed"])
        return (st["param"], *st["m"], *st["r"])
    if op == "orth":
        return ops.orthogonalize(st["g"], steps=5, coefficients=COEF, eps=EPS_NORM)
    ops.orthogonal_update(st["param"], st["g"], st["momentum"], LR_ORTH, beta=BETA, nesterov=st["nesterov"],
                          weight_decay=DECAY, steps=5, coefficients=COEF, eps=EPS_NORM)
    return st["param"], st["momentum"]


# ---------------------------------------------------------------------------
# work and the 64-bit definition
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("write", "read"):
        D, n = case["D"], case["n"] or case["N"]
        G = -(-D // case["group"])
        wide = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
        index = 8 * n if case["n"] else 0
        if op == "write":
            back = n * (D + 4 * G + 2 * D) if case["kind"] == "int8" else 0
            return {"bytes": n * (D * wide + D + 4 * G) + index + back, "flops": 4 * n * D}
        return {"bytes": n * (D * wide + D + 4 * G) + index, "flops": n * D}
    if op.startswith("adam"):
        M = case["M"]
        G = -(-M // case["group"])
        n = case["n"] if op == "adam_rows" else 0.4 * case["N"]
        index = 8 * n if op == "adam_rows" else case["N"]
        return {"bytes": n * (16 * M + 16 * G) + index, "flops": 20 * n * M}
    B, r, c = case["B"], case["rows"], case["cols"]
    n, m = min(r, c), max(r, c)
    wide = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    moved = B * r * c * (2 * wide if op == "orth" else wide + 16)
    return {"bytes": moved, "flops": B * 5 * (3 * n * n * m + n ** 3)}


def _pow2(e):
    """2^e in 64 bits from whole exponents."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _quantise64(x, kind, group, u, never_zero=False):
    n, D = x.shape
    p = _grouped(x, group)
    up = None if u is None else _grouped(u.double(), group)
    amax = p.abs().amax(-1, keepdim=True)
    some = amax > 0
    if kind == "int8":
        s = amax / 127.0
        y = torch.where(some, p / torch.where(some, s, torch.ones_like(s)), torch.zeros_like(p))
        q = (torch.round(y) if u is None else torch.floor(y + up)).clamp(-127, 127)
    else:
        f, e = torch.frexp(amax)
        s = torch.where(some, _pow2((e - 9 + (f > 0.875).to(e.dtype)).clamp(min=-126)), torch.zeros_like(amax))
        y = torch.where(some, p / torch.where(some, s, torch.ones_like(s)), torch.zeros_like(p))
        step = _pow2((torch.frexp(y.abs())[1] - 1).clamp(min=-6) - 3)
        z = y.abs() / step
        q = (torch.round(z) if u is None else torch.floor(z + up)) * step * torch.sign(y)
        if never_zero:
            q = torch.where((p > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return q.view(n, -1)[:, :D], s.squeeze(-1)


def _values64(codes, scales, group):
    D = codes.shape[1]
    return codes.to(torch.float32).double() * scales.double().repeat_interleave(group, 1)[:, :D]


def _orthogonal64(u):
    X = u.transpose(-1, -2) if u.shape[-2] > u.shape[-1] else u
    X = X / (torch.linalg.matrix_norm(X, keepdim=True) + EPS_NORM)
    for _ in range(5):
        A = torch.matmul(X, X.transpose(-1, -2))
        poly = COEF[1] * A + COEF[2] * torch.matmul(A, A)
        X = COEF[0] * X + torch.matmul(poly, X)
    return X.transpose(-1, -2) if u.shape[-2] > u.shape[-1] else X


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("write", "read"):
        rows = st["rows"] if st["rows"] is not None else torch.arange(case["N"], device=DEV)
        if op == "read":
            c = st["codes"].view(torch.uint8)[rows].view(st["codes"].dtype)
            return _values64(c, st["scales"][rows], case["group"])
        u = _uniform(st["seed"], rows, case["D"]) if case["dither"] else None
        q, s = _quantise64(st["values"].double(), case["kind"], case["group"], u)
        scales = st["scales"].double()
        scales[rows] = s
        if case["kind"] == "int8":
            return q * s.repeat_interleave(case["group"], 1)[:, :case["D"]], scales
        codes = st["codes"].to(torch.float32).double()
        codes[rows] = q
        return codes, scales
    if op.startswith("adam"):
        rows = st["rows"] if op == "adam_rows" else torch.nonzero(st["visible"]).flatten()
        g = (st["grad"] if op == "adam_rows" else st["grad"][rows]).double()
        group, M = case["group"], case["M"]
        pick = lambda s: _values64(s[0].view(torch.uint8)[rows].view(s[0].dtype), s[1][rows], group)  # noqa: E731
        m = B1 * pick(st["m"]) + (1 - B1) * g
        r = torch.sqrt(B2 * pick(st["r"]).square() + (1 - B2) * g.square())
        param = st["param"].double()
        param[rows] -= LR_ADAM * m / (r + EPS_ADAM)
        out = [param]
        for (codes, scales), x, salt in ((st["m"], m, 0), (st["r"], r, 0x5BF03635)):
            q, s = _quantise64(x, "e4m3", group, _uniform(st["seed"] ^ salt, rows, M), never_zero=salt != 0)
            c64, s64 = codes.to(torch.float32).double(), scales.double()
            c64[rows], s64[rows] = q, s
            out += [c64, s64]
        return tuple(out)
    g = st["g"].double()
    if op == "orth":
        return _orthogonal64(g)
    M = BETA * st["momentum"].double() + (1 - BETA) * g
    u = (1 - BETA) * g + BETA * M if case["nesterov"] else M
    s = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    return st["param"].double() * (1 - LR_ORTH * DECAY) - LR_ORTH * s * _orthogonal64(u), M
