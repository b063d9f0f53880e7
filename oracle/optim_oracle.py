"""CPU restatement (numpy) of the 8-bit row store, the Adam step on it and the
orthogonalised updates.  Codes are formed in the float32 arithmetic the format
is defined in (single IEEE operations), everything else in 64 bits."""
import numpy as np

ROOT_SALT = 0x5BF03635


def row_uniforms(seed, rows, D):
    """float32 [n, D]: 20 bits of a hash of (seed, row, column), in [0, 1)."""
    with np.errstate(over="ignore"):
        u32 = np.uint32
        r = np.asarray(rows, np.int64).astype(np.uint64).astype(u32)
        k = u32(seed & 0xFFFFFFFF) * u32(0x9E3779B1) + r * u32(0x85EBCA77)
        k = (k ^ (k >> u32(16))) * u32(0x7FEB352D)
        k = (k ^ (k >> u32(15))) * u32(0x846CA68B)
        k = k ^ (k >> u32(16))
        h = k[:, None] + np.arange(D, dtype=u32)[None, :] * u32(0x9E3779B1)
        h = (h ^ (h >> u32(15))) * u32(0x2C1B3C6D)
        h = h ^ (h >> u32(12))
    return (h >> u32(12)).astype(np.float32) * np.float32(2.0 ** -20)


def e4m3_values():
    """float64 [256]: the value of every e4m3 byte (NaN for 0x7f and 0xff)."""
    out = np.empty(256)
    for c in range(256):
        s, e, m = (-1.0 if c & 128 else 1.0), (c >> 3) & 15, c & 7
        out[c] = s * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    out[127] = out[255] = np.nan
    return out


def _round_e4m3(y, u, never_zero):
    """float32 |y| <= 448 -> e4m3 values (float32), nearest even or dithered by u."""
    mag = np.abs(y)
    with np.errstate(divide="ignore"):
        e = np.where(mag > 0, np.frexp(mag)[1] - 1, -6)
    step = np.ldexp(np.float32(1), np.maximum(e, -6) - 3).astype(np.float32)
    z = mag.astype(np.float64) / step
    q = np.rint(z) if u is None else np.floor(z + u)
    q = q.astype(np.float32)
    v = np.copysign((q * step).astype(np.float32), y)
    return np.where(y > 0, np.maximum(v, np.float32(2.0 ** -9)), v) if never_zero else v


def quantise(x, kind, group, u=None, never_zero=False):
    """float32 [n, D] -> (code numbers float32 [n, D], scales float32 [n, G])."""
    x = np.asarray(x, np.float32)
    n, D = x.shape
    G = -(-D // group)
    codes, scales = np.zeros((n, D), np.float32), np.zeros((n, G), np.float32)
    for g in range(G):
        sl = slice(g * group, min(D, (g + 1) * group))
        p = x[:, sl]
        ok = np.isfinite(p).all(1)
        p = np.where(ok[:, None], p, np.float32(0))
        amax = np.abs(p).max(1) if p.size else np.zeros(n, np.float32)
        uu = None if u is None else u[:, sl]
        if kind == "int8":
            s = (amax / np.float32(127)).astype(np.float32)
            with np.errstate(over="ignore"):  # a step less where 127 s would pass the largest float
                s = np.where(np.isfinite(s * np.float32(127)), s, np.nextafter(s, np.float32(0)))
            y = np.divide(p, s[:, None], out=np.zeros_like(p), where=s[:, None] > 0)
            q = np.rint(y) if u is None else np.floor((y + uu).astype(np.float32))
            q = np.clip(q, -127, 127)
        else:
            f, e = np.frexp(amax.astype(np.float64))
            k = np.maximum(np.where(f > 0.875, e - 8, e - 9), -126)
            s = np.where(amax > 0, np.ldexp(1.0, k), 0.0).astype(np.float32)
            y = np.where(amax[:, None] > 0, np.ldexp(p.astype(np.float64), -k[:, None]), 0.0).astype(np.float32)
            q = _round_e4m3(y, uu, never_zero)
            top = np.where(k == 120, np.float32(240), np.float32(448))[:, None]  # 256 * 2^120 is no float
            q = np.clip(q, -top, top)
        codes[:, sl], scales[:, g] = q, np.where(ok, s, np.float32(np.nan))
        codes[:, sl][~ok] = 0
    return codes, scales


def dequantise(codes, scales, group):
    """float32 values of code numbers and scales."""
    D = codes.shape[1]
    return (codes.astype(np.float32) * np.repeat(scales, group, 1)[:, :D]).astype(np.float32)


def adam8(param, grad, m, r, rows, lr, b1, b2, eps, seed, group):
    """One step of the rows listed: param [N, M], grad [n, M], m and r the rows'
    stored values [n, M].  Returns (param rows, (m codes, scales), (r codes, scales))
    in the kernel's order of single float32 operations."""
    f = np.float32
    b1c, b2c = f(1.0 - b1), f(1.0 - b2)
    lr, b1, b2, eps = f(lr), f(b1), f(b2), f(eps)
    m = m * b1 + grad * b1c
    r = np.sqrt((r * r) * b2 + (grad * grad) * b2c)
    p = param[rows] - (m * lr) / (r + eps)
    D = param.shape[1]
    return (p, quantise(m, "e4m3", group, row_uniforms(seed, rows, D)),
            quantise(r, "e4m3", group, row_uniforms(seed ^ ROOT_SALT, rows, D), never_zero=True))


def orthogonalize(u, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """Newton-Schulz steps of [..., rows, cols] in 64 bits."""
    X = np.asarray(u, np.float64)
    tall = X.shape[-2] > X.shape[-1]
    if tall:
        X = np.swapaxes(X, -1, -2)
    a, b, c = (float(np.float32(v)) for v in coefficients)
    X = X / (np.sqrt((X * X).sum((-2, -1), keepdims=True)) + float(np.float32(eps)))
    for _ in range(steps):
        A = X @ np.swapaxes(X, -1, -2)
        X = a * X + (b * A + c * (A @ A)) @ X
    return np.swapaxes(X, -1, -2) if tall else X
