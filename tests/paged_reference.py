"""Plain implementations of the rotary and paged-cache operators, for tests:
attention and rotation in float64; appending in the float32 steps that the
operator documents (each product, sum and quotient rounded on its own), so
that codes can be compared for equality."""

import math

import numpy as np

TOP = {"i8": np.float32(127), "e4m3": np.float32(448)}


def e4m3_values():
    """The 256 e4m3 codes' values (sign, 4 exponent bits of bias 7, 3 mantissa bits)."""
    out = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        out[c] = math.nan if (c & 127) == 127 else -v if c & 128 else v
    return out


E4M3 = e4m3_values()


def decode(codes, fmt):
    """uint8 codes as float64 values."""
    return E4M3[codes] if fmt == "e4m3" else codes.view(np.int8).astype(np.float64)


def encode(x, fmt):
    """float32 values within the codes' range to uint8 codes, nearest, ties to even."""
    if fmt == "i8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.abs(x.astype(np.float64))
    _, e = np.frexp(np.maximum(a, 2.0 ** -30))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    a = np.rint(a / step) * step
    place = np.searchsorted(E4M3[:127], a)
    assert np.array_equal(E4M3[:127][place], a)
    return (place | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def rotate(x, table, positions, layout, inverse=False, dtype=np.float64):
    """x [rows][heads][dim] with table [positions][pairs][2]."""
    y = x.astype(dtype).copy()
    cs = table[positions].astype(dtype)
    n = cs.shape[1]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1] * (-1 if inverse else 1)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if layout == "interleaved" else (slice(0, n),
                                                                                              slice(n, 2 * n))
    a, b = y[..., first].copy(), y[..., second].copy()
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y


def append(codes, scales, x, rows, lens, page_table, fmt):
    """float32 x [rows][kv heads][dim] into uint8 codes [pages][kv heads][page]
    [dim] and float32 scales, in place."""
    page, top, at = codes.shape[2], TOP[fmt], 0
    with np.errstate(divide="ignore", invalid="ignore"):
        for b, (n, m) in enumerate(zip(lens, rows)):
            for p0 in range(n - m, n):
                if p0 < 0 or (p0 > max(n - m, 0) and p0 % page):
                    continue
                stop, begin = min(n, (p0 // page + 1) * page), p0 % page
                part = x[at + p0 - (n - m):at + stop - (n - m)]
                pg = page_table[b][p0 // page]
                for h in range(codes.shape[1]):
                    z = part[:, h].astype(np.float32)
                    fine = np.isfinite(z)
                    old = scales[pg, h] if begin else np.float32(0)
                    new = max(old, np.float32(np.max(np.abs(z[fine]), initial=0) / top))
                    if new > old and begin:
                        ratio = np.float32(old / new)
                        held = decode(codes[pg, h, :begin], fmt).astype(np.float32) * ratio
                        codes[pg, h, :begin] = encode(held, fmt)
                    y = np.clip(z / new, -top, top) if new > 0 else np.zeros_like(z)
                    codes[pg, h, begin:begin + stop - p0] = encode(np.where(np.isnan(z), np.float32(0), y), fmt)
                    scales[pg, h] = new
            at += m


def attend(q, k, v, position, window, sinks, scale):
    """One row: q [heads][dim], float64 k, v [kv heads][positions][dim]; gives
    out [heads][dim], lse [heads] and the largest sum |q k| of a score."""
    heads, kv_heads = q.shape[0], k.shape[0]
    low = max(0, position + 1 - window) if window else 0
    out, lse, size = np.zeros(q.shape), np.full(heads, -np.inf), 0.0
    if position < 0:
        return out, lse, size
    for h in range(heads):
        kk, vv = k[h // (heads // kv_heads), low:position + 1], v[h // (heads // kv_heads), low:position + 1]
        s = kk @ q[h] * scale
        size = max(size, float((np.abs(kk) @ np.abs(q[h])).max() * abs(scale)))
        m = s.max()
        p = np.exp(s - m)
        lse[h] = m + math.log(p.sum())
        total = p.sum() + (math.exp(sinks[h] - m) if sinks is not None else 0.0)
        out[h] = p @ vv / total
    return out, lse, size
