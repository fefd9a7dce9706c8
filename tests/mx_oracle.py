"""Block-scaled 4-bit matrices in numpy, written from the definition in include/b200const.h: quotients are rounded to
32 bits where the header says so, everything else is 64 bits wide."""
import numpy as np

BLOCK = {1: 32, 2: 16}  # by format: mxfp4, nvfp4
MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def e2m1(q):
    """64-bit values -> codes: the nearest magnitude, the even code of two that are equally near, the sign in bit 3."""
    a = np.minimum(np.abs(q), 64.0)[..., None]  # beyond 6 all is 6; very large numbers would be equally far from every code
    far = np.abs(a - MAGNITUDES)
    best = far.min(-1, keepdims=True)
    near = far == best
    rank = np.where(near, np.arange(8) % 2, 9)  # even codes first
    return (np.argmin(rank, -1) | (np.signbit(q).astype(np.int64) << 3)).astype(np.uint8)


def e4m3(v):
    """Non-negative 64-bit values up to 448 -> bytes, to nearest even."""
    table = e4m3_values()[:127]  # ascending
    low = np.clip(np.searchsorted(table, v, side="right") - 1, 0, 126)
    high = np.minimum(low + 1, 126)
    down, up = v - table[low], table[high] - v
    pick = np.where(down < up, low, np.where(up < down, high, np.where(low % 2 == 0, low, high)))
    return pick.astype(np.uint8)


def e4m3_values():
    b = np.arange(256)
    e, f = (b >> 3) & 15, (b & 7).astype(np.float64)
    v = np.where(e > 0, 2.0 ** (e - 7.0) * (1 + f / 8), f * 2.0 ** -9)
    v = np.where(b >= 128, -v, v)
    v[[127, 255]] = np.nan
    return v


def tensor_scale_of(top):
    t = 2.0 ** -126
    while top > 2688.0 * t:
        t *= 2.0
    if top > 0:
        return np.float32(t)
    return np.float32(1.0)


def quantize(x, fmt, t=None):
    """x: float32 or float64 [rows, cols] holding the input's values.  -> dict of codes [rows, cols], scale bytes
    [rows, blocks], t, top, and the 64-bit values they stand for."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    b = BLOCK[fmt]
    blocks = -(-cols // b)
    v = np.zeros((rows, blocks * b))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, b)
    finite = np.isfinite(v)
    bad = ~finite.all(2)
    top_all = float(np.abs(np.where(finite, v, 0)).max()) if v.size else 0.0
    amax = np.abs(np.where(finite, v, 0)).max(2) if cols else np.zeros((rows, 0))
    clean = np.where(bad[..., None], 0.0, v)
    if fmt == 1:
        _, e = np.frexp(amax)
        X = np.where(amax > 0, np.maximum(e - 1 - 2, -127), -127)
        scales = np.where(bad, 255, X + 127).astype(np.uint8)
        d = np.where(bad, np.nan, 2.0 ** X.astype(np.float64))
        codes = e2m1(clean / np.where(bad, 1.0, d)[..., None])
        codes[bad] = 0
        t = top = None
    else:
        t = tensor_scale_of(top_all) if t is None else np.float32(t)
        top = np.float32(top_all)
        with np.errstate(over="ignore", under="ignore"):
            s = (amax.astype(np.float32) / (np.float32(6) * t)).astype(np.float32)
            scales = e4m3(np.minimum(s.astype(np.float64), 448.0))
            scales[bad] = 127
            d32 = (e4m3_values()[scales].astype(np.float32) * t).astype(np.float32)
            use = ~bad & (d32 > 0)
            q = (clean.astype(np.float32) / np.where(use, d32, 1)[..., None]).astype(np.float32)
        codes = e2m1(q.astype(np.float64))
        codes[~use] = 0
        d = d32.astype(np.float64)
    values = (decode(codes) * d[..., None]).reshape(rows, -1)[:, :cols]
    return dict(codes=codes.reshape(rows, -1)[:, :cols], scales=scales, t=t, top=top, values=values, fmt=fmt)


def decode(codes):
    return np.where(codes & 8, -1.0, 1.0) * MAGNITUDES[codes & 7]


def values_of(codes, scales, fmt, t=None):
    """64-bit values of codes [rows, cols] and scale bytes [rows, blocks]."""
    b = BLOCK[fmt]
    if fmt == 1:
        s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    else:
        s = e4m3_values()[scales] * np.float64(t)
    return decode(codes) * np.repeat(s, b, 1)[:, :codes.shape[1]]


def pack(codes, ld=None):
    """codes [rows, cols] -> bytes [rows, 16 * ceil(cols / 32)]."""
    rows, cols = codes.shape
    full = np.zeros((rows, -(-cols // 32) * 32), np.uint8)
    full[:, :cols] = codes
    return (full[:, 0::2] | (full[:, 1::2] << 4)).astype(np.uint8)


def lay(scales, layout):
    """Scale bytes [rows, blocks] as stored: in rows (0), or in tiles of 128 rows x 4 blocks (1)."""
    if layout == 0:
        return scales.reshape(-1).copy()
    rows, blocks = scales.shape
    chunks = -(-blocks // 4)
    out = np.zeros(-(-rows // 128) * chunks * 512, np.uint8)
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None]
    out[((r // 128) * chunks + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4] = scales
    return out
