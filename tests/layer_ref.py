"""The layer operators' definitions in 64 bits (numpy), for the tests."""
import numpy as np

FLT_MAX = float(np.finfo(np.float32).max)


def q8_rows(v, factor):
    """8-bit rows of v * factor: (q, scale); v in 64 bits."""
    q = np.zeros(v.shape, np.int8)
    scale = np.zeros(v.shape[0], np.float32)
    for i in range(v.shape[0]):
        top = np.max(np.abs(v[i]))  # NaN if there is one
        if top == 0:
            continue
        size = top * factor[i]
        if not size <= FLT_MAX:
            scale[i] = np.nan
        else:
            q[i] = np.rint(127.0 * v[i] / top).astype(np.int8)
            scale[i] = np.float32(size / 127.0)
    return q, scale


def norm_q8(h, w, eps):
    """h [rows, n] (already rounded to its type), in 64 bits."""
    with np.errstate(all="ignore"):
        factor = 1.0 / np.sqrt((h * h).sum(1) / h.shape[1] + eps)
        return q8_rows(h * w.astype(np.float64), factor)


def swiglu_q8(g, u):
    with np.errstate(all="ignore"):
        return q8_rows(g / (1.0 + np.exp(-g)) * u, np.ones(g.shape[0]))


def half(v, up):
    """v (not negative) in f16, rounded up or down, element by element."""
    out = np.asarray(v, np.float64).astype(np.float16)
    with np.errstate(over="ignore"):
        wrong = out.astype(np.float64) < v if up else out.astype(np.float64) > v
        to = np.nextafter(out, np.float16(np.inf if up else -np.inf))
    return np.where(wrong, to, out)


def row_bytes(cols):
    return (cols + 31) // 32 * 16


def pack(q, fill=0):
    """[rows, cols] of 4-bit numbers in the layout of lal_tail_q4.d_q."""
    rows, cols = q.shape
    full = np.full((rows, row_bytes(cols) * 2), fill, np.uint8)
    full[:, :cols] = q
    b = full.reshape(rows, -1, 2, 16)
    return (b[:, :, 0] | (b[:, :, 1] << 4)).reshape(rows, -1)


def unpack(p, cols):
    b = p.reshape(p.shape[0], -1, 16)
    return np.stack([b & 15, b >> 4], 2).reshape(p.shape[0], -1)[:, :cols]


def quantize_q4(w, group, minimum):
    """w [rows, cols] in 64 bits: (q, scale, min or None)."""
    rows, cols = w.shape
    groups = -(-cols // group)
    q = np.full((rows, cols), 0 if minimum else 8, np.uint8)
    scale = np.zeros((rows, groups), np.float16)
    low = np.zeros((rows, groups), np.float16) if minimum else None
    for g in range(groups):
        c = slice(g * group, min(cols, (g + 1) * group))
        v = w[:, c]
        bad = ~np.isfinite(v).all(1)
        v = np.where(bad[:, None], 0.0, v)
        if minimum:
            lo, hi = v.min(1), v.max(1)
            m = np.where(lo < 0, -half(np.maximum(-lo, 0), True), half(np.maximum(lo, 0), False))
            bad |= np.isinf(m)
            m64 = np.where(np.isinf(m), 0, m).astype(np.float64)
            s = half((hi - m64) / 15.0, True)
        else:
            m64 = np.zeros(rows)
            s = half(np.abs(v).max(1) / 7.0, True)
        bad |= np.isinf(s)
        ok = ~bad & (s > 0)
        n = np.rint((v - m64[:, None]) / np.where(ok, s, 1).astype(np.float64)[:, None])
        q[:, c] = np.where(ok[:, None], n if minimum else n + 8, 0 if minimum else 8)
        scale[:, g] = np.where(bad, np.nan, s)
        if minimum:
            low[:, g] = np.where(bad, np.nan, m)
    return q, scale, low


def weights_q4(q, scale, low, group):
    """The weights that (q, scale, low) stand for, in 64 bits."""
    of = np.arange(q.shape[1]) // group
    s = scale.astype(np.float64)[:, of]
    if low is None:
        return s * (q.astype(np.float64) - 8.0)
    return s * q + low.astype(np.float64)[:, of]


def matvec_q4(xq, sx, q, scale, low, group):
    """(y, the sum of its terms' sizes) in 64 bits, [streams, rows]: what each
    group of each block of 32 columns adds, for the error bound."""
    x, y, size = xq.astype(np.float64), 0.0, 0.0
    cols = q.shape[1]
    for c in range(0, cols, 32):
        k = slice(c, min(cols, c + 32))
        s = scale[:, c // group].astype(np.float64)
        if low is None:
            parts = [x[:, k] @ (q[:, k].astype(np.float64) - 8.0).T * s]
        else:
            parts = [x[:, k] @ q[:, k].astype(np.float64).T * s,
                     x[:, k].sum(1)[:, None] * low[:, c // group].astype(np.float64)]
        for p in parts:
            y, size = y + p, size + np.abs(p)
    sx = sx.astype(np.float64)[:, None]
    return y * sx, size * np.abs(sx)
