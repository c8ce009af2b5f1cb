"""The microscaled formats, their products and the routing in float64 NumPy, for the tests.

mxfp4: E = clamp(floor(log2 max|x|) - 2, -127, 127) per 32 values, e2m1 codes of x / 2^E.  nvfp4: s = e4m3(max|x / t| / 6)
per 16 values, e2m1 codes of x / t / s.  Nearest, ties to the even code, saturating; a block with a NaN or an infinity
stands for NaNs.
"""
import numpy as np

BLOCK = {"mxfp4": 32, "nvfp4": 16}
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127])


def _nearest(grid, a):
    """Index of the grid value nearest to each a >= 0, ties to the even index, past the last: the last."""
    hi = np.searchsorted(grid, a).clip(1, len(grid) - 1)
    up, dn = grid[hi] - a, a - grid[hi - 1]
    return np.where((up < dn) | ((up == dn) & (hi % 2 == 0)), hi, hi - 1)


def auto_scale(x):
    """The smallest power of two t (at least 2^-126) with max|x| / t <= 2688 over the finite values; 1 for zeros."""
    a = np.abs(np.asarray(x, np.float64))
    top = a[np.isfinite(a)].max(initial=0.0)
    if top == 0:
        return 1.0
    e = -126
    while top > 2688 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def quantize(x, fmt, t=1.0):
    """(codes [R, Kp] of 0..15, scale bytes [R, blocks], values [R, K] in float64) of float rows, K padded to 32."""
    x = np.asarray(x, np.float64)
    R, K = x.shape
    b, Kp = BLOCK[fmt], -(-K // 32) * 32
    v = np.zeros((R, Kp))
    v[:, :K] = x
    v = v.reshape(R, -1, b)
    if fmt == "nvfp4":
        v = (v / t).astype(np.float32).astype(np.float64)
    a = np.abs(v).max(-1)
    bad = ~np.isfinite(np.abs(x)).all() and ~np.isfinite(np.pad(np.abs(x), ((0, 0), (0, Kp - K))).reshape(R, -1, b)).all(-1)
    bad = np.broadcast_to(bad, a.shape)
    a = np.where(bad, 0, a)
    v = np.where(bad[..., None], 0, v)
    if fmt == "mxfp4":
        with np.errstate(divide="ignore"):
            e = np.where(a > 0, np.frexp(a)[1] - 1 - 2, -127).clip(-127, 127).astype(int)
        byte, d = e + 127, 2.0 ** e
    else:
        byte = _nearest(E4M3, np.minimum(a / 6, 448.0))
        d = E4M3[byte]
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(d[..., None] > 0, v / d[..., None], 0.0)
    i = _nearest(GRID, np.minimum(np.abs(q), 6.0))
    code = i | (np.signbit(v) << 3)
    val = np.where(np.signbit(v), -GRID[i], GRID[i]) * d[..., None] * (t if fmt == "nvfp4" else 1.0)
    val = np.where(bad[..., None], np.nan, val)
    byte = np.where(bad, 255 if fmt == "mxfp4" else 127, byte)
    return code.reshape(R, Kp), byte.astype(np.uint8), val.reshape(R, Kp)[:, :K]


def values(codes, scales, K, fmt, t=1.0):
    """Values of packed rows: codes uint8 [R, bytes] (even element low), scale bytes [R, blocks]."""
    q = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)[:, :K]
    s = scales.astype(int)
    d = np.where(s == 255, np.nan, 2.0 ** (s - 127.0)) if fmt == "mxfp4" else np.append(E4M3, np.nan)[s & 127] * t
    d = np.repeat(d, BLOCK[fmt], -1)[:, :K]
    return np.where(q >= 8, -GRID[q & 7], GRID[q & 7]) * d


def route(logits, k, normalize):
    lg = np.asarray(logits, np.float64)
    lg = np.where(np.isnan(lg), -np.inf, lg)
    T, E = lg.shape
    order = np.argsort(-lg, axis=1, kind="stable")[:, :k]
    m = lg.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        p = np.where(lg == m, 1.0, np.exp(lg - m))
    p = np.where(m == -np.inf, 0.0, p)
    best = np.take_along_axis(p, order, 1)
    den = (best if normalize else p).sum(1, keepdims=True)
    w = np.where(den > 0, best / np.where(den > 0, den, 1), 0.0)
    flat = order.reshape(-1)
    at = np.argsort(flat, kind="stable")
    slots = np.empty_like(at)
    slots[at] = np.arange(at.size)
    offsets = np.concatenate(([0], np.cumsum(np.bincount(flat, minlength=E))))
    return w, order, offsets, at // k, slots.reshape(T, k)


def combine(z, w, slots):
    z, w = np.asarray(z, np.float64), np.asarray(w, np.float64)
    y = np.zeros((w.shape[0], z.shape[1]))
    for j in range(w.shape[1]):
        on = w[:, j] != 0
        y[on] += w[on, j, None] * z[slots[on, j]]
    return y
