"""Plain 64-bit restatements of the paged 4-bit cache, the attention over it and sampling, for the tests.

Cache bytes are numpy arrays as the library lays them out: codes [page][head][slot][D / 2], scales
[page][head][slot][D / 16]."""
import numpy as np

E4M3 = np.array([(b & 7) * 2.0 ** -9 if b < 8 else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7) for b in range(127)] + [np.nan])


def nearest(y, grid):
    """Index of the nearest grid point to y >= 0, the even index when halfway."""
    hi = np.clip(np.searchsorted(grid, y), 1, len(grid) - 1)
    lo = hi - 1
    a, b = y - grid[lo], grid[hi] - y
    return np.where((b < a) | ((b == a) & (hi % 2 == 0)), hi, lo)


def quantise(x, unit=1.0):
    """FP32 [..., D] -> (codes [..., D / 2], scales [..., D / 16]) bytes."""
    x = np.asarray(x, np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        g = (x if unit == 1.0 else x / np.float32(unit)).astype(np.float64)
    g = g.reshape(*g.shape[:-1], g.shape[-1] // 16, 16)
    amax = np.max(np.abs(g), -1)
    fine = np.isfinite(amax)
    s = np.where(fine, nearest(np.minimum(np.where(fine, amax, 0) / 7, 448), E4M3[:127]), 127)
    scale = np.where(fine & (s > 0), E4M3[s], np.inf)[..., None]
    y = np.where(np.isfinite(g), g, 0) / scale
    c = (np.clip(np.rint(y), -7, 7) + 8).reshape(*x.shape).astype(np.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), s.astype(np.uint8)


def values(codes, scales, unit=1.0):
    c = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    v, s = c.astype(np.float64) - 8, E4M3[scales]
    v = v.reshape(*s.shape, 16) * s[..., None]
    return v.reshape(*c.shape) * float(np.float32(unit))


def rotate(x, pos, base):
    """[T, H, D] by the angles of its positions, pairs (2c, 2c + 1)."""
    x = np.asarray(x, np.float64)
    d = x.shape[-1]
    a = np.asarray(pos, np.float64)[:, None, None] * float(base) ** (-np.arange(0, d, 2) / d)
    y = np.empty_like(x)
    y[..., 0::2] = x[..., 0::2] * np.cos(a) - x[..., 1::2] * np.sin(a)
    y[..., 1::2] = x[..., 0::2] * np.sin(a) + x[..., 1::2] * np.cos(a)
    return y


def attention(q, k, v, limits):
    """q [n, Hq, D], k and v [len, Hkv, D]; row i sees keys 0 .. limits[i] - 1; no key: zeros. Also returns the
    largest sum of |q||k| / sqrt(D) over a row's keys, which bounds the scores' rounding."""
    n, hq, d = q.shape
    g = hq // k.shape[1]
    out, size = np.zeros((n, hq, d)), 0.0
    for i in range(n):
        for h in range(hq):
            if limits[i] <= 0:
                continue
            kk, vv = k[:limits[i], h // g], v[:limits[i], h // g]
            s = kk @ q[i, h] / np.sqrt(d)
            size = max(size, float(np.max(np.abs(kk) @ np.abs(q[i, h]))) / np.sqrt(d))
            p = np.exp(s - np.max(s))
            out[i, h] = p @ vv / p.sum()
    return out, size


def kept(x, temperature, top_k, top_p, min_p):
    """Weights of a row of logits with 0 for what the filters drop, and the kept mask; None: nothing to draw from."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    m = x.max()
    if m == -np.inf:
        return None
    with np.errstate(invalid="ignore"):
        w = np.where(x == m, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - m) / temperature)))
    order = np.lexsort((np.arange(len(x)), -x))
    ws = w[order]
    rank = np.arange(len(x))
    keep = np.ones(len(x), bool)
    if top_k > 0:
        keep &= rank < top_k
    if min_p > 0:
        keep &= ws >= min(min_p, 1.0)
    mass = np.cumsum(np.where(keep, ws, 0.0))
    if top_p < 1:
        keep &= (np.concatenate(([0.0], mass[:-1])) < top_p * mass[-1]) | (rank == 0)
    mask = np.zeros(len(x), bool)
    mask[order[keep]] = True
    return np.where(mask, w, 0.0), mask


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, distance of u from the nearer border of that token as a part of the kept mass)."""
    xs = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    if xs.max() == -np.inf:
        return -1, 1.0
    if not temperature > 0:
        return int(np.argmax(xs)), 1.0
    w, mask = kept(x, temperature, top_k, top_p, min_p)
    c = np.cumsum(w)
    t = u * c[-1]
    i = int(np.searchsorted(c, t, side="right"))
    last = int(np.flatnonzero(w > 0)[-1])
    if i > last:
        return last, 1.0
    return i, float(min(c[i] - t, t - (c[i] - w[i])) / c[-1])
