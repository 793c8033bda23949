"""The shared pool of cached keys and values restated in numpy: rows by their fp32 definition, attention in 64 bits.  Shares nothing with the library."""
import numpy as np

CENTROIDS = np.array([-127, -96, -75, -58, -44, -31, -18, -6, 6, 18, 31, 44, 58, 75, 96, 127], np.float32)
F = np.float32


def signs(d):
    out = []
    for i in range(d):
        m = (1 << 64) - 1
        z = (0x9E3779B97F4A7C15 + (i // 64) * 0xBF58476D1CE4E5B9 + (i % 64 + 1) * 0x9E3779B97F4A7C15) & m
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & m
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & m
        out.append(-1.0 if (z ^ (z >> 31)) & 1 else 1.0)
    return np.array(out, F)


def butterflies(x):
    x, h = x.copy(), 1
    while h < 64:
        y = x.reshape(*x.shape[:-1], x.shape[-1] // (2 * h), 2, h)
        a, b = y[..., 0, :].copy(), y[..., 1, :].copy()
        y[..., 0, :], y[..., 1, :] = a + b, a - b
        h *= 2
    return x


def rotate(x):
    with np.errstate(invalid="ignore", over="ignore"):
        return butterflies(x * signs(x.shape[-1]).astype(x.dtype) * x.dtype.type(0.125))


def rotate_back(r):
    with np.errstate(invalid="ignore"):
        return butterflies(r) * r.dtype.type(0.125) * signs(r.shape[-1]).astype(r.dtype)


def quant8(r):
    """(codes, scales) of transformed fp32 rows: scale NaN and codes 0 where a value is not finite."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        bad = ~np.isfinite(r).all(-1)
        top = np.abs(r).max(-1)
        zero = (top <= F(1.1920929e-07)) | bad
        code = np.where(zero[..., None], F(0), np.rint(r * (F(127) / top)[..., None]))
        return code, np.where(bad, F(np.nan), np.where(zero, F(0), top / F(127))).astype(F)


def nearest(y):
    p = np.searchsorted(np.array([12, 24.5, 37.5, 51, 66.5, 85.5, 111.5], F), np.abs(y), side="right")
    return np.where(y >= 0, 8 + p, 7 - p)


def quant4(r):
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        bad = ~np.isfinite(r).all(-1)
        g = r.reshape(*r.shape[:-1], r.shape[-1] // 64, 64)
        top = np.abs(g).max(-1)
        zero = (top < F(1e-30)) | bad[..., None]
        g = np.where(zero[..., None], F(0), g)
        c = CENTROIDS[nearest(g * (F(127) / np.where(zero, F(1), top))[..., None])]
        num = np.zeros(top.shape, F)
        for i in range(64):
            num = num + g[..., i] * c[..., i]
        den = (c * c).sum(-1)
        fit = np.where((den > F(1e-12)) & (num > 0), num / den, top / F(127)).astype(F)
        bits = fit.view(np.uint32)
        s = (((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(F)
        inv = np.where(s > F(1e-30), F(1) / s, F(0)).astype(F)
        idx = np.where(zero[..., None], 8, nearest(g * inv[..., None]))
        s = np.where(bad[..., None], F(np.nan), np.where(zero, F(0), s)).astype(F)
        return CENTROIDS[idx].reshape(r.shape), s


def stored(x, bits):
    """Rows as they are kept, still transformed (fp32)."""
    code, scale = (quant8 if bits == 8 else quant4)(rotate(x.astype(F)))
    with np.errstate(invalid="ignore"):
        if bits == 8:
            return code * scale[..., None]
        return (code.reshape(*code.shape[:-1], code.shape[-1] // 64, 64) * scale[..., None]).reshape(code.shape)


def read_back(x, bits):
    return rotate_back(stored(x, bits))


def attend(q, k, v, scale, half):
    """One token: q [heads][d], k / v [rows][kv heads][d] transformed rows -> (out, bound of each 64 values' distance in the 2-norm).
    The bound: a query operand is off by at most `half` of its value (2^-11 for one half, 2^-21 for two), a weight's exponent by a few
    roundings of numbers below 64 (2^-17 together), a weight by `half`; a sum of weights times values by these times the sum of magnitudes."""
    heads, d = q.shape
    kh = k.shape[1]
    out, bound = np.zeros((heads, d)), np.zeros((heads, d // 64))
    if k.shape[0]:
        qr = rotate(q.astype(np.float64))
        for h in range(heads):
            kk, vv = k[:, h * kh // heads].astype(np.float64), v[:, h * kh // heads].astype(np.float64)
            s = kk @ qr[h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h] = rotate_back(p @ vv)
            off = np.expm1(2 * (np.abs(kk) @ np.abs(qr[h])).max() * scale * half + 2.0 ** -17) + half
            bound[h] = np.linalg.norm((off * (p @ np.abs(vv))).reshape(-1, 64), axis=-1)
    return out, bound


def block_key(k):
    """(codes, scale) of a whole page's transformed keys [rows][kv heads][d]."""
    total = np.zeros(k.shape[1:], F)
    for row in k:
        with np.errstate(invalid="ignore"):
            total = total + row
    return quant8(total * F(1 / len(k)))


def select(q, keys, scales, pages, top, sinks, local):
    """One token: q [heads][d] fp32, keys [pages][kv heads][d], scales [pages][kv heads] of its whole pages -> [kv heads][top]."""
    kh, d = keys.shape[1:]
    g = q.shape[0] // kh
    out = np.full((kh, top), -1, np.int32)
    for h in range(kh):
        total = q[h * g].astype(F)
        for i in range(1, g):
            total = total + q[h * g + i].astype(F)
        code, _ = quant8(rotate(total))
        ids = list(range(pages))
        if pages > top:
            free = [i for i in ids if sinks <= i < pages - local]
            with np.errstate(invalid="ignore"):
                score = [F(code.astype(np.float64) @ keys[i, h].astype(np.float64)) * scales[i, h] for i in free]
            order = sorted(range(len(free)), key=lambda j: (np.isnan(score[j]), -score[j] if not np.isnan(score[j]) else 0, j))
            best = {free[j] for j in order[:top - sinks - local]}
            ids = [i for i in ids if i < sinks or i >= pages - local or i in best]
        out[h, :len(ids)] = ids
    return out
