"""The cached-attention operators in 64 bits, from their definitions, with bounds on what fp32 arithmetic and the stated
roundings to fp16 may move a result by (u = 2^-24, h = 2^-11: half a unit in the last place of fp32 and fp16)."""
import numpy as np

U, HU, TINY = 2.0 ** -24, 2.0 ** -11, 2.0 ** -25


def rotate(x, pos, rd, pairs, freq):
    """x [n][heads][dk] at positions pos [n]: values and the error of 32-bit arithmetic on exact angles. cos and sin are off by
    the reduced angle's rounding (0.8 u), the series' five roundings of values up to 1 (3 u) and its rest (0.04 u); the two
    products and their sum by 2 u more."""
    y, err = x.astype(np.float64), np.zeros(x.shape)
    if rd:
        e = np.arange(rd // 2)
        i, j = (2 * e, 2 * e + 1) if pairs else (e, e + rd // 2)
        a = (np.asarray(pos, np.float64)[:, None] * freq.astype(np.float64))[:, None]
        c, s = np.cos(a), np.sin(a)
        u, v = y[..., i].copy(), y[..., j].copy()
        y[..., i], y[..., j] = u * c - v * s, u * s + v * c
        err[..., i] = err[..., j] = 6 * U * (np.abs(u) + np.abs(v))
    return y, err


def attention(q, k, v, seen, scale, part):
    """q [n][H][dk], k [L][Hk][dk], v [L][Hk][dv], seen [n][Hk][L] -> o [n][H][dv] and its error bound. `part`: what the
    weights are rounded by as factors (0 in fp32), relative to them; what is below the largest one's smallest unit is lost."""
    n, H, dk = q.shape
    L, hk, dv = v.shape
    o, err = np.zeros((n, H, dv)), np.zeros((n, H, dv))
    q = q.astype(np.float64)
    for h in range(H):
        g = h * hk // H
        on = seen[:, g]
        some = on.any(0)[:, None]
        kk, vv = np.where(some, k[:, g], 0).astype(np.float64), np.where(some, v[:, g], 0).astype(np.float64)
        s, mag = scale * (q[:, h] @ kk.T), abs(scale) * (np.abs(q[:, h]) @ np.abs(kk).T)
        s = np.where(on, s, -np.inf)
        with np.errstate(all="ignore"):
            m = s.max(1, keepdims=True) if L else np.zeros((n, 1))
            m = np.where(m == -np.inf, 0, m)
            e = np.exp(s - m)
            total = e.sum(1, keepdims=True)
            w = np.where(on, e / np.where(total == 0, 1, total), 0)
            far = np.where(on, np.abs(s - m), 0)
            rel = (dk + 2) * U * mag + U * (2 * np.abs(np.where(on, s, 0)) + 2.5 * far + 20 + 0.1 * L)
            fine = np.where(np.isfinite(vv), vv, 0)
            o[:, h] = w @ fine
            # a value that is not finite reaches those that see it
            for j, d in zip(*np.nonzero(~np.isfinite(vv))):
                o[on[:, j], h, d] += w[on[:, j], j] * vv[j, d]
            size = w @ np.abs(fine)
            small = (2.0 ** -37 if part else 0) * (on @ np.abs(fine)) / np.where(total == 0, 1, total)
            err[:, h] = (w * rel) @ np.abs(fine) + (w * rel).sum(1, keepdims=True) * np.abs(o[:, h]) + part * size + small + \
                (2 * L + 20) * U * size
    return o, err


def scores(q, lo, hi):
    """q [H][dk], lo, hi [pages][Hk][dk] -> [Hk][pages]"""
    hk = lo.shape[1]
    q = q.astype(np.float64).reshape(hk, -1, 1, q.shape[-1])
    lo, hi = (x.astype(np.float64).transpose(1, 0, 2)[:, None] for x in (lo, hi))
    with np.errstate(all="ignore"):
        return (q * np.where(q >= 0, hi, lo)).sum((1, 3))


def select(q, lo, hi, there, at, page, window, first, last, n):
    """A row's pages by head of keys [Hk][n]; lo, hi [pages of the sequence][Hk][dk], there [pages]"""
    s = scores(q, lo, hi)
    i = np.arange(len(there))
    s = np.where(np.isnan(s), -np.inf, s)
    forced = (i < first) | (i > at // page - last)  # above any score, +infinity too
    can = there & (i * page <= at) & (((i + 1) * page > at - window + 1) if window else True)
    out = np.full((len(s), n), -1, np.int32)
    for g in range(len(s)):
        mine = sorted(i[can], key=lambda x: (not forced[x], -s[g, x], x))[:n]
        out[g, :len(mine)] = sorted(mine)
    return out
