"""The temporal context operators in 64 bits, from their definitions, with bounds on what fp32 sums and the stated
roundings to fp16 may move a result by. u = 2^-24 and h = 2^-11: half a unit in the last place of fp32 and fp16."""
import numpy as np

U, HU, TINY = 2.0 ** -24, 2.0 ** -11, 2.0 ** -25


def act(z, a):
    z = np.asarray(z, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        s = 1 / (1 + np.exp(-z))
        return {0: z, 1: z * s, 2: np.maximum(z, 0), 3: s}[a]


def norm(u, kind, eps, w, b):
    """(values, error of 32-bit arithmetic on them) of one norm over the last axis."""
    c = u.shape[-1]
    if kind == 0:
        return u, np.zeros_like(u)
    mean = u.mean(-1, keepdims=True) if kind == 2 else 0.0
    d = u - mean
    r = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    w = np.ones(c) if w is None else w.astype(np.float64)
    b = np.zeros(c) if b is None else b.astype(np.float64)
    # up to 32 terms a lane and a tree of at most 10: 42 roundings a sum; the mean's error stays in every difference
    lost = (np.abs(u) * 2 + 44 * np.abs(u).mean(-1, keepdims=True)) * U if kind == 2 else 2 * np.abs(u) * U
    dr = 30 * U + r * r * (np.abs(d) * lost).mean(-1, keepdims=True)  # of r, relative
    y = d * r * w
    return y + b, np.abs(w) * r * (lost + np.abs(d) * (dr + 4 * U)) + U * np.abs(y + b)


def block_norm(f, post, gate, gact, scale, rs, x, pre):
    """y, n and their 32-bit errors; post / pre are (kind, eps, w, b)."""
    shape = (f if f is not None else x).shape
    y, dy = (np.zeros(shape),) * 2 if x is None else (x.astype(np.float64), np.zeros(shape))
    if f is not None:
        v, dv = norm(f.astype(np.float64), *post)
        g = np.ones(1) if gate is None else act(gate, gact)
        dg = 0.0 if gate is None or gact in (0, 2) else (np.abs(gate.astype(np.float64)) * 3 + 6) * U * np.abs(g)
        k = rs * (np.ones(shape[-1]) if scale is None else scale.astype(np.float64))
        t = k * g * v
        y = y + t
        dy = np.abs(k) * (np.abs(g) * dv + dg * np.abs(v)) + 3 * U * np.abs(t) + U * np.abs(y)
    n, dn = norm(y, *pre)
    kind, eps, w, _ = pre
    amp = 1.0 if kind == 0 else (1 / np.sqrt(((y - (y.mean(-1, keepdims=True) if kind == 2 else 0)) ** 2).mean(
        -1, keepdims=True) + eps) * (1 if w is None else np.abs(w)))
    # an error of y moves its own value, the mean and the statistics: three times its size at most, on the whole
    return y, dy, n, dn + amp * (dy + 2 * np.sqrt((dy * dy).mean(-1, keepdims=True)) * (1 + (np.abs(n) if kind else 0)))


def lora(x, w, bias, a, b, scale, idx, act_, res):
    """out and its error bound; x [B][M][K]."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    K = x.shape[-1]
    y = x @ w.T + (0 if bias is None else bias.astype(np.float64))
    err = (K + 2) * U * (np.abs(x) @ np.abs(w).T) + 2 * U * np.abs(y)
    for i, j in enumerate(idx):
        if a is None or not 0 <= j < len(a):
            continue
        aj, bj, s = a[j].astype(np.float64), b[j].astype(np.float64), 1.0 if scale is None else float(scale[j])
        t = s * (x[i] @ aj.T)
        dt = (K + 2) * U * abs(s) * (np.abs(x[i]) @ np.abs(aj).T) + HU * np.abs(t) + TINY
        y[i] += t @ bj.T
        err[i] += dt @ np.abs(bj).T + (aj.shape[0] + 2) * U * (np.abs(t) @ np.abs(bj).T)
    out = act(y, act_)
    err = 1.1 * err + (np.abs(y) * 3 + 6) * U * np.abs(out) * (act_ == 1)
    if res is not None:
        out = out + res.astype(np.float64)
        err = err + U * np.abs(out)
    return out, err


def linattn(q, k, v, g, scale, s0):
    """One sequence: q, k [T][H][dk], v [T][H][dv], g [T][H], s0 [H][dk][dv] -> o, s and the bounds of their 32-bit
    errors, with o's magnitude (the same sums of absolute values) for what roundings of its factors may do."""
    T, H, dk = q.shape
    s = s0.astype(np.float64).copy()
    m, e = np.abs(s), np.zeros_like(s)
    o, eo, mo = (np.zeros((T, H, v.shape[2])) for _ in range(3))
    q, k, v, g = (z.astype(np.float64) for z in (q, k, v, g))
    with np.errstate(invalid="ignore", over="ignore"):
        for t in range(T):
            d = np.exp(g[t])[:, None, None]
            kv = k[t][:, :, None] * v[t][:, None, :]
            s = d * s + kv
            m = d * m + np.abs(kv)
            e = d * e + (6 + 2 * np.abs(np.maximum(g[t], -100))[:, None, None]) * U * m
            o[t] = scale * (q[t][:, :, None] * s).sum(1)
            mo[t] = abs(scale) * (np.abs(q[t])[:, :, None] * m).sum(1)
            eo[t] = abs(scale) * (np.abs(q[t])[:, :, None] * e).sum(1) + (dk + 8) * U * mo[t]
    return o, s, eo, e + 4 * U * m, mo
