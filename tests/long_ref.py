"""Plain restatements, in 64 bits, of the 4-bit cache's values, attention over a window and the next token's draw."""
import numpy as np

F32 = np.float32


def held_ref(x):
    """The values that 4-bit blocks hold of x [..., 32 m] (float32): d = -m / 8 to 8 significant bits and a
    multiple of 2^-24, at most 2720; levels rint(x / d) held to -8..7; NaN where a block is not finite."""
    x = np.asarray(x, F32)
    b = x.reshape(-1, 32)
    out = np.empty(b.shape, F32)
    for i, r in enumerate(b):
        if not np.isfinite(r).all():
            out[i] = np.nan
            continue
        m = float(r[int(np.argmax(np.abs(r)))])  # the first of several
        d = -m / 8
        if d:
            e = max(int(np.floor(np.log2(abs(d)))) - 7, -24)
            d = float(np.rint(d / 2.0 ** e)) * 2.0 ** e
            d = min(max(d, -2720.0), 2720.0)
        n = np.clip(np.rint(r.astype(np.float64) / d), -8, 7) if d else np.zeros(32)
        out[i] = (n * d).astype(F32)
    return out.reshape(x.shape)


def sees_ref(p, n, window, sinks):
    j = np.arange(n)
    see = j <= p
    return see & ((j < sinks) | (j > p - window)) if window else see


def attention_span_ref(q, K, V, pos, window, sinks, scale):
    """q [T][H][HD], K and V [n][KH][HD], row t at pos[t]: outputs in 64 bits, and a bound of what 32-bit
    arithmetic may be off. A score's error is taken as 4 u sqrt(HD) of its sum of |q k| (a random walk of
    rounded additions, four deviations), its parts' as 2^-22 of it and the exponential's argument's as u
    of its size; an output's as the largest |v| times twice the largest of these, and 4 u sqrt(n)."""
    T, H, HD = q.shape
    G = H // K.shape[1]
    q, K, V = q.astype(np.float64), K.astype(np.float64), V.astype(np.float64)
    out, tol = np.empty_like(q), np.empty((T, H, 1))
    u = 2.0 ** -24
    for t in range(T):
        at = np.flatnonzero(sees_ref(pos[t], K.shape[0], window, sinks))
        for h in range(H):
            k, v = K[at, h // G], V[at, h // G]
            s = k @ q[t, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ v
            size = float((np.abs(k) @ np.abs(q[t, h])).max() * abs(scale))
            d = (4 * u * np.sqrt(HD) + 2.0 ** -22) * size + u * float(s.max() - s.min())
            tol[t, h] = np.abs(v).max() * (2 * d + 4 * u * np.sqrt(len(at)) + 4 * u)
    return out, tol


def sample_ref(l, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, how near the draw or a filter comes to a border, relative to the weight) of one row."""
    l = np.asarray(l, F32)
    if temperature == 0 and np.isnan(l[0]):
        return 0, 1.0
    l = np.where(np.isnan(l), F32(-np.inf), l)
    if l.max() == -np.inf:
        return 0, 1.0
    order = np.argsort(-l.astype(np.float64), kind="stable")
    if temperature == 0:
        return int(order[0]), 1.0
    l = l[order].astype(np.float64)
    with np.errstate(invalid="ignore"):
        w = np.where(l == l[0], 1.0, np.exp((l - l[0]) / float(F32(temperature))))
    c = np.cumsum(w)
    n = top_k if 0 < top_k < len(w) else len(w)
    near = 1.0
    if top_p < 1:
        want = float(F32(top_p)) * c[n - 1]
        near = min(near, float(np.abs(c[:n] - want).min() / c[n - 1]))
        n = min(n, 1 + int(np.count_nonzero(c[:n - 1] < want)))
    if min_p > 0:
        near = min(near, float(np.abs(w - float(F32(min_p))).min()) or 1.0)
        n = min(n, int(np.count_nonzero(w >= float(F32(min_p)))))
    x = float(F32(u)) * c[n - 1]
    near = min(near, float(np.abs(c[:n] - x).min() / c[n - 1]))
    return int(order[min(n - 1, int(np.count_nonzero(c[:n] <= x)))]), near
