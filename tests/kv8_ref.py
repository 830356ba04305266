"""The 8-bit key/value cache in 64 bits, written from its definition: what it holds, the attention over it, eviction."""
import numpy as np

BLOCK = 32


def stored(x):
    """What a cache stands for of one sequence's rows x [len, kv, hd] (fp32), as fp32."""
    x = np.asarray(x, dtype=np.float32)
    y = x.copy()
    for b in range(len(x) // BLOCK):
        for h in range(x.shape[1]):
            blk = x[b * BLOCK:(b + 1) * BLOCK, h]
            if not np.all(np.isfinite(blk)):
                y[b * BLOCK:(b + 1) * BLOCK, h] = np.nan
                continue
            s = np.float32(np.max(np.abs(blk)) / np.float32(127.0))
            q = np.rint(blk.astype(np.float64) / np.float64(s)) if s > 0 else np.zeros(blk.shape)
            y[b * BLOCK:(b + 1) * BLOCK, h] = (np.clip(q, -127, 127) * np.float64(s)).astype(np.float32)
    return y


def visible(pos, n, window, prefix):
    """[n, pos + n]: which positions the queries at pos .. pos + n - 1 see."""
    i = (pos + np.arange(n))[:, None]
    j = np.arange(pos + n)[None, :]
    see = j <= i
    if window:
        see = see & (i - j < window)
    return see | (j < prefix)


def attend(q, k, v, pos, scale, cap=0.0, window=0, prefix=0):
    """q [n, H, hd] over the stored k, v [pos + n, kv, hd]: outputs [n, H, hd], the weights summed over queries
    and a group's heads [kv, pos + n], and a bound of what fp32 may lose in the outputs. The bound: a score is a sum of hd
    products in fp32 (each operand exact to 2^-22 as a pair of halves) and a few roundings of its own, so it is off by at most
    ds = (hd + 16) 2^-24 sum |q k| scale + 2^-21 (its size in log2 units, the exponent's argument; the cap's function: 4
    2^-24 cap); its weight is off by the factor 1 + ds, numerator and sum alike, and the sum of len weighted values by
    (len + 16) 2^-24 of the largest value."""
    n, H, hd = q.shape
    kv = k.shape[1]
    G = H // kv
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    see = visible(pos, n, window, prefix)
    out = np.zeros((n, H, hd))
    w = np.zeros((kv, pos + n))
    tol = np.zeros((n, H, 1))
    e = 2.0 ** -24
    for h in range(H):
        kk, vv = k[:, h // G], v[:, h // G]
        with np.errstate(all="ignore"):
            s = (q[:, h] @ kk.T) * scale
            size = (np.abs(q[:, h]) @ np.abs(kk.T)) * abs(scale)
            if cap:
                s = cap * np.tanh(s / cap)
            s = np.where(see, s, -np.inf)
            p = np.exp(s - s.max(axis=1, keepdims=True))
            p = np.where(see, p, 0.0)
            p = p / p.sum(axis=1, keepdims=True)
            out[:, h] = np.where(see[:, :, None], p[:, :, None] * vv[None], 0.0).sum(axis=1)
            w[h // G] += p.sum(axis=0)
            ds = (np.where(see, size, 0.0).max(axis=1) * (hd + 16) + 8.0) * e + 4 * e * cap
            top = np.where(see[:, :, None], np.abs(vv)[None], 0.0).max(axis=(1, 2))
            tol[:, h, 0] = (2 * ds + (pos + n + 16) * e) * top
    return out, w, tol


def keep_rule(w, keep, recent):
    """Positions that stay, of one head's weights w [len]."""
    old = len(w) - recent
    bad = np.isnan(w[:old])
    order = np.lexsort((np.arange(old), np.where(bad, 0.0, -w[:old].astype(np.float64)), bad))
    return np.concatenate([np.sort(order[:keep - recent]), np.arange(old, len(w))]).astype(np.uint32)
