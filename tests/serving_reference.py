"""Plain 64-bit forms of the serving-step operators (rotary positions, append, attention over a paged cache, sampling)."""
import math

import numpy as np


def rope(x, pos, freqs, rotary_dim, layout, amplitude=1.0, sign=1.0):
    """x [tokens, heads, hd]; also returns |a| + |b| of each element's pair (0 where copied), the scale of its error."""
    x = np.asarray(x, np.float64)
    y, size = x.copy(), np.zeros_like(x)
    ang = sign * np.asarray(pos, np.float64)[:, None] * freqs[None, :]
    c, s = (amplitude * np.cos(ang))[:, None, :], (amplitude * np.sin(ang))[:, None, :]
    h = rotary_dim // 2
    ia, ib = (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if layout == "interleaved" else (slice(0, h), slice(h, rotary_dim))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = (np.abs(a) + np.abs(b)) * amplitude
    return y, size


def frequencies(cfg):
    rd = cfg.rotary_dim
    i = np.arange(rd // 2, dtype=np.float64)
    base, s, L = float(cfg.base), float(cfg.factor), float(cfg.original_len)
    f = base ** (-2.0 * i / rd)
    if cfg.scaling == 1:
        f = f / s
    elif cfg.scaling == 2 and rd > 2:
        f = (base * s ** (rd / (rd - 2.0))) ** (-2.0 * i / rd)
    elif cfg.scaling == 3:
        at = lambda t: rd * math.log(L / (t * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(0, math.floor(at(float(cfg.beta_fast)))), min(rd - 1, math.ceil(at(float(cfg.beta_slow))))
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        f = f / s * ramp + f * (1 - ramp)
    elif cfg.scaling == 4:
        lo, hi = float(cfg.low_freq_factor), float(cfg.high_freq_factor)
        share = np.clip((L * f / (2 * math.pi) - lo) / (hi - lo), 0, 1)
        f = (1 - share) * f / s + share * f
    return f


def slots(q_lens, kv_lens, table, page):
    """(row, sequence, position, page, slot) of every new row with a slot."""
    out, row = [], 0
    for s, (n, m) in enumerate(zip(q_lens, kv_lens)):
        for i in range(n):
            p = m - n + i
            if p >= 0:
                out.append((row + i, s, p, int(table[s, p // page]), p % page))
        row += n
    return out


def attention(q, k_pages, v_pages, q_lens, kv_lens, table, scale=None):
    """q [rows, heads, hd], pages [n, page, kv heads, hd] -> (o, lse, weight, noise): weight = sum p |v| of each output element, noise =
    scale * sum |q k|, the largest over the keys a row sees (the scales that rounding errors go with)."""
    rows, nH, hd = q.shape
    page, nKV = k_pages.shape[1:3]
    G = nH // nKV
    scale = 1 / math.sqrt(hd) if scale is None else scale
    o, lse = np.zeros(q.shape), np.full((rows, nH), -np.inf)
    weight, noise = np.zeros(q.shape), np.zeros((rows, nH))
    row = 0
    for s, (n, m) in enumerate(zip(q_lens, kv_lens)):
        if n and m:
            ids = table[s, :-(-m // page)]
            k = k_pages[ids].reshape(-1, nKV, hd)[:m].astype(np.float64)
            v = v_pages[ids].reshape(-1, nKV, hd)[:m].astype(np.float64)
            pos = m - n + np.arange(n)
            see = np.arange(m)[None, :] <= pos[:, None]
            for h in range(nH):
                x = q[row:row + n, h].astype(np.float64)
                sc = np.where(see, x @ k[:, h // G].T * scale, -np.inf)
                top = sc.max(-1, keepdims=True)
                ok = top[:, 0] > -np.inf
                p = np.exp(sc - np.where(ok[:, None], top, 0))
                t = p.sum(-1, keepdims=True)
                p = p / np.where(t > 0, t, 1)
                o[row:row + n, h], weight[row:row + n, h] = p @ v[:, h // G], p @ np.abs(v[:, h // G])
                with np.errstate(divide="ignore"):
                    lse[row:row + n, h] = np.where(ok, np.log(t[:, 0]) + np.where(ok, top[:, 0], 0), -np.inf)
                noise[row:row + n, h] = np.where(see, np.abs(x) @ np.abs(k[:, h // G]).T * scale, 0).max(-1)
        row += n
    return o, lse, weight, noise


def sample(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """One row: (token, kept, probability)."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    if not (x > -np.inf).any():
        return -1, 0, 0.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not T > 0:
        return int(order[0]), 1, 1.0
    mx = x.max()
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == mx, 1.0, np.exp((x[order] - mx) / np.float64(T)))
    if 0 < k < len(x):
        order, w = order[:k], w[:k]
    cum = np.cumsum(w)
    n = len(w)
    if p < 1:
        n = max(1, 1 + int((cum[:-1] < p * cum[-1]).sum())) if p > 0 else 1
    keep = np.arange(len(w)) < n
    keep &= (w > 0) & (w >= (min(m, 1.0) if m > 0 else 0.0))
    ids = np.sort(order[keep])
    wi = dict(zip(order.tolist(), w.tolist()))
    w = np.array([wi[int(i)] for i in ids])
    cum = np.cumsum(w)
    u = min(max(u, 0.0), float(np.float32(0.99999994))) if u > 0 else 0.0
    t = int((cum <= u * cum[-1]).sum())
    return int(ids[t]), len(ids), w[t] / cum[-1]
