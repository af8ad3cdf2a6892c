"""Plain 64-bit forms of the drafted-token operators (fun_asr_gguf.ops), row by row, for the tests."""
import numpy as np


def norm_rope(x, w, cos, sin, pos, eps, inter):
    """x [T, heads, D] -> (y, scale of the arithmetic's rounding errors: |a| + |b| of each pair)."""
    x = np.array(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    size = np.abs(x)
    if cos is not None:
        half = cos.shape[1]
        i = np.arange(half)
        f, s = (2 * i, 2 * i + 1) if inter else (i, i + half)
        c, n = (np.asarray(t, np.float64)[pos][:, None] for t in (cos, sin))
        a, b = x[..., f].copy(), x[..., s].copy()
        x[..., f], x[..., s] = a * c - b * n, a * n + b * c
        size[..., f] = size[..., s] = np.abs(a) + np.abs(b)
    return x, size


def attention(q, kc, vc, table, ctx, drafts, mask, scale):
    """q [B, N, H, D], caches [pages, KV, page, D], mask [B, N, N] or None -> (out, sum p |v|, largest sum |q| |k| scale);
    rows behind drafts[b] are nan."""
    B, N, H, D = q.shape
    pages, KV, page = kc.shape[:3]
    out, mass, reach = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros((B, N, H, 1))
    cap = table.shape[1] * page
    for b in range(B):
        n = min(max(int(drafts[b]), 0), N)
        c = min(max(int(ctx[b]), 0), cap)
        total = min(c + n, cap)
        pos = np.arange(total)
        ids = table[b][pos // page]
        here = (ids >= 0) & (ids < pages)
        K = np.zeros((total, KV, D))
        V = np.zeros((total, KV, D))
        K[here] = kc[ids[here], :, pos[here] % page]
        V[here] = vc[ids[here], :, pos[here] % page]
        for i in range(n):
            j = pos - c
            seen = here & ((j < 0) | ((j <= i) if mask is None else mask[b, i][np.clip(j, 0, N - 1)] & (j < n)))
            for h in range(H):
                g = h // (H // KV)
                k, v = K[seen, g], V[seen, g]
                if not len(k):
                    out[b, i, h] = 0
                    continue
                s = (k @ q[b, i, h].astype(np.float64)) * scale
                e = np.exp(s - s.max())
                e /= e.sum()
                out[b, i, h] = (e[:, None] * v).sum(0)
                mass[b, i, h] = (e[:, None] * np.abs(v)).sum(0)
                reach[b, i, h] = (np.abs(k) @ np.abs(q[b, i, h].astype(np.float64))).max() * scale
    return out, mass, reach


def sample(x, u, temperature, top_k, top_p, min_p):
    """One row -> (token, probability, distance of u * total from the nearest border over the total). Settings arrive as
    float32 values."""
    x = np.array(x, np.float64)
    x[np.isnan(x)] = -np.inf
    if not (x > -np.inf).any():
        return -1, 0.0, 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    top = x[order[0]]
    if not temperature > 0:
        return int(order[0]), 1.0, 1.0
    if 0 < top_k < len(x):
        order = order[:top_k]
    rel = np.where(x[order] == top, 0.0, x[order] - top)
    if not top_p >= 1:
        w = np.exp(rel)
        cum = np.cumsum(w)
        n = 1 + int(((cum - w)[1:] < float(top_p) * cum[-1]).sum()) if top_p > 0 else 1
        order, rel = order[:n], rel[:n]
    if not min_p <= 0:
        keep = rel >= np.log(float(min_p)) if min_p <= 1 else np.arange(len(rel)) == 0
        order, rel = order[keep], rel[keep]
    with np.errstate(invalid="ignore"):
        w = np.where(rel == -np.inf, 0.0, np.exp(rel / float(temperature)))
    by_id = np.argsort(order)
    order, w = order[by_id], w[by_id]
    cum = np.cumsum(w)
    t = float(u) * cum[-1]
    at = min(int(np.searchsorted(cum, t, side="right")), int(np.nonzero(w > 0)[0][-1]))
    while w[at] == 0:  # (u = 0: the first with any mass)
        at += 1
    return int(order[at]), w[at] / cum[-1], np.abs(cum - t).min() / cum[-1]
