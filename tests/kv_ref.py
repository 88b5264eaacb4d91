"""Plain 64-bit forms of the drafted-token and bounded-cache operators, on the
CPU, one (sequence, kv head) at a time."""
import numpy as np


def f64(t):
    return t.detach().cpu().double().numpy()


def as_cached(rows, cache):
    """rows as a cache of this tensor's type holds them (one rounding)."""
    return rows.to(cache.dtype)


def attend(q, k, v, seen):
    """q [r, hd], k / v [t, hd], seen bool [r, t]: outputs, sum p |v| and weights.
    Rows that see nothing give zeros."""
    with np.errstate(all="ignore"):
        z = q @ k.T / np.sqrt(q.shape[1])
        out, mag, w = np.zeros_like(q), np.zeros_like(q), np.zeros(seen.shape)
        for r in range(q.shape[0]):
            at = np.flatnonzero(seen[r])
            if at.size == 0:
                continue
            e = np.exp(z[r, at] - z[r, at].max())
            p = e / e.sum()
            w[r, at] = p
            out[r], mag[r] = p @ v[at], p @ np.abs(v[at])
    return out, mag, w


def mask_bits(mask):
    """int64 [n, T, words] as bool [n, T, T]."""
    m = np.ascontiguousarray(mask.cpu().numpy())
    n, T, words = m.shape
    return np.unpackbits(m.view(np.uint8).reshape(n, T, words * 8), axis=-1,
                         bitorder="little")[:, :, :T].astype(bool)


def tree(q, k, v, lens, kd, vd, mask, nh, nk, n_nodes=None):
    """[n, T, nh * hd] outputs and sum p |v| (0 past a sequence's nodes)."""
    n, T, _ = q.shape
    ctx, hd, g = k.shape[1], k.shape[2] // nk, nh // nk
    kd, vd = f64(as_cached(kd, k)), f64(as_cached(vd, v))
    q, bits = f64(q).reshape(n, T, nh, hd), mask_bits(mask)
    out, mag = np.zeros_like(q), np.zeros_like(q)
    for s in range(n):
        t = min(max(int(lens[s]), 0), ctx)
        m = T if n_nodes is None else min(max(int(n_nodes[s]), 0), T)
        ks, vs = f64(k[s, :t]), f64(v[s, :t])
        seen = np.concatenate((np.ones((m, t), bool), bits[s, :m, :m]), 1)
        for h in range(nh):
            c = slice(h // g * hd, (h // g + 1) * hd)
            out[s, :m, h], mag[s, :m, h], _ = attend(
                q[s, :m, h], np.concatenate((ks[:, c], kd[s, :m, c])),
                np.concatenate((vs[:, c], vd[s, :m, c])), seen)
    return out.reshape(n, T, -1), mag.reshape(n, T, -1)


def scored(q, k, v, lens, nh, nk):
    """Outputs, sum p |v| and the weights of one step [n, nk, ctx]."""
    n, ctx, hd, g = q.shape[0], k.shape[1], k.shape[2] // nk, nh // nk
    q = f64(q).reshape(n, nh, hd)
    out, mag, w = np.zeros_like(q), np.zeros_like(q), np.zeros((n, nk, ctx))
    for s in range(n):
        t = min(max(int(lens[s]), 0), ctx)
        ks, vs = f64(k[s, :t]), f64(v[s, :t])
        for j in range(nk):
            c, hs = slice(j * hd, (j + 1) * hd), slice(j * g, (j + 1) * g)
            o, m, p = attend(q[s, hs], ks[:, c], vs[:, c], np.ones((g, t), bool))
            out[s, hs], mag[s, hs], w[s, j, :t] = o, m, p.sum(0)
    return out.reshape(n, -1), mag.reshape(n, -1), w


def keep(weights, length, budget, first, recent):
    """The positions one (sequence, kv head) keeps, ascending."""
    if length <= budget:
        return np.arange(length)
    mid = np.asarray(weights[first:length - recent], dtype=np.float64)
    key = np.where(np.isnan(mid), np.inf, mid)
    # NaN above +inf, then the value, then the lowest position
    order = np.lexsort((np.arange(mid.size), -key, ~np.isnan(mid)))
    best = np.sort(order[:budget - first - recent]) + first
    return np.concatenate((np.arange(first), best, np.arange(length - recent, length))).astype(int)
