"""64-bit references, in plain numpy, of the operators around the attention and at the ends of a serving step: step plans,
residual norms, page bounds, the choice of pages, attention over them, sampling."""
import numpy as np

import attn_step_ref as cache_ref

D, PAGE = 128, 16


def plan(table, lens, new, ring, state, rows):
    """(row_start, counts, lens_after, positions, row_lens, row_seq, slots), and copies of table, ring and state after it."""
    table, ring = table.copy(), ring.copy()
    (B, W), P = table.shape, len(ring)
    head, live = int(state[0]) % P, min(max(int(state[1]), 0), P)
    starts, counts, after = np.zeros(B + 1, np.int64), np.zeros(B, np.int64), np.zeros(B, np.int64)
    pos, seq, slots = np.full(rows, -1), np.full(rows, -1), np.full(rows, -1)
    row = asked = taken = 0
    back = []
    for b in range(B):
        n, grow = min(max(int(lens[b]), 0), W * PAGE), max(int(new[b]), 0)
        have = -(-n // PAGE)
        after[b] = n
        if new[b] < 0:
            after[b] = max(0, n + int(new[b]))
            back += table[b, -(-int(after[b]) // PAGE):have].tolist()
        elif n + grow <= W * PAGE and row + grow <= rows:
            need = -(-(n + grow) // PAGE) - have
            asked += need
            if need == 0 or asked <= live:
                for j in range(need):
                    table[b, have + j] = ring[(head + taken + j) % P]
                taken += need
                counts[b], after[b] = grow, n + grow
                for i in range(grow):
                    t = n + i
                    pos[row + i], seq[row + i] = t, b
                    slots[row + i] = int(table[b, t // PAGE]) * PAGE + t % PAGE
        row = min(row + grow, rows + 1)
        starts[b + 1] = min(row, rows)
    for j, page in enumerate(back):
        ring[(head + live + j) % P] = page
    state = np.array([(head + taken) % P, min(live - taken + len(back), P)])
    return (starts, counts, after, pos, pos + 1, seq, slots), table, ring, state


def add_norm(x, r, w, eps, post, gate, sigmoid, scale, offset):
    """float64 y and h, and the sum of the magnitudes of h's two terms."""
    u = x.astype(np.float64)
    if post is not None:
        u = u / np.sqrt((u * u).mean(-1, keepdims=True) + eps) * (post + offset)
    if gate is not None:
        u = u * (1 / (1 + np.exp(-gate)) if sigmoid else gate)
    u = scale * u
    h = u if r is None else r + u
    size = np.abs(u) if r is None else np.abs(r) + np.abs(u)
    y = None if w is None else h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * (w + offset)
    return y, h, size


def bounds(k_cache, old, table, lens, first, bits, max_new=1 << 30):
    out = old.copy()
    for b, n in enumerate(lens):
        n = min(n, table.shape[1] * PAGE)
        f = max(0, 0 if first is None else first[b], n - max_new)
        for lp in range(f // PAGE, -(-n // PAGE)):
            page = table[b, lp]
            if f < n and 0 <= page < len(k_cache):
                c = cache_ref.unpack(k_cache[page, :, :min(PAGE, n - lp * PAGE)], bits)
                out[page] = cache_ref.pack(np.stack([c.max(1), c.min(1)], axis=1), bits).astype(out.dtype)
    return out


def select(q, edge, k_scale, table, seen, bits, top, first, last, row_seq=None):
    """int32 [R, Hkv, top]"""
    R, Hq, _ = q.shape
    P, Hkv = k_scale.shape
    B, W = table.shape
    edge = cache_ref.unpack(edge, bits)
    out = np.full((R, Hkv, top), -1, np.int32)
    for r in range(R):
        b = r if row_seq is None else row_seq[r]
        n = 0 if not 0 <= b < B else min(max(int(seen[r]), 0), W * PAGE)
        pages = -(-n // PAGE)
        if pages <= top:
            out[r, :, :pages] = np.arange(pages)
            continue
        ids = np.clip(table[b, :pages], 0, P - 1)
        for h in range(Hkv):
            worth = np.full(pages, -np.inf, np.float32)
            for g in range(Hq // Hkv):
                x = q[r, h * (Hq // Hkv) + g].astype(np.float64)
                a = np.abs(x[np.isfinite(x)]).max(initial=0.0)
                with np.errstate(all="ignore"):
                    q8 = np.where(np.isnan(x) | (a == 0), 0, np.rint(np.clip(x, -a, a) * 127 / a)).astype(np.int64)
                total = (np.where(q8 > 0, edge[ids, h, 0], edge[ids, h, 1]) * q8).sum(1)
                with np.errstate(invalid="ignore"):
                    one = (total * (a * k_scale[ids, h].astype(np.float64))).astype(np.float32)
                worth = np.maximum(worth, np.where(np.isnan(one), -np.inf, one) + np.float32(0))
                low = np.isnan(one) if g == 0 else low & np.isnan(one)
            rest = np.arange(first, pages - last)
            # NaN below -inf; ties to the lower page
            order = rest[np.lexsort((rest, -worth[rest], low[rest]))][:top - first - last]
            out[r, h] = np.sort(np.concatenate([np.arange(first), order, np.arange(pages - last, pages)]))
    return out


def sparse_attention(q, cache, table, seen, bits, pages, sm, row_seq=None):
    """As tree_attention: float64 [R, Hq, 128], (sum p |v|) / sum p and the largest error of a logit."""
    kc, vc, ks, vs = cache
    R, Hq, _ = q.shape
    P, Hkv = ks.shape
    B, W = table.shape
    out, mean, slip = np.zeros(q.shape), np.zeros(q.shape), np.zeros((R, Hq, 1))
    q = q.astype(np.float64)
    for r in range(R):
        b = r if row_seq is None else row_seq[r]
        n = 0 if not 0 <= b < B else min(max(int(seen[r]), 0), W * PAGE)
        for hk in range(Hkv):
            mine = [p for p in pages[r, hk] if 0 <= p < -(-n // PAGE)]
            if not mine:
                continue
            ids = np.clip(table[b, mine], 0, P - 1)
            live = ((np.array(mine)[:, None] * PAGE + np.arange(PAGE)) < n).reshape(-1)
            k = (cache_ref.unpack(kc[ids, hk], bits) * ks[ids, hk].astype(np.float64)[:, None, None]).reshape(-1, D)[live]
            v = (cache_ref.unpack(vc[ids, hk], bits) * vs[ids, hk].astype(np.float64)[:, None, None]).reshape(-1, D)[live]
            step = ks[ids, hk].astype(np.float64).max()
            for h in range(hk * (Hq // Hkv), (hk + 1) * (Hq // Hkv)):
                s = k @ q[r, h] * sm
                p = np.exp(s - s.max())
                p /= p.sum()
                out[r, h], mean[r, h] = p @ v, p @ np.abs(v)
                slip[r, h] = 32 * 2.0 ** -24 * 1280.0 * step * np.abs(q[r, h]).sum() * abs(sm)
    return out, mean, slip


def sample(logits, u, t, k, p, m):
    """One row: (token, float64 probabilities)."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    V = len(x)
    probs = np.zeros(V)
    M = x.max()
    if M == -np.inf:
        return -1, probs
    order = np.lexsort((np.arange(V), -x))
    if not t > 0:
        t, k = 1.0, 1
    with np.errstate(all="ignore"):
        w = np.where(x == M, 1.0, np.exp((x - M) / t))[order]
    w = np.nan_to_num(w)
    count = V if k <= 0 else min(k, V)
    n = count
    if p < 1:
        run = np.concatenate([[0.0], np.cumsum(w[:count])])
        n = int((run[:-1] < max(p, 0) * run[-1]).sum())
    if m > 0:
        n = min(n, int((w >= min(m, 1.0)).sum()))
    n = max(1, n)
    probs[order[:n]] = w[:n] / w[:n].sum()
    run = np.cumsum(probs)
    at = np.flatnonzero(run > max(u, 0.0) * run[-1])
    return (int(at[0]) if len(at) else int(np.flatnonzero(probs > 0)[-1])), probs
