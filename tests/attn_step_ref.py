"""64-bit references, in plain numpy loops, of what a decode or speculative step does around the quantized KV cache: norms
with rotation, cache writes and read-back, attention of drafted tokens, verification of drafts."""
import numpy as np

D, PAGE = 128, 16


def norm_rope(x, w, cos_sin, positions, eps, interleaved):
    """float64 [T, H, 128], and the sum of the magnitudes of each value's two terms."""
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    z, size = y.copy(), np.abs(y)
    if cos_sin is not None:
        r = cos_sin.shape[1]
        row = cos_sin[np.clip(positions, 0, len(cos_sin) - 1)].astype(np.float64)
        for i in range(r // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
            c, s = row[:, None, i], row[:, None, r // 2 + i]
            z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
            size[..., a] = np.abs(y[..., a] * c) + np.abs(y[..., b] * s)
            size[..., b] = np.abs(y[..., b] * c) + np.abs(y[..., a] * s)
    return z, size


def unpack(codes, bits):
    """int64 codes [..., 128] of a cache array."""
    c = codes.astype(np.int64)
    if bits == 8:
        return c
    out = np.empty(c.shape[:-1] + (D,), dtype=np.int64)
    out[..., 0::2], out[..., 1::2] = c & 15, (c >> 4) & 15
    return out - 16 * (out > 7)


def pack(codes, bits):
    if bits == 8:
        return codes.astype(np.int8)
    u = codes & 15
    return (u[..., 0::2] | (u[..., 1::2] << 4)).astype(np.uint8)


def page_scale(most, qmax):
    """The smallest float16 that is not below most / qmax; the largest finite one past its range."""
    if most / qmax >= 65504.0:
        return np.float16(65504.0)
    h = np.float16(most / qmax)
    return h if float(h) * qmax >= most else np.nextafter(h, np.float16(np.inf))


def _codes_of(x, scale, qmax):
    with np.errstate(all="ignore"):
        r = np.rint(x / scale)
    return np.clip(np.where(np.isnan(r), 0, r), -qmax, qmax).astype(np.int64)


def append(x, cache, scales, table, lens, bits, rows_of):
    """Writes, per sequence, the rows x[rows_of[b]] (float64 [rows, H, 128]; -1: a token that is not there) at lens[b] on into
    copies of cache and scales."""
    qmax = 127 if bits == 8 else 7
    cache, scales = cache.copy(), scales.copy()
    for b, rows in enumerate(rows_of):
        for lp in range(lens[b] // PAGE, min(table.shape[1], -(-(lens[b] + len(rows)) // PAGE))):
            page = table[b, lp]
            slots = [(lp * PAGE + s, s) for s in range(PAGE) if lens[b] <= lp * PAGE + s < lens[b] + len(rows)]
            new = [(s, x[rows[t - lens[b]]]) for t, s in slots if rows[t - lens[b]] >= 0]
            if not new or not 0 <= page < len(cache):
                continue
            kept = max(lens[b] - lp * PAGE, 0)
            for h in range(cache.shape[1]):
                v = np.abs(np.stack([r[h] for _, r in new]))
                grown = page_scale(v[np.isfinite(v)].max(initial=0.0), qmax)
                s = grown
                if kept:
                    old = scales[page, h]
                    s = max(old, grown)
                    if s > old:
                        c = unpack(cache[page, h, :kept], bits)
                        cache[page, h, :kept] = pack(_codes_of(c * float(old), float(s), qmax), bits)
                scales[page, h] = s
                for slot, r in new:
                    cache[page, h, slot] = pack(_codes_of(r[h], float(s), qmax), bits)
    return cache, scales


def values(cache, scales, table_row, n, bits):
    """float64 [n, H, 128]: the first n tokens of a sequence (page ids clamped into the cache)."""
    pages = np.clip(table_row[:-(-n // PAGE)], 0, len(cache) - 1)
    v = unpack(cache[pages], bits) * scales[pages].astype(np.float64)[..., None, None]
    return v.transpose(0, 2, 1, 3).reshape(-1, cache.shape[1], D)[:n]


def tree_attention(q, k_new, v_new, seen, cache, table, lens, bits, sm):
    """float64 [B, N, Hq, 128] and, per value, the sums that its error is held to: (sum p |v|) / sum p, and the largest error
    of a logit as an fp32 sum over biased codes (both 0 where a node sees nothing).  seen: bool [B, N, N]."""
    kc, vc, ks, vs = cache
    B, N, Hq, _ = q.shape
    Hkv = kc.shape[1]
    out, mean, slip = np.zeros(q.shape), np.zeros(q.shape), np.zeros((B, N, Hq, 1))
    q = q.astype(np.float64)
    for b in range(B):
        n = lens[b]
        keys, vals = values(kc, ks, table[b], n, bits), values(vc, vs, table[b], n, bits)
        pages = np.clip(table[b, :-(-n // PAGE)], 0, len(kc) - 1)
        for h in range(Hq):
            hk = h // (Hq // Hkv)
            step = ks[pages, hk].astype(np.float64).max(initial=0.0)
            for i in range(N):
                at = np.flatnonzero(seen[b, i])
                k = np.concatenate([keys[:, hk], k_new[b, at, hk].astype(np.float64)])
                v = np.concatenate([vals[:, hk], v_new[b, at, hk].astype(np.float64)])
                if not len(k):
                    continue
                s = k @ q[b, i, h] * sm
                p = np.exp(s - s.max())
                p /= p.sum()
                with np.errstate(invalid="ignore"):
                    out[b, i, h], mean[b, i, h] = p @ v, p @ np.abs(v)
                size = max(1280.0 * step, np.abs(k_new[b, at, hk]).astype(np.float64).max(initial=0.0))
                slip[b, i, h] = 32 * 2.0 ** -24 * size * np.abs(q[b, i, h]).sum() * abs(sm)
    return out, mean, slip


def tree_tolerance(out, mean, slip, keys, vmax):
    """|error| allowed: fp16 probabilities (half a step each, 2^-25 where they are subnormal) and logits off by `slip` in the
    numerator and in the sum, fp32 sums, the fp16 result."""
    return mean * (2.0 ** -11 + 2.2 * slip + 64 * 2.0 ** -24) + keys * vmax * 2.0 ** -24 + np.abs(out) * 2.0 ** -11 + 2.0 ** -25


def verify(p, q, tokens, parents, u, num_nodes):
    """(accepted_nodes, counts, out_tokens); p, q float32 [B, N, V] (q None: candidates), parents None: a chain."""
    B, N, V = p.shape
    accepted, out = np.full((B, N), -1), np.full((B, N), -1)
    counts = np.zeros(B, dtype=np.int64)
    weight = lambda row: np.where((row > 0) & np.isfinite(row), row, 0).astype(np.float64)   # noqa: E731
    for b in range(B):
        n = N if num_nodes is None else min(max(int(num_nodes[b]), 0), N)
        if n == 0:
            continue
        path, left, refused = [0], 1.0, []
        for i in range(1, n):
            if (i - 1 if parents is None else parents[b, i]) != path[-1] or (q is not None and refused):
                continue
            t = int(tokens[b, i])
            known = 0 <= t < V
            pt = float(p[b, path[-1], t]) if known and t not in refused and np.isfinite(p[b, path[-1], t]) else 0.0
            bar = float(u[b, i]) * (left if q is None else float(q[b, path[-1], t]) if known else 0.0)
            if pt > 0 and bar < pt:
                path.append(i)
                left, refused = 1.0, []
            else:
                left -= pt if pt > 0 else 0.0
                refused.append(t)
        row = weight(p[b, path[-1]])
        w = row.copy()
        if refused and q is not None:
            qr = q[b, path[-1]]
            w = np.maximum(row - np.where(qr > 0, qr, 0).astype(np.float64), 0)
        for t in refused if q is None else []:
            if 0 <= t < V:
                w[t] = 0
        w = w if w.sum() > 0 else row
        nxt = -1
        if w.sum() > 0:
            run = np.cumsum(w)
            over = np.flatnonzero(run > max(float(u[b, 0]), 0.0) * run[-1])
            nxt = int(over[0]) if len(over) else int(np.flatnonzero(w > 0)[-1])
        counts[b] = len(path)
        accepted[b, :len(path)] = path
        out[b, :len(path)] = [int(tokens[b, i]) for i in path[1:]] + [nxt]
    return accepted, counts, out
