"""Plain 64-bit forms of the 4-bit key/value cache's operators, in numpy on the host: head
norms with rotation, quantization, paged attention with weights, eviction.

A cache is a dict of arrays k, ks, v, vs, score in the library's layout plus fmt, page; a
sequence's tokens are looked up one by one through its table."""
import numpy as np

GROUP = {4: 64, 7: 32}
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6.0])
LUT7 = np.concatenate((GRID, -GRID))
HELD, TINY = 6.0 * 2.0 ** 125, 2.0 ** -100


def norm_rope(x, w, eps, pos, freq, rot, interleaved):
    """x [T, H, D] -> (y, size): size bounds the magnitudes that met in each element."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if w is not None:
        y = y * w.astype(np.float64)
    size = np.abs(y)
    if freq is not None:
        ang = pos.astype(np.float64)[:, None, None] * freq
        c, s = np.cos(ang), np.sin(ang)
        j = np.arange(rot // 2)
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + rot // 2)
        ya, yb = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
        size[..., a] = size[..., b] = np.abs(ya) + np.abs(yb)
    return y, size


def quantize(fmt, x):
    """x [..., D] -> codes [..., D / 2] uint8, scales (f32, or ue8m0 bytes)."""
    x = np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=HELD, neginf=-HELD).clip(-HELD, HELD)
    g = x.reshape(*x.shape[:-1], -1, GROUP[fmt])
    top = np.abs(g).max(-1)
    if fmt == 4:
        s = np.where(top < TINY, 0.0, (top.astype(np.float32) * np.float32(1 / 7)).astype(np.float64))
        n = np.where(s[..., None] > 0, np.rint(g / np.where(s > 0, s, 1)[..., None]), 0).clip(-7, 7)
        n, s = n.astype(np.int64) + 8, s.astype(np.float32)
    else:
        e = np.maximum(np.ceil(np.log2(np.maximum(top, 2.0 ** -200) / 6)), -126)
        e = np.where(top > 6 * 2.0 ** e, e + 1, e)
        e = np.where((top <= 6 * 2.0 ** (e - 1)) & (e > -126), e - 1, e)
        q = g / 2.0 ** e[..., None]
        n = np.searchsorted((GRID[1:] + GRID[:-1]) / 2, np.abs(q).clip(0, 6), side="left")
        n = np.where((q < 0) & (n > 0), n + 8, n)
        s = (e + 127).astype(np.uint8)
    n = n.reshape(x.shape).astype(np.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), s


def values(fmt, codes, scales):
    n = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    v = n.astype(np.float64) - 8 if fmt == 4 else LUT7[n]
    with np.errstate(over="ignore"):
        s = scales.astype(np.float64) if fmt == 4 else \
            np.where(scales == 255, np.inf, np.where(scales == 0, 0, 2.0 ** (scales.astype(int) - 127.0)))
    with np.errstate(invalid="ignore"):
        return v * np.repeat(s, GROUP[fmt], -1)


def place(c, table_row, t):
    """(page, slot) of token t, or None where it is not there."""
    pg = t // c["page"]
    if t < 0 or pg >= len(table_row):
        return None
    p = int(table_row[pg])
    return (p, t % c["page"]) if 0 <= p < len(c["k"]) else None


def rows_of(q_start, lens):
    """(row, sequence, token in it) of each row that belongs to a sequence."""
    for b in range(len(lens)):
        for r in range(q_start[b], q_start[b + 1]):
            yield r, b, int(lens[b]) - int(q_start[b + 1]) + r


def attention(c, q, q_start, lens, table, scale, window, weights):
    """-> out [T, Hq, D], mag (sum of P |v|), sizes, score (or None); rows of no sequence are
    NaN in out.  sizes, in log2 units of the exponents: the largest |exponent|, the largest sum of
    |q k| and the largest root of the sum of (q k)^2."""
    T, Hq, D = q.shape
    Hkv = c["k"].shape[1]
    G = Hq // Hkv
    out, mag = np.full((T, Hq, D), np.nan), np.zeros((T, Hq, D))
    top, err, err2 = 0.0, 0.0, 0.0
    score = c["score"].astype(np.float64) if weights else None
    for b in range(len(lens)):
        n = min(max(int(lens[b]), 0), table.shape[1] * c["page"])
        at = [place(c, table[b], t) for t in range(n)]
        here = np.array([p is not None for p in at], bool)
        pg, sl = (np.array([p[i] if p else 0 for p in at], int) for i in (0, 1))
        r0, r1 = int(q_start[b]), int(q_start[b + 1])
        pos = int(lens[b]) - r1 + np.arange(r0, r1)
        for h in range(Hkv):
            k = values(c["fmt"], c["k"][pg, h, sl], c["ks"][pg, h, sl])
            v = values(c["fmt"], c["v"][pg, h, sl], c["vs"][pg, h, sl])
            got = np.zeros(n)
            for i, r in enumerate(range(r0, r1)):
                sees = here & (np.arange(n) <= pos[i])
                if window:
                    sees &= np.arange(n) > pos[i] - window
                out[r, h * G:(h + 1) * G] = 0
                if not sees.any():
                    continue
                for j in range(h * G, (h + 1) * G):
                    qr = q[r, j].astype(np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = (k[sees] @ qr) * scale
                        e = np.exp(s - s.max())
                    p = e / e.sum()
                    out[r, j], mag[r, j] = p @ v[sees], p @ np.abs(v[sees])
                    got[sees] += p
                    if np.isfinite(s).all():
                        top = max(top, np.abs(s).max() * 1.4427)
                        err = max(err, (np.abs(k[sees]) @ np.abs(qr)).max() * abs(scale) * 1.4427)
                        err2 = max(err2, np.sqrt((k[sees] ** 2 @ qr ** 2).max()) * abs(scale) * 1.4427)
            if weights:
                old = score[pg[here], h, sl[here]]
                score[pg[here], h, sl[here]] = got[here] + (old if weights == 1 else 0)
    return out, mag, (top, err, err2), score


def evict(c, lens, table, keep, recent):
    """-> kept [B, Hkv, keep] int32, new_lens."""
    Hkv = c["k"].shape[1]
    kept = np.full((len(lens), Hkv, keep), -1, np.int32)
    for b, n in enumerate(lens):
        n = min(max(int(n), 0), table.shape[1] * c["page"])
        for h in range(Hkv):
            w = np.full(n, -np.inf)
            rank = np.zeros(n)  # what is not there, and NaN, comes after -inf
            for t in range(n):
                p = place(c, table[b], t)
                if p is not None and not np.isnan(c["score"][p[0], h, p[1]]):
                    w[t], rank[t] = c["score"][p[0], h, p[1]], 1
            old = max(0, n - recent) if n > keep else 0
            best = sorted(range(old), key=lambda t: (-rank[t], -w[t], t))[:max(0, keep - (n - old))]
            ids = sorted(best) + list(range(old, n))
            kept[b, h, :len(ids)] = ids
    return kept, np.minimum(np.maximum(lens, 0), keep).astype(np.int32)
