"""The sequence-cache operators in numpy float64, written from their definitions (the oracle of their tests).

rope: pairs turned by positions of several axes.  write / read: the paged 8-bit cache.  attention: softmax over the
cached tokens.  The cache is a dict of arrays: k_codes, v_codes int8 [pages][heads][P][D], k_scale, v_scale float32
[pages][heads].  A batch is (table, row_start, kv_len) as int arrays.
"""
import numpy as np


def rope_plan(sections, deal, restart, base):
    """(axis, frequency) of every pair."""
    pairs, plan = sum(sections), []
    used, axis = [0] * len(sections), 0
    for i in range(pairs):
        while used[axis] == sections[axis]:
            axis = (axis + 1) % len(sections)
        power = used[axis] / sections[axis] if restart else i / pairs
        plan.append((axis, float(base) ** -power))
        used[axis] += 1
        if deal:
            axis = (axis + 1) % len(sections)
    return plan


def rope(x, pos, sections, neighbours=False, deal=False, restart=False, base=10000.0, pos_scale=1.0, inverse=False):
    """x [rows][heads][D], pos [axes][rows] -> float64 of x's shape."""
    x = np.asarray(x, np.float64)
    y = x.copy()
    n = sum(sections)
    for i, (axis, w) in enumerate(rope_plan(sections, deal, restart, base)):
        angle = np.asarray(pos, np.float64)[axis] * pos_scale * w * (-1.0 if inverse else 1.0)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        d0, d1 = (2 * i, 2 * i + 1) if neighbours else (i, i + n)
        y[..., d0] = x[..., d0] * c - x[..., d1] * s
        y[..., d1] = x[..., d1] * c + x[..., d0] * s
    return y


def empty_cache(pages, heads, P, D, seed=0):
    """A cache whose memory holds anything: random codes, scales of all sorts."""
    r = np.random.default_rng(seed)
    c = {}
    for n in "kv":
        c[n + "_codes"] = r.integers(-128, 128, (pages, heads, P, D)).astype(np.int8)
        c[n + "_scale"] = r.choice(np.array([np.nan, np.inf, 0.0, 1.0, 1e30], np.float32), (pages, heads))
    return c


def _write_one(codes, scale, x, table, row_start, kv_len):
    P = codes.shape[2]
    x = np.asarray(x, np.float64)
    for s, length in enumerate(kv_len):
        rows = x[row_start[s]:row_start[s + 1]]
        begin = length - len(rows)
        if not len(rows):
            continue
        for i in range(begin // P, (length - 1) // P + 1):
            page, lo, hi = table[s][i], max(begin - i * P, 0), min(length - i * P, P)
            new = rows[i * P + lo - begin:i * P + hi - begin]  # [t][heads][D]
            for h in range(codes.shape[1]):
                v = new[:, h]
                finite = np.abs(v[np.isfinite(v)])
                amax = finite.max() if finite.size else 0.0
                held = scale[page, h] if lo > 0 else np.float32(0)
                to = max(held, np.float32(amax) * (np.float32(1) / np.float32(127)) if amax >= 2.0 ** -100 else np.float32(0))
                with np.errstate(invalid="ignore", over="ignore"):
                    q = np.rint(v / np.float64(to)) if to > 0 else np.zeros_like(v)
                q = np.clip(np.where(np.isnan(v), 0.0, q), -127, 127)
                if lo > 0 and to > held:
                    old = codes[page, h, :lo].astype(np.float64)
                    codes[page, h, :lo] = np.rint(old * np.float64(held) / np.float64(to)).astype(np.int8)
                codes[page, h, lo:hi] = q.astype(np.int8)
                scale[page, h] = to


def write(cache, k, v, table, row_start, kv_len):
    for n, x in (("k", k), ("v", v)):
        _write_one(cache[n + "_codes"], cache[n + "_scale"], x, table, row_start, kv_len)


def tokens(cache, n, table_row, begin, end):
    """float64 values of positions begin .. end - 1: [t][heads][D]."""
    codes, scale = cache[n + "_codes"], cache[n + "_scale"]
    P = codes.shape[2]
    at = np.arange(begin, end)
    page = np.asarray(table_row)[at // P]
    return codes[page, :, at % P].astype(np.float64) * scale[page].astype(np.float64)[..., None]


def read(cache, table, row_start, kv_len):
    """(k, v) rows [rows][heads][D] float64: the last rows of each sequence."""
    out = []
    for n in "kv":
        parts = [tokens(cache, n, table[s], length - (row_start[s + 1] - row_start[s]), length)
                 for s, length in enumerate(kv_len)]
        out.append(np.concatenate(parts))
    return out


def attention(cache, q, table, row_start, kv_len, scale, causal=True, window=0):
    """q [rows][n_heads][D] -> float64 of its shape; rows that belong to no sequence are NaN."""
    q = np.asarray(q, np.float64)
    y = np.full_like(q, np.nan)
    for s, length in enumerate(kv_len):
        r0, r1 = row_start[s], row_start[s + 1]
        k, v = tokens(cache, "k", table[s], 0, length), tokens(cache, "v", table[s], 0, length)
        group = q.shape[1] // cache["k_codes"].shape[1]
        place = np.arange(length - (r1 - r0), length)[:, None] if causal else np.full((r1 - r0, 1), length - 1)
        key = np.arange(length)
        seen = key <= place
        if window:
            seen &= key > place - window
        for h in range(q.shape[1]):
            z = np.where(seen, q[r0:r1, h] @ k[:, h // group].T * scale, -np.inf)
            top = z.max(1, keepdims=True, initial=-np.inf)
            p = np.exp(z - np.where(np.isfinite(top), top, 0.0))
            total = p.sum(1, keepdims=True)
            y[r0:r1, h] = (p @ v[:, h // group]) / np.where(total > 0, total, 1.0)
    return y
