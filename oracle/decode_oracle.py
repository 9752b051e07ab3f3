"""The operators of a decoding step in numpy float64, written from their definitions (the oracle of their tests).

norm: heads normalised, weighted, and turned by their positions.  kv4_*: the paged 4-bit cache and the attention over it;
the cache is a dict of arrays: k_codes, v_codes uint8 [pages][heads][P][D / 2], k_scale, v_scale uint16 (the bits of a
bf16) [pages][heads][P][D / 32]; a batch is (table, row_start, kv_len) as int arrays.  blocks / weight: ggml's Q4_0 and
Q4_1 blocks as bytes, and the numbers they stand for.
"""
import numpy as np

import seq_cache_oracle as sc

SMALL = 2.0 ** -100


def bf16_bits(x):
    """float array -> bits of the nearest bf16 (ties to even); finite values below bf16's largest."""
    u = np.asarray(x, np.float32).view(np.uint32)
    return ((u + np.uint32(0x7FFF) + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


# ---- norm and rotation -----------------------------------------------------------------------------------------


def normalised(x, weight, bias, eps, layer):
    x = np.asarray(x, np.float64)
    if layer:
        x = x - x.mean(-1, keepdims=True)
    u = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    return u * (1.0 if weight is None else np.asarray(weight, np.float64)) + (0.0 if bias is None else np.asarray(bias, np.float64))


def norm(x, weight, bias, eps, layer, pos, sections, **kw):
    return sc.rope(normalised(x, weight, bias, eps, layer), pos, sections, **kw)


# ---- the 4-bit cache -------------------------------------------------------------------------------------------


def kv4_empty(pages, heads, P, D, seed=0):
    """A cache whose memory holds anything: random codes, scales that are not numbers among them."""
    r = np.random.default_rng(seed)
    c = {}
    for n in "kv":
        c[n + "_codes"] = r.integers(0, 256, (pages, heads, P, D // 2)).astype(np.uint8)
        c[n + "_scale"] = r.choice(np.array([0x7FC0, 0xFF80, 0x7F80, 0x0000, 0x3F80, 0xFF7F, 0x7F00, 0x0001], np.uint16), (pages, heads, P, D // 32))
    return c


def kv4_quantise(x):
    """[..., D] -> (codes + 8 as whole numbers [..., D], scale bits [..., D / 32])."""
    x = np.asarray(x, np.float64)
    y = x.reshape(*x.shape[:-1], -1, 32)
    finite = np.where(np.isfinite(y), y, 0.0)
    high, low = finite.max(-1), finite.min(-1)
    top = np.where(high >= -low, high, low)
    most = (2 - 2.0 ** -7) * 2.0 ** 124
    bits = bf16_bits(np.where(np.abs(top) < SMALL, 0.0, np.clip(top / -8, -most, most)).astype(np.float32))
    bits = np.where(np.abs(top) < SMALL, np.uint16(0), bits)
    d = bf16_value(bits)[..., None]
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        q = np.rint(y / d)
    q = np.where(np.isnan(y) | (d == 0), 0.0, np.clip(q, -8, 7))
    return (q + 8).astype(np.int64).reshape(x.shape), bits


def kv4_write(cache, k, v, table, row_start, kv_len):
    P = cache["k_codes"].shape[2]
    for n, x in (("k", k), ("v", v)):
        codes, bits = kv4_quantise(x)
        packed = (codes[..., 0::2] | codes[..., 1::2] << 4).astype(np.uint8)
        for s, length in enumerate(kv_len):
            for r in range(row_start[s], row_start[s + 1]):
                t = length - row_start[s + 1] + r
                cache[n + "_codes"][table[s][t // P], :, t % P] = packed[r]
                cache[n + "_scale"][table[s][t // P], :, t % P] = bits[r]


def kv4_tokens(cache, n, table_row, begin, end):
    """float64 values of positions begin .. end - 1: [t][heads][D]."""
    P, at = cache["k_codes"].shape[2], np.arange(begin, end)
    page = np.asarray(table_row)[at // P]
    codes, d = cache[n + "_codes"][page, :, at % P], bf16_value(cache[n + "_scale"][page, :, at % P])
    x = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1]).astype(np.float64) - 8
    return x * d.repeat(32, -1)


def kv4_read(cache, table, row_start, kv_len):
    return [np.concatenate([kv4_tokens(cache, n, table[s], length - (row_start[s + 1] - row_start[s]), length)
                            for s, length in enumerate(kv_len)]) for n in "kv"]


def kv4_attention(cache, q, table, row_start, kv_len, scale, causal=True, window=0):
    """q [rows][n_heads][D] -> float64 of its shape; rows that belong to no sequence are NaN.  Tokens that no row of a
    sequence sees are not looked at."""
    q = np.asarray(q, np.float64)
    y = np.full_like(q, np.nan)
    for s, length in enumerate(kv_len):
        r0, r1 = row_start[s], row_start[s + 1]
        first = max(length - (r1 - r0) - window + 1, 0) if window else 0
        k, v = (kv4_tokens(cache, n, table[s], first, length) for n in "kv")
        group = q.shape[1] // cache["k_codes"].shape[1]
        place = np.arange(length - (r1 - r0), length)[:, None] if causal else np.full((r1 - r0, 1), length - 1)
        key = np.arange(first, length)
        seen = key <= place
        if window:
            seen &= key > place - window
        for h in range(q.shape[1]):
            with np.errstate(invalid="ignore", over="ignore"):
                z = np.where(seen, q[r0:r1, h] @ k[:, h // group].T * scale, -np.inf)
                top = z.max(1, keepdims=True, initial=-np.inf)
                p = np.exp(z - np.where(np.isfinite(top), top, 0.0))
                total = p.sum(1, keepdims=True)
                y[r0:r1, h] = (p @ v[:, h // group]) / np.where(total > 0, total, np.where(np.isnan(total), np.nan, 1.0))
    return y


# ---- 4-bit weights ---------------------------------------------------------------------------------------------


def blocks(rng, kind, N, K, size=0.05):
    """Random blocks of N rows of K weights, as bytes [N * K / 32][18 or 20]."""
    n = N * (K // 32)
    d = (rng.normal(size=(n, 1)) * size).astype(np.float16)
    codes = rng.integers(0, 256, (n, 16)).astype(np.uint8)
    head = [d] if kind == "q4_0" else [d, (rng.normal(size=(n, 1)) * size * 4).astype(np.float16)]
    return np.concatenate([h.view(np.uint8) for h in head] + [codes], 1)


def parts(raw, kind, N, K):
    """(d, code - 8, minimum + 8 d) of each weight, float64 [N][K]."""
    h = 2 if kind == "q4_0" else 4
    d = raw[:, :2].copy().view(np.float16).astype(np.float64)
    code = np.concatenate([raw[:, h:] & 15, raw[:, h:] >> 4], 1).astype(np.float64) - 8
    low = np.zeros_like(d) if kind == "q4_0" else raw[:, 2:4].copy().view(np.float16).astype(np.float64) + 8 * d
    wide = lambda x: np.broadcast_to(x, code.shape).reshape(N, K)
    return wide(d), code.reshape(N, K), wide(low)


def weight(raw, kind, N, K):
    d, code, low = parts(raw, kind, N, K)
    return d * code + low
