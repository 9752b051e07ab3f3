"""The operators of a decoding step (sam3b200_rope_norm_run, sam3b200_kv4_*, sam3b200_mul_mat_vec) against the float64 oracle.

Tolerances, all derived from the number of roundings.
norm: a head's sum of squares is a sum of positive terms in at most 20 roundings of 2^-24 (16 in a thread, 4 across), so the
reciprocal root is off by 10 of them, and root, quotient, product and weight add 4: 2^-20 of u - bias.  A layer norm's mean is
off by at most 21 roundings of the mean magnitude, which 1 / sigma carries over.  The rotation adds 2^-21 of a pair's length
(see test_seq_cache_gpu.py), the output half a step of its type.
kv4: codes and scales are equal.  attention: each weight times a scale is rounded to f16 (2^-11), scores and sums are f32, so
2^-10 of the largest cached magnitude of the sequence's head covers the weights twice over, plus half a step.
mul_mat_vec: a block's sum in f32 takes 33 terms in any order, each rounded or truncated once (2^-23 of the sum of
magnitudes); blocks add K / 32 + 12 roundings of 2^-24; x loses 2^-23 of an element (F32), 2^-26 of a row's largest (F32,
BF16); half a step on top."""
import importlib.util
import os
import sys

import numpy as np
import pytest

import decode_oracle as do
import seq_cache_oracle as sc
from test_seq_cache_gpu import GROUPS, HALF_STEP, TYPES, dtype, pages_for, store, value

pytestmark = pytest.mark.gpu


def at_least_half_step(want, t):
    return np.abs(want) * HALF_STEP[t] * 1.01 + 2.0 ** -25 * (t == "f16")


# ---- norm and rotation -----------------------------------------------------------------------------------------


def norm_tolerance(x, w, b, eps, layer, want, t_out, sections, neighbours):
    w = np.ones(x.shape[-1]) if w is None else w
    b = np.zeros(x.shape[-1]) if b is None else b
    center = x - x.mean(-1, keepdims=True) if layer else x
    sigma = np.sqrt((center ** 2).mean(-1, keepdims=True) + eps)
    u = center / sigma * w
    tol = 2.0 ** -20 * np.abs(u) + 2.0 ** -23 * np.abs(b)
    if layer:
        tol = tol + np.abs(w) * (22 * 2.0 ** -24 * np.abs(x).mean(-1, keepdims=True) + 2.0 ** -23 * np.abs(x)) / sigma
    u = np.abs(u) + np.abs(b)
    n = sum(sections)
    for i in range(n):
        d0, d1 = (2 * i, 2 * i + 1) if neighbours else (i, i + n)
        both = np.hypot(tol[..., d0], tol[..., d1]) + 2.0 ** -21 * np.hypot(u[..., d0], u[..., d1])
        tol[..., d0] = tol[..., d1] = both
    return tol + at_least_half_step(want, t_out)


NORM_SHAPES = [(64, [16, 16], dict(neighbours=True, restart=True)), (128, [24, 20, 20], dict(deal=True, base=5e6)), (128, [0, 32], dict()),
               (80, [40], dict()), (96, [24], dict(neighbours=True)), (72, [20, 16], dict()), (256, [128], dict(pos_scale=0.25)), (16, [8], dict()),
               (20, [3, 4], dict(deal=True)), (2, [1], dict()), (250, [100, 25], dict(neighbours=True))]


def run_norm(b200, be, xs, ws, bs, t_in, t_out, t_w, pos, sections, eps, layer, nb=None, offset=0, in_place=False, pos_stride=None, **kw):
    """xs: raw arrays [rows][heads][D] (or wider, with nb = element strides and the head where each set starts)."""
    keep, sets, out = [], [], []
    raw = lambda a, t, o: be.upload(np.concatenate([np.zeros(o, dtype(t)), np.asarray(a).reshape(-1)]))
    for x, w, b in zip(xs, ws, bs):
        rows, heads, D = x.shape
        xb = raw(x, t_in, offset)
        yb = xb if in_place else be.upload(np.full(x.size + offset + 3, 77, dtype(t_out)))
        wb, bb = (None if a is None else raw(a, t_w, offset) for a in (w, b))
        keep += [xb, yb, wb, bb]
        at = lambda buf, t: None if buf is None else buf.ptr + offset * np.dtype(dtype(t)).itemsize
        sets.append(b200.NormHeads(at(xb, t_in), heads, at(wb, t_w), at(yb, t_out), bias=at(bb, t_w)))
        out.append((yb, x.shape))
    pb = be.upload(np.ascontiguousarray(pos, np.int32))
    r = be.rope(xs[0].shape[2], sections, **kw)
    r.norm(sets, TYPES[t_in], pb.ptr, xs[0].shape[0], TYPES[t_out], w_type=TYPES[t_w], eps=eps, layer=layer, pos_stride=pos_stride)
    be.synchronize()
    r.free()
    got = []
    for yb, shape in out:
        n = int(np.prod(shape))
        y = yb.get(n + offset + (0 if in_place else 3), dtype(t_out))
        assert in_place or np.all(y[n + offset:] == 77)
        got.append(y[offset:n + offset].reshape(shape))
    return got


@pytest.mark.parametrize("t_in,t_out,t_w", [("f32", "f32", "f32"), ("f16", "f16", "f16"), ("bf16", "bf16", "bf16"), ("f32", "f16", "f32"), ("bf16", "f32", "f16")])
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("D,sections,kw", NORM_SHAPES)
def test_norm(b200, backend, t_in, t_out, t_w, layer, D, sections, kw):
    """Queries, keys and a third set with weights of their own, some without, offsets that leave rows unaligned."""
    rng = np.random.default_rng(D + len(sections) + layer)
    for rows, heads, offset in ((1, (1, 1), 0), (7, (12, 3), 0), (130, (3, 1, 9), 0), (19, (5, 2), 1)):
        xs = [store(rng.normal(size=(rows, h, D)) * 3 + rng.normal(size=(1, h, 1)), t_in) for h in heads]
        ws = [store(1 + 0.3 * rng.normal(size=D), t_w) if i != 1 else None for i in range(len(heads))]
        bs = [store(0.2 * rng.normal(size=D), t_w) if (i == 0) == layer else None for i in range(len(heads))]
        pos = rng.integers(-50, 1 << rng.integers(3, 20), (len(sections), rows))
        eps = 1e-5
        got = run_norm(b200, backend, xs, ws, bs, t_in, t_out, t_w, pos, sections, eps, layer, offset=offset, **kw)
        for x, w, b, y in zip(xs, ws, bs, got):
            x, w, b = value(x, t_in), None if w is None else value(w, t_w), None if b is None else value(b, t_w)
            want = do.norm(x, w, b, eps, layer, pos, sections, **kw)
            tol = norm_tolerance(x, w, b, eps, layer, want, t_out, sections, kw.get("neighbours", False))
            assert np.all(np.abs(value(y, t_out) - want) <= tol), float((np.abs(value(y, t_out) - want) - tol).max())


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("D,sections", [(128, [20, 20, 16]), (40, [13])])
def test_norm_views_in_place(b200, backend, layer, offset, D, sections):
    """Queries and keys inside a fused projection's rows, in place; the values behind them and the rest are left alone;
    and heads outside rows."""
    rng = np.random.default_rng(3)
    rows, hq, hk, t = 37, 6, 2, "bf16"
    wide = store(rng.normal(size=(rows, hq + 2 * hk, D)) + 0.5, t)
    w = [store(1 + 0.2 * rng.normal(size=D), "f32") for _ in range(2)]
    pos = rng.integers(0, 5000, (len(sections), rows + 4))
    row = (hq + 2 * hk) * D
    xb = backend.upload(np.concatenate([np.zeros(offset, np.uint16), wide.reshape(-1)]))
    wb, pb = [backend.upload(x) for x in w], backend.upload(pos.astype(np.int32))
    out = backend.upload(np.full(rows * hq * D, 77, np.uint16))
    r = backend.rope(D, sections)
    at = lambda head: xb.ptr + 2 * (offset + head * D)
    H = b200.NormHeads
    r.norm([H(at(0), hq, wb[0].ptr, out.ptr, x_nb=(row, D), y_nb=(D, rows * D))], TYPES[t], pb.ptr, rows, TYPES[t], layer=layer, pos_stride=rows + 4)
    r.norm([H(at(0), hq, wb[0].ptr, at(0), x_nb=(row, D), y_nb=(row, D)), H(None, 0, None, None),
            H(at(hq), hk, wb[1].ptr, at(hq), x_nb=(row, D), y_nb=(row, D))], TYPES[t], pb.ptr, rows, TYPES[t], layer=layer, pos_stride=rows + 4)
    backend.synchronize()
    r.free()
    got = xb.get(wide.size + offset, np.uint16)[offset:].reshape(wide.shape)
    assert np.array_equal(got[:, hq + hk:], wide[:, hq + hk:])
    assert np.array_equal(out.get((hq, rows, D), np.uint16).transpose(1, 0, 2), got[:, :hq])
    for part, weight in ((slice(0, hq), w[0]), (slice(hq, hq + hk), w[1])):
        x = value(wide, t)[:, part]
        want = do.norm(x, weight, None, 1e-6, layer, pos[:, :rows], sections)
        assert np.all(np.abs(value(got, t)[:, part] - want) <= norm_tolerance(x, weight.astype(np.float64), None, 1e-6, layer, want, t, sections, False))


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("D,sections", [(128, [64]), (40, [13])])
def test_norm_extreme_values(b200, backend, layer, D, sections):
    """Heads of zeros, of huge and tiny elements, of one size throughout, and with a NaN or an infinity: other heads do not
    see them."""
    rng = np.random.default_rng(4)
    base = rng.normal(size=(1, 1, D))
    sizes = [0.0, 1.0, 1e-30, 1e-3, 1e15, 1e19, 1e25, 1e37]
    x = np.concatenate([base * s for s in sizes], 1).astype(np.float32)
    x = np.concatenate([x, np.full((1, 1, D), 5.0, np.float32), x[:, 1:2], x[:, 1:2], x[:, 1:2]], 1)
    x[0, -1, 3], x[0, -2, 4] = np.nan, np.inf
    w = store(1 + 0.2 * rng.normal(size=D), "f32")
    got, = run_norm(b200, backend, [x], [w], [None], "f32", "f32", "f32", [[7]], sections, 1e-6, layer)
    fine = x[:, :-2].astype(np.float64)
    want = do.norm(fine, w, None, 1e-6, layer, [[7]], sections)
    tol = norm_tolerance(fine, w.astype(np.float64), None, 1e-6, layer, want, "f32", sections, False) + 2.0 ** -120
    assert np.all(np.abs(got[:, :-2] - want) <= tol)
    assert np.isnan(got[0, -1]).all() and np.isnan(got[0, -2]).any()


# ---- the 4-bit cache -------------------------------------------------------------------------------------------


class Device:
    """A 4-bit cache and its batches on the GPU, next to the oracle's copy."""

    def __init__(self, b200, be, cache, table):
        self.b200, self.be, self.host = b200, be, {k: v.copy() for k, v in cache.items()}
        self.buf = {k: be.upload(v) for k, v in cache.items()}
        pages, heads, P, half = cache["k_codes"].shape
        self.D = 2 * half
        self.cache = b200.KV4Cache(*(self.buf[n].ptr for n in ("k_codes", "v_codes", "k_scale", "v_scale")), pages, heads, P, self.D)
        self.table_host = np.ascontiguousarray(table, np.int32)
        self.table = be.upload(self.table_host)

    def batch(self, row_start, kv_len, n_rows=None, max_len=None):
        keep = [self.be.upload(np.asarray(row_start, np.int32)), self.be.upload(np.asarray(kv_len, np.int32))]
        b = self.b200.KVBatch(self.table.ptr, self.table_host.shape[1], keep[0].ptr, keep[1].ptr, len(kv_len),
                              int(row_start[-1]) if n_rows is None else n_rows,
                              int(max(np.diff(row_start), default=0)), int(max(kv_len, default=0)) if max_len is None else max_len)
        b._keep = keep
        return b

    def put(self):
        for n, x in self.host.items():
            self.buf[n].set(x)

    def get(self):
        return {k: self.buf[k].get(v.shape, v.dtype) for k, v in self.host.items()}

    def write(self, k, v, t, row_start, kv_len):
        kb, vb = self.be.upload(store(k, t)), self.be.upload(store(v, t))
        self.be.kv4_write(self.cache, self.batch(row_start, kv_len), TYPES[t], kb.ptr, vb.ptr)
        self.be.synchronize()
        do.kv4_write(self.host, value(store(k, t), t), value(store(v, t), t), self.table_host, row_start, kv_len)

    def same(self):
        got = self.get()
        for n, want in self.host.items():
            assert np.array_equal(got[n], want), (n, np.argwhere(got[n] != want)[:5])


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("P,D,H", [(16, 64, 1), (16, 128, 3), (32, 64, 2), (64, 128, 2), (128, 64, 1), (128, 128, 9)])
def test_kv4_write_and_read(b200, backend, t, P, D, H):
    """Ragged runs of tokens appended in several calls; every code and scale of the cache, untouched ones included, equals
    the oracle's; then read back whole and in ragged ends."""
    rng = np.random.default_rng(P + D + H)
    steps = [[0, 5, P, 3], [1, 0, 2 * P + 7, P - 3], [P, 1, 1, 1], [1, 1, 1, 1], [2 * P, 3, 0, P + 1]]
    lens = np.sum(steps, 0)
    table, n = pages_for(lens, P)
    dev = Device(b200, backend, do.kv4_empty(n, H, P, D), table)
    at = np.zeros(4, int)
    for i, new in enumerate(steps):
        at += new
        rows = np.concatenate([[0], np.cumsum(new)])
        dev.write(rng.normal(size=(rows[-1], H, D)) * rng.choice([0.01, 1.0, 30.0], (rows[-1], 1, 1)), rng.normal(size=(rows[-1], H, D)) * 2.0 ** i,
                  t, rows, at)
        dev.same()
    for new in (lens, np.minimum(lens, [0, 1, P + 5, 9])):
        rows = np.concatenate([[0], np.cumsum(new)])
        want_k, want_v = do.kv4_read(dev.host, table, rows, lens)
        N = rows[-1]
        kb, vb = (backend.upload(np.full(N * H * D + 8, 77, dtype(t))) for _ in range(2))
        backend.kv4_read(dev.cache, dev.batch(rows, lens), TYPES[t], kb.ptr, vb.ptr, None, (D, N * D))
        backend.synchronize()
        got_k, got_v = kb.get(N * H * D + 8, dtype(t)), vb.get(N * H * D + 8, dtype(t))
        assert np.array_equal(got_k[:-8].reshape(N, H, D), store(want_k.astype(np.float32), t))
        assert np.array_equal(got_v[:-8].reshape(H, N, D).transpose(1, 0, 2), store(want_v.astype(np.float32), t))
        assert np.all(got_k[-8:] == 77) and np.all(got_v[-8:] == 77)


@pytest.mark.parametrize("D,H,t", [(64, 3, "bf16"), (128, 1, "f16"), (64, 1, "f32"), (128, 20, "bf16")])
@pytest.mark.parametrize("rows", [1, 2, 17])
def test_kv4_many_sequences(b200, backend, D, H, t, rows):
    """Hundreds of sequences with a few rows each: blocks of all slabs, heads that do not fill a block's turns."""
    rng = np.random.default_rng(rows)
    S, P = 700 // rows + 500, 16
    lens = rng.integers(rows, rows + 40, S)
    table, n = pages_for(lens, P)
    dev = Device(b200, backend, do.kv4_empty(n, H, P, D), table)
    start = np.arange(S + 1) * rows
    dev.write(rng.normal(size=(S * rows, H, D)), rng.normal(size=(S * rows, H, D)) * 5, t, start, lens)
    dev.same()
    want = do.kv4_read(dev.host, table, start, lens)
    out = [backend.alloc(S * rows * H * D * 4) for _ in range(2)]
    backend.kv4_read(dev.cache, dev.batch(start, lens), TYPES["f32"], out[0].ptr, out[1].ptr)
    backend.synchronize()
    assert all(np.array_equal(o.get(w.shape, np.float32), w.astype(np.float32)) for o, w in zip(out, want))


def test_kv4_write_rounds_the_exact_quotient(b200, backend):
    """Values on and next to the borders between two codes, largest magnitudes of both signs at once, NaN, infinities,
    zeros, subnormal and huge magnitudes."""
    rng = np.random.default_rng(5)
    P, D, H = 32, 128, 2
    for amax in (1.0, 8.0, 0.7300001, 3.1e38, 3.4e38, 1e-29, 2.0 ** -100, 2.0 ** -101, 5e-41):
        top = np.float32(amax)
        d = do.bf16_value(do.bf16_bits(top / np.float32(-8)))
        half = (np.arange(P * D) % 16 - 8 + 0.5) * d
        k = half.astype(np.float32).reshape(P, 1, D).repeat(H, 1)
        u = k.view(np.int32)
        u[:, 1] += rng.integers(-2, 3, u[:, 1].shape)  # a few steps to either side
        k = np.clip(u.view(np.float32).copy(), -top, top)
        k[:, 0, ::32], k[:, 1, 5::32] = top, -top
        k[::2, :, 7::32] = top  # of two of one magnitude the positive one
        v = (rng.normal(size=(P, H, D)) * np.float64(amax) / 4).clip(-top, top).astype(np.float32)
        v[3, 0, 5], v[4, 0, 6], v[5, 0, 7] = np.nan, np.inf, -np.inf
        v[6, 0, :32], v[7, 0, 32:64], v[8, 0] = np.nan, np.inf, 0.0
        for t in ("f32", "bf16") if amax > 65504 or amax < 1e-4 else ("f32", "bf16", "f16"):
            dev = Device(b200, backend, do.kv4_empty(3, H, P, D), [[1]])
            dev.write(k, v, t, [0, P], [P])
            dev.same()


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_kv4_write_of_every_16_bit_number(b200, backend, t):
    """Each number of the type next to largest ones of many sizes: every quotient that the type can make, ties among them."""
    P, D, H = 128, 128, 4
    every = np.arange(1 << 16, dtype=np.uint16).view(np.float16) if t == "f16" else np.arange(1 << 16, dtype=np.uint16)
    x = value(every, t)
    x = np.sort(np.where(np.isfinite(x), x, 0.0))
    rng = np.random.default_rng(7)
    for shift in range(3):  # a group's 32 numbers: of one size, from -7 steps to the largest
        base = np.abs(rng.choice(x[np.abs(x) > 2.0 ** -10], (P * H * D // 32 * 4, 1))).clip(2.0 ** -9, 2.0 ** 14)
        group = base * (np.arange(-16, 16) / 16 + (shift / 64 if shift else 0)) + base * rng.choice([0, 2.0 ** -9, -2.0 ** -9], (len(base), 32))
        group[np.arange(len(group)), rng.integers(0, 32, len(group))] = base[:, 0] * rng.choice([-1, 1], len(group))
        k, v = group[:2 * P * H * D // 32].reshape(2 * P, H, D), group[2 * P * H * D // 32:].reshape(2 * P, H, D)
        dev = Device(b200, backend, do.kv4_empty(3, H, P, D), [[2, 0]])
        dev.write(k, v, t, [0, 2 * P], [2 * P])
        dev.same()
    pages = len(x) // (P * D)  # and all of them in order
    dev = Device(b200, backend, do.kv4_empty(pages, 1, P, D), [list(range(pages))])
    dev.write(x.reshape(-1, 1, D), x[::-1].reshape(-1, 1, D), t, [0, pages * P], [pages * P])
    dev.same()


def test_kv4_views_and_broadcast_rows(b200, backend):
    """Keys and values inside one fused projection row, unaligned, and one row for all tokens."""
    rng = np.random.default_rng(6)
    P, D, H, N = 16, 64, 2, 41
    table, n = pages_for([N], P)
    for t, offset in (("bf16", 0), ("bf16", 3), ("f32", 1)):
        wide = store(rng.normal(size=(N * 6 * D + 8)), t)
        buf = backend.upload(wide)
        size = wide.itemsize
        dev = Device(b200, backend, do.kv4_empty(n, H, P, D), table)
        b = dev.batch([0, N], [N])
        backend.kv4_write(dev.cache, b, TYPES[t], buf.ptr + offset * size, buf.ptr + (offset + 2 * D) * size, (6 * D, D), (6 * D, 2 * D))
        rows = value(wide, t)[offset:offset + N * 6 * D].reshape(N, 6, D)
        do.kv4_write(dev.host, rows[:, :2], rows[:, 2::2][:, :2], table, [0, N], [N])
        backend.synchronize()
        dev.same()
        backend.kv4_write(dev.cache, b, TYPES[t], buf.ptr, buf.ptr, (0, D), (0, 0))
        one = value(wide, t)[:2 * D].reshape(1, 2, D)
        do.kv4_write(dev.host, one.repeat(N, 0), one[:, :1].repeat(N, 0).repeat(2, 1), table, [0, N], [N])
        backend.synchronize()
        dev.same()
        out = [backend.upload(np.full(N * (4 * D + 1) + 8, 77, dtype(t))) for _ in range(2)]
        backend.kv4_read(dev.cache, b, TYPES[t], out[0].ptr + size, out[1].ptr, (4 * D + 1, 2 * D), (2 * D, D))
        backend.synchronize()
        want = do.kv4_read(dev.host, table, [0, N], [N])
        got = out[0].get(N * (4 * D + 1) + 8, dtype(t))[1:N * (4 * D + 1) + 1].reshape(N, -1)
        assert np.array_equal(got[:, :4 * D].reshape(N, 4, D)[:, ::2], store(want[0].astype(np.float32), t))
        assert np.all(got[:-1, 4 * D] == 77) and np.all(got[:, :4 * D].reshape(N, 4, D)[:, 1::2] == 77)


def test_kv4_bad_tables_and_lengths_are_reported(b200, backend):
    """Entries outside the cache and arrays that contradict the sizes: an error at the next synchronize, nothing outside is
    touched, and the backend goes on."""
    P, D, H = 16, 64, 1
    host = do.kv4_empty(4, H, P, D)
    q = backend.upload(np.zeros((64, 2, D), np.float16))
    y = backend.upload(np.full((72, 2, D), 7, np.float16))
    rows = backend.upload(np.zeros((72, H, D), np.float16))
    att = backend.kv_attention()
    for table, row_start, kv_len, why in (([[9, 1]], [0, 20], [20], "page index"), ([[0, -1]], [0, 20], [20], "page index"),
                                          ([[0, 1]], [0, 20], [200], "contradicts"), ([[0, 1]], [0, 20], [-3], "contradicts"),
                                          ([[0, 1]], [-4, 20], [20], "contradicts"), ([[0, 1]], [0, 400], [20], "contradicts"),
                                          ([[0, 1], [2, 3]], [0, 20, 10], [20, 20], "contradicts")):
        for call in ("write", "read", "attend", "attend many"):
            dev = Device(b200, backend, host, table)
            b = dev.batch(row_start, kv_len, n_rows=64, max_len=32)
            b.max_rows = 64 if call == "attend many" or max(row_start) > 16 else 16
            if call == "write":
                backend.kv4_write(dev.cache, b, b200.TYPE_F16, rows.ptr, rows.ptr)
            elif call == "read":
                backend.kv4_read(dev.cache, b, b200.TYPE_F16, rows.ptr, rows.ptr + 36 * D * 2 * H)
            else:
                att.run(dev.cache, b, b200.TYPE_F16, q.ptr, 2, y.ptr, 0.1)
            with pytest.raises(b200.B200Error, match=why):
                backend.synchronize()
            backend.synchronize()
    assert np.all(y.get((72, 2, D), np.float16)[64:] == 7)
    att.free()


# ---- attention over it -----------------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def attend(backend):
    h = backend.kv_attention()
    yield h
    h.free()


def filled(b200, backend, lens, P, D, H, seed=0, size=1.0, spread=0.0):
    """A cache with tokens of all sequences, written by the oracle, memory behind them holding anything."""
    rng = np.random.default_rng(seed)
    table, n = pages_for(lens, P, seed=seed)
    host = do.kv4_empty(n, H, P, D, seed)
    rows = np.concatenate([[0], np.cumsum(lens)])
    scale = size * np.exp(spread * rng.normal(size=(rows[-1], 1, D // 32, 1)))
    v = (rng.normal(size=(rows[-1], H, D // 32, 32)) * scale).reshape(rows[-1], H, D)
    do.kv4_write(host, rng.normal(size=(rows[-1], H, D)), v, table, rows, lens)
    return Device(b200, backend, host, table)


def check_attention(dev, attend, q_raw, t, row_start, kv_len, n_heads, scale, causal=True, window=0, t_out=None, q_nb=None, y_nb=None,
                    n_rows=None, q=None, max_len=None):
    """Runs the call on packed or strided rows and compares every row of every sequence."""
    be, D = dev.be, dev.D
    t_out = t_out or t
    N = int(row_start[-1]) if n_rows is None else n_rows
    q = value(q_raw, t).reshape(N, n_heads, D) if q is None else q
    qb = be.upload(q_raw)
    size = N * n_heads * D if y_nb is None else (N - 1) * y_nb[0] + (n_heads - 1) * y_nb[1] + D
    yb = be.upload(np.full(size, 77, dtype(t_out)))
    attend.run(dev.cache, dev.batch(row_start, kv_len, n_rows=N, max_len=max_len), TYPES[t], qb.ptr, n_heads, yb.ptr, scale, causal=causal, window=window,
               y_type=TYPES[t_out], q_nb=q_nb, y_nb=y_nb)
    be.synchronize()
    raw = yb.get(size, dtype(t_out))
    s = raw.itemsize
    nb = (n_heads * D, D) if y_nb is None else y_nb
    raw = np.lib.stride_tricks.as_strided(raw, (N, n_heads, D), (nb[0] * s, nb[1] * s, s))
    got = value(raw, t_out)
    want = do.kv4_attention(dev.host, q, dev.table_host, row_start, kv_len, scale, causal, window)
    for i, length in enumerate(kv_len):
        r = slice(row_start[i], row_start[i + 1])
        first = max(length - (row_start[i + 1] - row_start[i]) - window + 1, 0) if window else 0
        v = np.abs(do.kv4_tokens(dev.host, "v", dev.table_host[i], first, length)).max((0, 2), initial=0.0)
        tol = 2.0 ** -10 * np.repeat(v, n_heads // len(v))[None, :, None] + at_least_half_step(want[r], t_out)
        assert np.array_equal(np.isnan(got[r]), np.isnan(want[r]))
        err = np.nan_to_num(np.abs(got[r] - want[r])) - np.nan_to_num(tol)
        over = (np.abs(want[r]) + tol > 65504) & (t_out == "f16")  # f16 has no such number: infinity, or its largest
        assert np.all((np.abs(got[r]) >= 65504 - tol)[over]) and np.array_equal(np.sign(got[r][over]), np.sign(want[r][over]))
        err[over] = 0
        assert np.all(err <= 0), (i, float(err.max()))
    owned = np.zeros(N, bool)
    owned[row_start[0]:row_start[-1]] = True
    assert np.all(raw[~owned] == 77)
    return got


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("P,D", [(16, 64), (16, 128), (32, 128), (64, 64), (128, 128)])
@pytest.mark.parametrize("H,G", GROUPS)
def test_kv4_attention_single_tokens(b200, backend, attend, t, P, D, H, G):
    rng = np.random.default_rng(P + D + H + G)
    lens = [1, 15, 16, 17, P, P + 1, 333, 700]
    dev = filled(b200, backend, lens, P, D, H)
    q = store(rng.normal(size=(len(lens), H * G, D)) * 2, t)
    check_attention(dev, attend, q, t, np.arange(len(lens) + 1), lens, H * G, D ** -0.5)
    check_attention(dev, attend, q, t, np.arange(len(lens) + 1), lens, H * G, D ** -0.5, window=40, t_out="f32")


@pytest.mark.parametrize("t,t_out", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("P,D", [(16, 64), (32, 128), (128, 64)])
@pytest.mark.parametrize("H,G", GROUPS)
def test_kv4_attention_several_rows(b200, backend, attend, t, t_out, P, D, H, G):
    """Drafted tokens, parts of prompts and whole prompts in one ragged batch, sequences without rows or tokens among them;
    causal, windowed and full."""
    rng = np.random.default_rng(P + D + H + G)
    rows, lens = [3, 0, 130, 7, 1, 40, 2], [90, 50, 130, 300, 1, 515, 0]
    start = np.concatenate([[0], np.cumsum(rows)])
    dev = filled(b200, backend, lens, P, D, H)
    q = store(rng.normal(size=(start[-1], H * G, D)) * 2, t)
    for kw in (dict(), dict(window=1), dict(window=37), dict(causal=False)):
        check_attention(dev, attend, q, t, start, lens, H * G, D ** -0.5, t_out=t_out, **kw)


@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 33, 200])
@pytest.mark.parametrize("D", [64, 128])
def test_kv4_attention_windows_over_memory_never_written(b200, backend, attend, rows, D):
    """Only the tokens that some row sees were written; in front of them, in the same page, and behind them lies anything."""
    rng = np.random.default_rng(rows)
    for window, length in ((5, 300), (40, 333), (100, 1000)):
        table, n = pages_for([length], 64)
        dev = Device(b200, backend, do.kv4_empty(n, 2, 64, D, rows), table)
        keep = min(length, rows + window - 1)
        dev.write(rng.normal(size=(keep, 2, D)), rng.normal(size=(keep, 2, D)), "f16", [0, keep], [length])
        q = store(rng.normal(size=(rows, 4, D)), "bf16")
        check_attention(dev, attend, q, "bf16", [0, rows], [length], 4, 0.1, window=window)


@pytest.mark.parametrize("rows", [1, 4, 70, 300])
def test_kv4_attention_rows_without_keys_are_zero(b200, backend, attend, rows):
    """More rows than tokens: the first rows see nothing; an empty cache: none does."""
    lens = [min(rows, 3) - 1, 0, 20]
    dev = filled(b200, backend, lens, 16, 128, 2, size=1e20)
    q = store(np.random.default_rng(0).normal(size=(3 * rows, 4, 128)), "f16")
    got = check_attention(dev, attend, q, "f16", np.arange(4) * rows, lens, 4, 0.1, t_out="f32")
    assert np.all(got[:rows - lens[0]] == 0) and np.all(got[rows:2 * rows] == 0)
    got = check_attention(dev, attend, q, "f16", np.arange(4) * rows, lens, 4, 0.1, causal=False, t_out="f32")
    assert np.all(got[rows:2 * rows] == 0)


@pytest.mark.parametrize("rows", [1, 200])
def test_kv4_attention_long_contexts_in_parts(b200, backend, attend, rows):
    """Key ranges that are cut into parts, of lengths around the cuts; a length far below max_len."""
    lens = [20000, 4096, 4097, 63, 12345]
    dev = filled(b200, backend, lens, 64, 128, 1)
    start = np.arange(6) * rows
    q = store(np.random.default_rng(1).normal(size=(5 * rows, 4, 128)) * 3, "bf16")
    check_attention(dev, attend, q, "bf16", start, lens, 4, 128 ** -0.5)
    check_attention(dev, attend, q, "bf16", start, lens, 4, 128 ** -0.5, window=5000)
    for bound in (100000, 1 << 30):
        check_attention(dev, attend, q, "bf16", start, lens, 4, 128 ** -0.5, max_len=bound)
        check_attention(dev, attend, q[:rows], "bf16", start[:2], lens[:1], 4, 128 ** -0.5, max_len=bound)


@pytest.mark.parametrize("D", [64, 128])
def test_kv4_attention_batches_without_rows(b200, backend, attend, D):
    """Rows that no sequence owns stay as they are; the arrays are checked all the same."""
    dev = filled(b200, backend, [30, 5], 16, D, 2)
    q, y = backend.upload(np.zeros((4, 2, D), np.float16)), backend.upload(np.full((4, 2, D), 7, np.float16))
    attend.run(dev.cache, dev.batch([0, 0, 0], [30, 5], n_rows=4), TYPES["f16"], q.ptr, 2, y.ptr, 0.1)
    backend.synchronize()
    assert np.all(y.get((4, 2, D), np.float16) == 7)
    b = dev.batch([0, 1, 1], [30, 5], n_rows=4)
    b.max_rows = 0
    attend.run(dev.cache, b, TYPES["f16"], q.ptr, 2, y.ptr, 0.1)
    with pytest.raises(b200.B200Error, match="contradicts"):
        backend.synchronize()


def handle_is_whole(b200, backend, handle, D):
    """Valid calls whose key ranges are cut into 2 and 3 parts, which between them use the first hundred counters of a
    handle as the first of a tile: each against the oracle."""
    rng = np.random.default_rng(D)
    for lens in ([200] * 50, [100] + [200] * 50, [300] * 34, [100] + [300] * 34, [200] + [300] * 34):
        dev = filled(b200, backend, lens, 16, D, 1)
        q = store(rng.normal(size=(len(lens), 1, D)), "f16")
        check_attention(dev, handle, q, "f16", np.arange(len(lens) + 1), lens, 1, 0.1)


@pytest.mark.parametrize("lens", [[200] + [300] * 11, [200] * 6 + [300] * 6])
def test_kv4_falling_starts_leave_the_handle_whole(b200, backend, lens):
    """Runs of rows that lie over one another, which make more parts than the host counted on: an error, and the calls
    behind it find every counter as it was."""
    D, rows = 64, 48
    dev = filled(b200, backend, lens, 16, D, 1)
    handle = backend.kv_attention()
    b = dev.batch([0, 16] + [0, rows] * 5 + [0], lens, n_rows=rows)
    b.max_rows = rows
    q, y = backend.upload(np.zeros((rows, 1, D), np.float16)), backend.upload(np.full((rows + 8, 1, D), 7, np.float16))
    for _ in range(2):
        handle.run(dev.cache, b, TYPES["f16"], q.ptr, 1, y.ptr, 0.1)
        with pytest.raises(b200.B200Error, match="contradicts"):
            backend.synchronize()
        handle_is_whole(b200, backend, handle, D)
    assert np.all(y.get((rows + 8, 1, D), np.float16)[rows:] == 7)
    handle.free()


@pytest.mark.parametrize("D,G,most", [(64, 1, 5), (64, 2, 24), (128, 2, 8)])
def test_kv4_bad_batches_of_few_rows(b200, backend, D, G, most):
    """The bad tables, lengths and starts by as few rows as the few-row kernel takes, over several parts: each is reported,
    nothing outside is touched, and the handle goes on."""
    P, rows = 16, 64
    host = do.kv4_empty(40, 1, P, D)
    good = np.arange(40).reshape(2, 20)
    bad = good.copy()
    bad[0, 3], bad[1, 19] = 40, -1
    handle = backend.kv_attention()
    q, y = backend.upload(np.zeros((rows, G, D), np.float16)), backend.upload(np.full((rows + 8, G, D), 7, np.float16))
    for table, row_start, kv_len, why in ((bad, [0, 5, 10], [320, 320], "page index"), (good, [0, most, most + 2], [320, 2000], "contradicts"),
                                          (good, [0, 3, 5], [-3, 300], "contradicts"), (good, [-4, 5, 9], [320, 300], "contradicts"),
                                          (good, [0, 5, 400], [320, 320], "contradicts"), (good, [0, 5, 2], [320, 320], "contradicts"),
                                          (good, [60, 5, 64], [320, 310], "contradicts"), (good, [0, most + 1, most + 2], [320, 200], "contradicts")):
        dev = Device(b200, backend, host, table)
        b = dev.batch(row_start, kv_len, n_rows=rows, max_len=320)
        b.max_rows = most
        for window in (0, 30):
            handle.run(dev.cache, b, TYPES["f16"], q.ptr, G, y.ptr, 0.1, window=window)
            with pytest.raises(b200.B200Error, match=why):
                backend.synchronize()
            backend.synchronize()
        handle_is_whole(b200, backend, handle, D)
    assert np.all(y.get((rows + 8, G, D), np.float16)[rows:] == 7)
    handle.free()


@pytest.mark.parametrize("S,H,D,rows", [(129, 2, 128, 1), (300, 1, 64, 3), (1200, 8, 64, 2), (257, 3, 128, 9)])
def test_kv4_attention_many_sequences(b200, backend, attend, S, H, D, rows):
    """More sequences than a block has threads, some without rows, one far longer than the others, so that most blocks
    have parts of it; more tiles than the workspace has parts."""
    rng = np.random.default_rng(S)
    lens = rng.integers(0, 40, S)
    lens[S // 2], lens[-1] = 9000, 3000
    n = rng.integers(0, rows + 1, S)
    n[[0, S // 2, S - 1]] = 0, rows, 1
    start = np.concatenate([[0], np.cumsum(n)])
    dev = filled(b200, backend, lens, 16, D, H)
    q = store(rng.normal(size=(start[-1], H, D)) * 2, "f16")
    check_attention(dev, attend, q, "f16", start, lens, H, D ** -0.5)
    check_attention(dev, attend, q, "f16", start, lens, H, D ** -0.5, window=700)
    check_attention(dev, attend, q, "f16", start, lens, H, D ** -0.5, max_len=1 << 30)


@pytest.mark.parametrize("rows", [2, 150])
def test_kv4_attention_views_and_rows_outside_sequences(b200, backend, attend, rows):
    """Queries inside a fused projection's rows, outputs with heads outside, unaligned data; rows in front of the first and
    behind the last sequence are left as they were."""
    rng = np.random.default_rng(2)
    D, H, G, lens = 64, 2, 3, [300, rows, 77 + rows]
    dev = filled(b200, backend, lens, 32, D, H)
    start = 5 + np.arange(4) * rows
    N = start[-1] + 9
    wide = store(rng.normal(size=(N, 10, D)), "f16")
    check_attention(dev, attend, wide, "f16", start, lens, 6, 0.2, q_nb=(10 * D, D), y_nb=(D, N * D), n_rows=N, q=value(wide, "f16")[:, :6])
    odd = store(rng.normal(size=(N, 6 * D + 3)), "f16")
    check_attention(dev, attend, odd, "f16", start, lens, 6, 0.2, q_nb=(6 * D + 3, D), y_nb=(6 * D + 1, D), n_rows=N,
                    q=value(odd, "f16")[:, :6 * D].reshape(N, 6, D))
    one = store(rng.normal(size=(1, D)), "f16")  # one query for all rows and heads
    check_attention(dev, attend, one, "f16", start, lens, 6, 0.2, q_nb=(0, 0), n_rows=N, q=np.broadcast_to(value(one, "f16"), (N, 6, D)))


@pytest.mark.parametrize("rows", [1, 12, 140])
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1.0, 1e-20, 1e30])
def test_kv4_attention_extreme_values(b200, backend, attend, t, rows, size):
    """Groups and tokens of very different scales, tokens of zeros, scores far apart, a NaN in one query, queries of huge
    and tiny size, a zero scale, values far from 1."""
    rng = np.random.default_rng(3)
    lens = [400 + rows, 64 + rows]
    dev = filled(b200, backend, lens, 16, 128, 1, size=size, spread=4.0)
    N, start = 2 * rows, [0, rows, 2 * rows]
    if size <= 1:
        for n in ("k", "v"):  # a page of zeros, and a group of zeros in another
            for page, g in ((dev.table_host[0][2], slice(0, 4)), (dev.table_host[0][4], slice(1, 2))):
                dev.host[n + "_scale"][page, :, :, g] = 0
        dev.put()
    x = rng.normal(size=(N, 2, 128))
    kw = dict(t_out="f32")
    check_attention(dev, attend, store(x * 30, t), t, start, lens, 2, 0.3, **kw)
    check_attention(dev, attend, store(x, t), t, start, lens, 2, 0.0, **kw)
    x[0, 1, 7] = np.nan
    got = check_attention(dev, attend, store(x, t), t, start, lens, 2, 0.1, **kw)
    assert np.isnan(got[0, 1]).all() and not np.isnan(got[0, 0]).any()
    if t == "bf16":
        x = rng.normal(size=(N, 2, 128))
        check_attention(dev, attend, store(x * 1e30, t), t, start, lens, 2, 1e-30, **kw)
        check_attention(dev, attend, store(x * 1e-30, t), t, start, lens, 2, 1e30, **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,rows", [(1, 1), (600, 1), (600, 5), (8, 70)])
@pytest.mark.parametrize("power", [-90, 0, 100, 115, 120, 124])
def test_kv4_light_tokens_count_at_every_size(b200, backend, attend, D, S, rows, power):
    """16000 tokens whose value scales are all next to 2^power, read by one sequence and by so many that parts of it are
    long: weights spread over many powers of two, and peaks with hundreds of light tokens around each, whose values differ in
    their mean.  The sum of the weights must not lose what the results keep, nor the results what the sum keeps."""
    rng = np.random.default_rng(rows)
    N, P = 16000, 128
    table, n = pages_for([N], P)
    dev = Device(b200, backend, do.kv4_empty(n, 1, P, D), np.repeat(table, S, 0))
    peaks = np.arange(77, N, 509)
    for peaked in (False, True):
        k = rng.normal(size=(N, 1, D)) * (0.05 if peaked else 1.0)
        k[peaks] = 1.0
        v = rng.uniform(-0.5, 0.5, (N, 1, D)) + 0.4
        v[peaks] -= 0.8
        v[..., ::32] = 1.0  # the largest of each group: -8 steps
        do.kv4_write(dev.host, k, v * 2.0 ** (power + 3), table, [0, N], [N])
        dev.put()
        q = store(np.ones((S * rows, 1, D)) if peaked else rng.normal(size=(S * rows, 1, D)) * 2, "bf16")
        scale = np.log(2.0 ** 14) / D if peaked else D ** -0.5  # a peak weighs as much as 2^14 light tokens
        qb, y = backend.upload(q), backend.alloc(S * rows * D * 4)
        attend.run(dev.cache, dev.batch(np.arange(S + 1) * rows, [N] * S), TYPES["bf16"], qb.ptr, 1, y.ptr, scale, causal=False, y_type=TYPES["f32"])
        backend.synchronize()
        got, want = y.get((S * rows, 1, D), np.float32), do.kv4_attention(dev.host, value(q, "bf16"), table, [0, S * rows], [N], scale, causal=False)
        assert np.all(np.abs(got - want) <= 2.0 ** -10 * 2.0 ** (power + 3) + at_least_half_step(want, "f32"))


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [4, 48])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_kv4_queries_that_are_not_numbers(b200, backend, attend, t, rows, bad):
    """One element of every other row: NaN makes the row NaN however few tokens it sees, infinities what the definition
    makes of them; the rows between are as without."""
    dev = filled(b200, backend, [48 + rows], 16, 64, 1)
    for n in ("k_codes", "v_codes"):  # no zeros: the sums of infinities are the definition's
        x = dev.host[n]
        x[:] = np.where(x & 15 == 8, x + 1, x)
        x[:] = np.where(x >> 4 == 8, x + 16, x)
    dev.put()
    x = np.random.default_rng(2).normal(size=(rows, 1, 64))
    x[::2, 0, 5] = bad
    for window in (1, 2, 4, 20, 0):
        got = check_attention(dev, attend, store(x, t), t, [0, rows], [48 + rows], 1, 0.125, window=window)
        assert not np.isnan(got[1::2]).any()
        if np.isnan(bad):
            assert np.isnan(got[::2]).all()


def test_kv4_and_8_bit_calls_share_a_handle(b200, backend, attend):
    """Calls over both caches, in parts, in turn with one handle: the same numbers as each alone."""
    from test_seq_cache_gpu import filled as filled8
    lens = [5000, 700]
    dev4, dev8 = filled(b200, backend, lens, 32, 128, 2), filled8(b200, backend, lens, 32, 128, 2)
    alone, own = {}, backend.kv_attention()
    for rows in (1, 40):
        q = backend.upload(store(np.random.default_rng(rows).normal(size=(2 * rows, 8, 128)), "f16"))
        for round_ in range(3):
            for name, dev in (("4", dev4), ("8", dev8)):
                y = backend.alloc(2 * rows * 8 * 128 * 2)
                (own if round_ == 0 else attend).run(dev.cache, dev.batch(np.arange(3) * rows, lens), TYPES["f16"], q.ptr, 8, y.ptr, 0.1)
                if round_ == 0:
                    backend.synchronize()
                alone.setdefault((name, rows), []).append(y)
    backend.synchronize()
    for (name, rows), ys in alone.items():
        first, *others = [y.get((2 * rows, 8, 128), np.uint16) for y in ys]
        assert all(np.array_equal(first, x) for x in others)
    own.free()


@pytest.mark.parametrize("rows", [1, 50])
def test_kv4_sequences_share_pages(b200, backend, attend, rows):
    """A common prompt's pages, a page that is not full among them, stand in the tables of several sequences; the first
    goes on in that page, the others from a copy of it; codes that lie there do not change."""
    P, D, H = 32, 64, 2
    common = 2 * P + 10
    table = np.array([[5, 2, 7, 0], [5, 2, 1, 3], [5, 2, 6, 4]])
    dev = Device(b200, backend, do.kv4_empty(8, H, P, D), table)
    rng = np.random.default_rng(9)
    k, v = rng.normal(size=(common, H, D)), rng.normal(size=(common, H, D))
    dev.write(k, v, "f16", [0, common, common, common], [common] * 3)
    for n, x in dev.host.items():
        x[1], x[6] = x[7], x[7]
    dev.put()
    lens = [common + rows, common + rows + 3, common + 20]
    start = np.concatenate([[0], np.cumsum(np.array(lens) - common)])
    before = dev.get()
    dev.write(rng.normal(size=(start[-1], H, D)) * 100, rng.normal(size=(start[-1], H, D)) * 100, "f16", start, lens)
    dev.same()
    assert all(np.array_equal(before[n][[1, 6, 7], :, :10], dev.get()[n][[1, 6, 7], :, :10]) for n in before)
    q = store(rng.normal(size=(3 * rows, 4, D)), "f16")
    check_attention(dev, attend, q, "f16", np.arange(4) * rows, lens, 4, 0.125)


def test_kv4_pages_behind_four_gigabytes(b200, backend, attend):
    """Codes whose offsets pass 32 bits: written, read and attended to as in a small cache, bit for bit."""
    P, D, H, lens = 128, 128, 8, [300, 1000]
    small_table, n = pages_for(lens, P)
    far = 66000  # pages of 64 KiB
    far_table = np.where(small_table < n, small_table + far, small_table).astype(np.int32)
    rng = np.random.default_rng(10)
    start = np.concatenate([[0], np.cumsum(lens)])
    k, v = (backend.upload(store(rng.normal(size=(start[-1], H, D)), "bf16")) for _ in range(2))
    q = {r: backend.upload(store(rng.normal(size=(2 * r, 16, D)), "bf16")) for r in (1, 40)}
    results = []
    for pages, table in ((n, small_table), (n + far, far_table)):
        codes, scales = [backend.alloc(pages * H * P * D // 2) for _ in range(2)], [backend.alloc(pages * H * P * D // 16) for _ in range(2)]
        cache = b200.KV4Cache(codes[0].ptr, codes[1].ptr, scales[0].ptr, scales[1].ptr, pages, H, P, D)
        keep = [backend.upload(np.ascontiguousarray(x, np.int32)) for x in (table, start, lens)]
        batch = b200.KVBatch(keep[0].ptr, table.shape[1], keep[1].ptr, keep[2].ptr, 2, int(start[-1]), max(lens), max(lens))
        backend.kv4_write(cache, batch, TYPES["bf16"], k.ptr, v.ptr)
        out = [backend.alloc(int(start[-1]) * H * D * 4) for _ in range(2)]
        backend.kv4_read(cache, batch, TYPES["f32"], out[0].ptr, out[1].ptr)
        got = [o.get((start[-1], H, D), np.float32) for o in out]
        for r in q:
            at = backend.upload(np.array([0, r, 2 * r], np.int32))
            y = backend.alloc(2 * r * 16 * D * 2)
            b = b200.KVBatch(keep[0].ptr, table.shape[1], at.ptr, keep[2].ptr, 2, 2 * r, r, max(lens))
            attend.run(cache, b, TYPES["bf16"], q[r].ptr, 16, y.ptr, 0.09)
            backend.synchronize()
            got.append(y.get((2 * r, 16, D), np.uint16))
        results.append(got)
        for x in codes + scales:
            x.free()
    assert all(np.array_equal(a, b) for a, b in zip(*results))
    assert np.abs(results[0][0]).max() > 1


def test_kv4_results_repeat_bit_for_bit(b200, backend, attend):
    lens = [9000, 100, 5000]
    dev = filled(b200, backend, lens, 32, 128, 2)
    for rows in (1, 33):
        q = store(np.random.default_rng(4).normal(size=(3 * rows, 8, 128)), "f16")
        runs = [check_attention(dev, attend, q, "f16", np.arange(4) * rows, lens, 8, 0.1) for _ in range(3)]
        assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])


@pytest.mark.parametrize("rows,G", [(1, 4), (6, 2), (60, 2)])
def test_kv4_results_over_the_queries(b200, backend, attend, rows, G):
    """y is q: the same numbers as into a tensor of its own."""
    lens = [300, 2000]
    dev = filled(b200, backend, lens, 32, 64, 2)
    q = store(np.random.default_rng(5).normal(size=(2 * rows, 2 * G, 64)), "f16")
    want = check_attention(dev, attend, q, "f16", np.arange(3) * rows, lens, 2 * G, 0.1)
    buf = backend.upload(q)
    attend.run(dev.cache, dev.batch(np.arange(3) * rows, lens), TYPES["f16"], buf.ptr, 2 * G, buf.ptr, 0.1)
    backend.synchronize()
    assert np.array_equal(buf.get(q.shape, np.float16), want.astype(np.float16))


# ---- products with 4-bit weights -------------------------------------------------------------------------------


def check_vec(b200, be, raw, kind, N, K, x, t, t_out, bias=None, ldx=None, ldy=None, offset=0, handle=None):
    """x: raw rows [M][K]; returns the raw results [M][N]."""
    M = x.shape[0]
    w = handle or be.weight(b200.TYPE_Q4_0 if kind == "q4_0" else b200.TYPE_Q4_1, raw, K, N)
    ldx, ldy = ldx or K, ldy or N
    rows = np.full(offset + M * ldx, 7, dtype(t))
    for m in range(M):
        rows[offset + m * ldx:offset + m * ldx + K] = x[m]
    xb, yb = be.upload(rows), be.upload(np.full(offset + M * ldy + 5, 77, dtype(t_out)))
    bb = None if bias is None else be.upload(bias)
    be.mul_mat_vec(w, xb.ptr + offset * rows.itemsize, TYPES[t], M, yb.ptr + offset * np.dtype(dtype(t_out)).itemsize, TYPES[t_out],
                   bias=None if bb is None else bb.ptr, ldx=ldx, ldy=ldy)
    be.synchronize()
    y = yb.get(offset + M * ldy + 5, dtype(t_out))
    got = np.lib.stride_tricks.as_strided(y[offset:], (M, N), (ldy * y.itemsize, y.itemsize)).copy()
    rest = y[offset:offset + (M - 1) * ldy + N].copy()
    for m in range(M):
        rest[m * ldy:m * ldy + N] = 77
    assert np.all(rest == 77) and np.all(y[:offset] == 77) and np.all(y[offset + (M - 1) * ldy + N:] == 77)
    if handle is None:
        w.free()
    d, code, low = do.parts(raw, kind, N, K)
    v = value(x, t)
    with np.errstate(invalid="ignore", over="ignore"):
        want = v @ (d * code + low).T + (0 if bias is None else bias.astype(np.float64))
        most = np.abs(v) @ (np.abs(d * code) + np.abs(low)).T
        tol = most * (33 * 2.0 ** -23 + (K / 32 + 12) * 2.0 ** -24) + np.abs(want) * 2.0 ** -23
        if t != "f16":
            tol += most * 2.0 ** -23 + 2.0 ** -26 * np.abs(v).max(1, keepdims=True) * (np.abs(d * code) + np.abs(low)).sum(1)
        tol += at_least_half_step(want, t_out)
    got_v = value(got, t_out)
    assert np.array_equal(np.isfinite(got_v), np.isfinite(want))
    fine = np.isfinite(want)
    assert np.all(np.abs(got_v - want)[fine] <= tol[fine]), float((np.abs(got_v - want) - tol)[fine].max())
    return got


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("t,t_out", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("K", [32, 64, 160, 1024, 4128])
def test_vec(b200, backend, kind, t, t_out, K):
    rng = np.random.default_rng(K)
    for N, M, bias in ((1, 1, False), (16, 2, True), (17, 5, False), (300, 8, True), (1029, 9, False), (40, 16, True)):
        raw = do.blocks(rng, kind, N, K)
        x = store(rng.normal(size=(M, K)), t)
        check_vec(b200, backend, raw, kind, N, K, x, t, t_out, bias=rng.normal(size=N).astype(np.float32) if bias else None)


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_vec_long_rows_in_phases(b200, backend, kind, t):
    """More k than x has shared memory for, and few and many rows of the weights."""
    rng = np.random.default_rng(1)
    for N, K, M in ((33, 16384 + 96, 16), (2500, 8192, 7), (5, 65536, 3), (20000, 1056, 15)):
        raw = do.blocks(rng, kind, N, K)
        check_vec(b200, backend, raw, kind, N, K, store(rng.normal(size=(M, K)), t), t, "f32")


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_vec_views(b200, backend, t):
    """Rows inside wider ones, unaligned, results into wider rows; a weight with many more rows than a wave has tiles."""
    rng = np.random.default_rng(2)
    N, K = 90, 320
    raw = do.blocks(rng, "q4_0", N, K)
    x = store(rng.normal(size=(3, K)), t)
    plain = check_vec(b200, backend, raw, "q4_0", N, K, x, t, t)
    for ldx, ldy, offset in ((K + 4, N + 3, 0), (K + 1, N, 1), (2 * K, 2 * N, 3)):
        assert np.array_equal(plain, check_vec(b200, backend, raw, "q4_0", N, K, x, t, t, ldx=ldx, ldy=ldy, offset=offset))
    raw = do.blocks(rng, "q4_1", 80001, 64)
    check_vec(b200, backend, raw, "q4_1", 80001, 64, store(rng.normal(size=(2, 64)), t), t, t)


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_vec_extreme_values(b200, backend, kind, t):
    """Rows of zeros, of huge and tiny elements, of elements far apart, an infinity or a NaN in one row; scales of zero."""
    rng = np.random.default_rng(3)
    N, K = 50, 256
    raw = do.blocks(rng, kind, N, K)
    raw[5 * (K // 32) + 2, :2] = 0
    x = rng.normal(size=(8, K))
    x[1] = 0
    if t == "f16":
        x[2] *= 60000 / np.abs(x[2]).max()
        x[3] *= 1e-5
    else:
        x[2] *= 1e30
        x[3] *= 1e-30
        x[4] *= 10.0 ** rng.uniform(-20, 20, K)
    check_vec(b200, backend, raw, kind, N, K, store(x, t), t, "f32")
    if t != "f16":  # rows at the ends of the sizes that are taken as usual ones, alone and beside others
        for size in (2.0 ** -5, 2.0 ** -5 * 0.99, 511.0, 512.0, 600.0):
            y = rng.normal(size=(3, K))
            y *= size / np.abs(y[1]).max()
            y[0], y[2] = y[0] / size, y[2] * 1e-3
            check_vec(b200, backend, raw, kind, N, K, store(y, t), t, "f32")
            check_vec(b200, backend, raw, kind, N, K, store(y[1:2], t), t, "f32")
    # no code is 0 and no weight 0, so that an infinity stays one
    raw[:, 2 if kind == "q4_0" else 4:] = 0x5B
    if kind == "q4_1":
        raw[:, 2:4] = 0
    raw[:, :2] = np.array([0.25], np.float16).view(np.uint8)
    x[6, 7], x[7, 9] = np.inf, np.nan
    if kind == "q4_0":
        check_vec(b200, backend, raw, kind, N, K, store(x, t), t, "f32")


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("t,t_out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("N,K,M", [(50, 256, 3), (301, 4128, 9), (33, 16384 + 96, 16)])
def test_vec_elements_that_are_not_numbers(b200, backend, kind, t, t_out, N, K, M):
    """Infinities alone, several of one sign and of both, NaN, beside finite elements of usual size and not, with weights
    above, below and exactly 0: the result is the definition's, sign and all, and rows without any are as ever."""
    rng = np.random.default_rng(K)
    raw = do.blocks(rng, kind, N, K)
    if kind == "q4_1":  # minima that are a whole number of steps, so that some weights are exactly 0
        d = np.float16(2.0) ** rng.integers(-6, -2, len(raw)).astype(np.float16) * rng.choice([-1, 1], len(raw)).astype(np.float16)
        raw[:, :2] = d[:, None].view(np.uint8)
        raw[:, 2:4] = (d * rng.integers(-15, 1, len(raw)).astype(np.float16))[:, None].view(np.uint8)
    assert (do.weight(raw, kind, N, K) == 0).any()
    w = backend.weight(b200.TYPE_Q4_0 if kind == "q4_0" else b200.TYPE_Q4_1, raw, K, N)
    plain = store(rng.normal(size=(M, K)), t)
    bias = rng.normal(size=N).astype(np.float32)
    usual = check_vec(b200, backend, raw, kind, N, K, plain, t, t_out, bias=bias, handle=w)
    for size in (1.0,) if t == "f16" else (1.0, 1e20):
        x = rng.normal(size=(M, K)) * size
        places = [rng.choice(K, 12, replace=False) for _ in range(3)]
        x[0, places[0][0]] = np.inf
        x[M - 1, places[1][:2]] = -np.inf
        x[M // 2, places[2][:6]] = rng.choice([np.inf, -np.inf], 6)
        got = check_vec(b200, backend, raw, kind, N, K, store(x, t), t, t_out, bias=bias, handle=w)
        with np.errstate(invalid="ignore"):
            want = value(store(x, t), t) @ do.weight(raw, kind, N, K).T
        odd = [0, M // 2, M - 1]
        assert np.isinf(want[0]).any() and np.isnan(want[0]).any()
        assert np.array_equal(value(got, t_out)[odd], want[odd], equal_nan=True)
        x = rng.normal(size=(M, K))
        x[:, 3] = np.nan
        x[0], x[1] = value(plain, t)[0], np.inf
        got = check_vec(b200, backend, raw, kind, N, K, store(x, t), t, t_out, bias=bias, handle=w)
        assert np.array_equal(got[0], usual[0]) and np.isnan(value(got, t_out)[2:]).all()
    w.free()


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_vec_sums_past_the_range(b200, backend, kind, t):
    """Finite elements whose sum no f32 holds give infinities of its sign."""
    N, K = 40, 128
    raw = do.blocks(np.random.default_rng(8), kind, N, K, size=0.5)
    sign = np.sign(do.weight(raw, kind, N, K))
    x = store(np.stack([sign[3], -sign[7], sign[0] * 1e-38]) * 3e38, t)
    xb, yb, w = backend.upload(x), backend.alloc(3 * N * 4), backend.weight(b200.TYPE_Q4_0 if kind == "q4_0" else b200.TYPE_Q4_1, raw, K, N)
    backend.mul_mat_vec(w, xb.ptr, TYPES[t], 3, yb.ptr, b200.TYPE_F32)
    backend.synchronize()
    got, want = yb.get((3, N), np.float32), value(x, t) @ do.weight(raw, kind, N, K).T
    past, within = np.abs(want) > 2.0 ** 128, np.abs(want) < 2.0 ** 127
    assert past[0, 3] and past[1, 7] and np.array_equal(got[past], np.sign(want[past]) * np.inf) and np.isfinite(got[within]).all()
    w.free()


def test_vec_beside_the_other_products(b200, backend, model):
    """One handle serves mul_mat, mul_mat_dq16 and mul_mat_vec; activations that Q8_0 holds exactly give the same sums up to
    f32; results repeat bit for bit."""
    rng = np.random.default_rng(4)
    N, K, M = 200, 512, 3
    raw = do.blocks(rng, "q4_0", N, K)
    w = backend.weight(b200.TYPE_Q4_0, raw, K, N)
    x = rng.integers(-127, 128, (M, K)).astype(np.float32)
    x[:, ::32] = 127
    xb, yb = backend.upload(x), backend.alloc(M * N * 4)
    backend.mul_mat(w, xb, M, yb)
    backend.synchronize()
    exact = yb.get((M, N), np.float32)
    runs = [check_vec(b200, backend, raw, "q4_0", N, K, x, "f32", "f32", handle=w) for _ in range(3)]
    assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])
    assert np.abs(runs[0] - exact).max() <= 2.0 ** -19 * (np.abs(x).astype(np.float64) @ np.abs(do.weight(raw, "q4_0", N, K)).T).max()
    w.free()


def test_vec_weights_from_device_memory(b200, backend):
    """Blocks that lie on the GPU, by address, are the same weight."""
    rng = np.random.default_rng(6)
    N, K = 70, 192
    for kind in ("q4_0", "q4_1"):
        raw = do.blocks(rng, kind, N, K)
        buf = backend.upload(raw)
        for at in (buf.ptr, np.int64(buf.ptr)):
            w = backend.weight(b200.TYPE_Q4_0 if kind == "q4_0" else b200.TYPE_Q4_1, at, K, N)
            check_vec(b200, backend, raw, kind, N, K, store(rng.normal(size=(2, K)), "f32"), "f32", "f32", handle=w)
            w.free()


def test_vec_refusals(b200, backend):
    K, N = 64, 8
    w = backend.weight(b200.TYPE_Q4_0, do.blocks(np.random.default_rng(0), "q4_0", N, K), K, N)
    dense = backend.weight(b200.TYPE_F16, np.zeros((N, K), np.float16).view(np.uint8), K, N)
    q8 = backend.weight(b200.TYPE_Q8_0, np.zeros((N * K // 32, 34), np.uint8), K, N)
    buf = backend.alloc(4096)
    F32, F16, BF16 = b200.TYPE_F32, b200.TYPE_F16, b200.TYPE_BF16
    good = dict(w=w, x=buf.ptr, x_type=F16, M=1, y=buf.ptr + 2048, y_type=F16)
    for change, why in ((dict(w=dense), "weight type"), (dict(w=q8), "weight type"), (dict(M=17), "bad shape"), (dict(M=-1), "bad shape"),
                        (dict(ldx=K - 1), "bad shape"), (dict(ldy=N - 1), "bad shape"), (dict(y_type=BF16), "unsupported types"),
                        (dict(x_type=b200.TYPE_Q8_0), "unsupported types"), (dict(x_type=F32, y_type=F16), "unsupported types"),
                        (dict(x=buf.ptr + 1), "unaligned"), (dict(y=buf.ptr + 1), "unaligned"), (dict(bias=buf.ptr + 2), "unaligned")):
        with pytest.raises(b200.B200Error, match=why):
            backend.mul_mat_vec(**{**good, **change})
    backend.mul_mat_vec(**{**good, "M": 0})
    backend.synchronize()
    for x in (w, dense, q8):
        x.free()


def test_vec_results_beside_and_over_x(b200, backend):
    """x and dst in the same rows side by side, and in turn, are fine; dst over x or the bias is refused."""
    rng = np.random.default_rng(7)
    N, K, M, F16, F32 = 96, 64, 5, b200.TYPE_F16, b200.TYPE_F32
    raw = do.blocks(rng, "q4_1", N, K)
    w, x = backend.weight(b200.TYPE_Q4_1, raw, K, N), rng.normal(size=(M, K)).astype(np.float16)
    want = check_vec(b200, backend, raw, "q4_1", N, K, x, "f16", "f16", handle=w)
    for first in (True, False):  # x in front of dst, and behind
        rows = np.zeros((M, K + N), np.float16)
        at_x, at_y = (0, K) if first else (N, 0)
        rows[:, at_x:at_x + K] = x
        buf = backend.upload(rows)
        backend.mul_mat_vec(w, buf.ptr + 2 * at_x, F16, M, buf.ptr + 2 * at_y, F16, ldx=K + N, ldy=K + N)
        backend.synchronize()
        got = buf.get(rows.shape, np.float16)
        assert np.array_equal(got[:, at_x:at_x + K], x) and np.array_equal(got[:, at_y:at_y + N], want)
    buf, b = backend.alloc(1 << 16), 1 << 12
    for kw in (dict(y=buf.ptr), dict(y=buf.ptr + 2 * K - 2), dict(y=buf.ptr + 2 * K, ldx=K + N - 1, ldy=K + N - 1), dict(y=buf.ptr, y_type=F32),
               dict(x=buf.ptr + 2 * N - 2, y=buf.ptr, M=1), dict(x=buf.ptr + 20 * N, y=buf.ptr, ldy=5 * N),
               dict(y=buf.ptr + b, bias=buf.ptr + b + 2 * N * M - 4), dict(y=buf.ptr + b, bias=buf.ptr + b - 4 * N + 4)):
        with pytest.raises(b200.B200Error, match="dst overlaps"):
            backend.mul_mat_vec(w, **{**dict(x=buf.ptr, x_type=F16, M=M, y_type=F16), **kw})
    w.free()


# ---- together --------------------------------------------------------------------------------------------------


class Layer:
    """A decoder layer's step: projection, norms and rotation, cache, attention, projection back."""

    def __init__(self, b200, be, rng, table, pages, P):
        self.b200, self.be = b200, be
        self.H, self.G, self.D, self.K, self.P = 2, 2, 64, 256, P
        self.heads, self.width = self.H * self.G, (self.H * self.G + 2 * self.H) * self.D
        self.raw = [do.blocks(rng, "q4_1", self.width, self.K), do.blocks(rng, "q4_0", self.K, self.heads * self.D)]
        self.w = [be.weight(b200.TYPE_Q4_1, self.raw[0], self.K, self.width), be.weight(b200.TYPE_Q4_0, self.raw[1], self.heads * self.D, self.K)]
        self.norms = [store(1 + 0.2 * rng.normal(size=self.D), "f32") for _ in range(2)]
        self.norm_bufs = [be.upload(x) for x in self.norms]
        self.rope, self.attend = be.rope(self.D, [16, 16], base=1e5), be.kv_attention()
        self.dev = Device(b200, be, do.kv4_empty(pages, self.H, P, self.D), table)

    def buffers(self, S):
        be = self.be
        return dict(x=be.alloc(S * self.K * 2), pos=be.alloc(2 * S * 4), qkv=be.alloc(S * self.width * 2), q=be.alloc(S * self.heads * self.D * 2),
                    o=be.alloc(S * self.heads * self.D * 2), y=be.alloc(S * self.K * 2))

    def step(self, b, batch, S):
        t, H, D, row = self.b200.TYPE_F16, self.b200.NormHeads, self.D, self.width
        at = lambda head: b["qkv"].ptr + head * D * 2
        self.be.mul_mat_vec(self.w[0], b["x"].ptr, t, S, b["qkv"].ptr, t)
        self.rope.norm([H(at(0), self.heads, self.norm_bufs[0].ptr, b["q"].ptr, x_nb=(row, D)),
                        H(at(self.heads), self.H, self.norm_bufs[1].ptr, at(self.heads), x_nb=(row, D), y_nb=(row, D))], t, b["pos"].ptr, S, t)
        self.be.kv4_write(self.dev.cache, batch, t, at(self.heads), at(self.heads + self.H), (row, D), (row, D))
        self.attend.run(self.dev.cache, batch, t, b["q"].ptr, self.heads, b["o"].ptr, 0.125)
        self.be.mul_mat_vec(self.w[1], b["o"].ptr, t, S, b["y"].ptr, t)

    def free(self):
        for h in (*self.w, self.rope, self.attend):
            h.free()


def test_steps_of_a_layer(b200, backend):
    """Steps of several sequences through all five calls, each result against the oracle on what the call was given, and
    the cache against the oracle's at the end."""
    rng = np.random.default_rng(11)
    S, P, steps = 3, 16, 20
    table, n = pages_for([steps] * S, P)
    m = Layer(b200, backend, rng, table, n, P)
    b, D = m.buffers(S), m.D
    for i in range(steps):
        x = store(rng.normal(size=(S, m.K)), "f16")
        pos = np.full((2, S), i) + [[0], [7]]
        lens = [i + 1] * S
        b["x"].set(x)
        b["pos"].set(pos.astype(np.int32))
        m.step(b, m.dev.batch(np.arange(S + 1), lens), S)
        backend.synchronize()
        qkv = b["qkv"].get((S, m.width // D, D), np.float16).astype(np.float64)
        q, o, y = (b[k].get(shape, np.float16).astype(np.float64) for k, shape in
                   (("q", (S, m.heads, D)), ("o", (S, m.heads, D)), ("y", (S, m.K))))
        first = x.astype(np.float64) @ do.weight(m.raw[0], "q4_1", m.width, m.K).T
        close = lambda got, want, size: np.abs(got - want).max() <= 2.0 ** -10 * size
        raw_q, raw_k = (first.reshape(S, -1, D)[:, s] for s in (slice(0, m.heads), slice(m.heads, m.heads + m.H)))
        want_q = do.norm(qkv[:, :m.heads], m.norms[0], None, 1e-6, False, pos, [16, 16], base=1e5)
        want_k = do.norm(store(raw_k, "f16").astype(np.float64), m.norms[1], None, 1e-6, False, pos, [16, 16], base=1e5)
        assert close(qkv[:, :m.heads], raw_q, np.abs(raw_q).max()) and close(q, want_q, np.abs(want_q).max())
        assert close(qkv[:, m.heads:m.heads + m.H], want_k, 4 * np.abs(want_k).max())
        assert close(qkv[:, m.heads + m.H:].reshape(S, -1), first[:, (m.heads + m.H) * D:], np.abs(first).max())
        do.kv4_write(m.dev.host, qkv[:, m.heads:m.heads + m.H], qkv[:, m.heads + m.H:], table, np.arange(S + 1), lens)
        want_o = do.kv4_attention(m.dev.host, q, table, np.arange(S + 1), lens, 0.125)
        most = max(np.abs(do.kv4_tokens(m.dev.host, "v", table[s], 0, i + 1)).max() for s in range(S))
        assert close(o, want_o, 2 * most)
        want_y = o.reshape(S, -1) @ do.weight(m.raw[1], "q4_0", m.K, m.heads * D).T
        assert close(y, want_y, np.abs(want_y).max())
    m.dev.same()
    m.free()


@pytest.mark.parametrize("again", [1, 2])
def test_a_captured_step_of_a_layer(b200, backend, again):
    """The step captured from the backend's stream and replayed with new inputs, lengths and positions matches direct calls
    bit for bit."""
    import torch
    rng = np.random.default_rng(12)
    S, P, steps = 5, 16, 12
    table, n = pages_for([steps] * S, P)
    m, twin = (Layer(b200, backend, np.random.default_rng(1), table, n, P) for _ in range(2))
    b, b2 = m.buffers(S), twin.buffers(S)
    batch = m.dev.batch(np.arange(S + 1), [1] * S, max_len=steps)
    stream, graph = torch.cuda.ExternalStream(backend.stream), torch.cuda.CUDAGraph()
    if again == 2:  # a graph may be the first use of every call, or not
        m.step(b, batch, S)
        backend.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        m.step(b, batch, S)
    for i in range(steps):
        x, pos = store(rng.normal(size=(S, m.K)), "f16"), np.full((2, S), i, np.int32)
        batch._keep[1].set(np.full(S, i + 1, np.int32))
        for d in (b, b2):
            d["x"].set(x)
            d["pos"].set(pos)
        with torch.cuda.stream(stream):
            graph.replay()
        twin.step(b2, twin.dev.batch(np.arange(S + 1), [i + 1] * S, max_len=steps), S)
        backend.synchronize()
        assert np.array_equal(b["y"].get((S, m.K), np.uint16), b2["y"].get((S, m.K), np.uint16))
    a, c = m.dev.get(), twin.dev.get()
    written = {k: [c[k][table[s][t // P], :, t % P] for s in range(S) for t in range(steps)] for k in c}
    assert all(np.array_equal([a[k][table[s][t // P], :, t % P] for s in range(S) for t in range(steps)], written[k]) for k in a)
    del graph
    m.free()
    twin.free()


@pytest.mark.parametrize("captured", [False, True])
def test_a_step_waits_for_another_stream_and_is_waited_for(b200, backend, captured):
    """Steps whose input slow work of another stream makes, ordered by events, with the results kept by that stream: any
    call that started early, or any work that did not see a call's results, gives other numbers."""
    import torch
    S, P = 4, 16
    table, n = pages_for([8] * S, P)
    m = Layer(b200, backend, np.random.default_rng(2), table, n, P)
    b = m.buffers(S)
    src = torch.randn(S, m.K, device="cuda").half()
    x, y = torch.zeros_like(src), torch.zeros_like(src)
    b["x"], b["y"] = type("B", (), {"ptr": x.data_ptr()}), type("B", (), {"ptr": y.data_ptr()})
    b["pos"].set(np.zeros((2, S), np.int32))
    kept, slow = torch.zeros(4, *y.shape, dtype=torch.float16, device="cuda"), torch.zeros(1 << 26, device="cuda")
    batches = [m.dev.batch(np.arange(S + 1), [i + 1] * S, max_len=8) for i in range(4)]
    own, side = torch.cuda.ExternalStream(backend.stream), torch.cuda.Stream()
    torch.cuda.synchronize()

    def work():
        for i in range(4):
            side.wait_stream(own)
            with torch.cuda.stream(side):
                if i:
                    kept[i - 1].copy_(y)
                slow.add_(1.0)
                x.copy_(src).mul_(1.0 + i)
            own.wait_stream(side)
            m.step(b, batches[i], S)
        side.wait_stream(own)
        with torch.cuda.stream(side):
            kept[3].copy_(y)
        own.wait_stream(side)

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=own):
            work()
        with torch.cuda.stream(own):
            graph.replay()
    else:
        work()
    torch.cuda.synchronize()
    backend.synchronize()
    got = kept.cpu().numpy()
    for i in range(4):
        x.copy_(src).mul_(1.0 + i)
        torch.cuda.synchronize()
        m.step(b, batches[i], S)
        backend.synchronize()
        assert np.array_equal(got[i], y.cpu().numpy())
    assert not np.array_equal(got[0], got[1])
    if captured:
        del graph
    m.free()


@pytest.mark.parametrize("name", ["norm_step", "cache_step", "attend_one", "vec_small"])
def test_the_measured_cases_are_ordered_with_torch(name):
    """The library form of the measured cases follows torch's current stream, and that stream follows it."""
    import torch
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "more_operators.py")
    spec = importlib.util.spec_from_file_location("more_measured_cases", path)
    cases = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = cases
    spec.loader.exec_module(cases)
    case = next(c for c in cases.listed() if c["name"] == name)
    before = torch.cuda.current_stream()
    inputs = {"norm": ["x"], "cache": ["k", "v"], "attend": ["q"], "vec": ["x"]}[case["op"]]
    slow = torch.zeros(1 << 28, device="cuda")
    try:
        cases.own = True
        for stream in (None, torch.cuda.Stream()):  # as prepare() leaves it, and under a stream of the program's own
            state = cases.prepare(case, 1)
            torch.cuda.synchronize()
            want = cases.run(state)
            torch.cuda.synchronize()
            want = [w.clone() for w in (want if isinstance(want, tuple) else [want])]
            source = {n: state[n].clone() for n in inputs}
            for n in inputs:
                state[n].zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                slow.add_(1.0)
                for n in inputs:
                    state[n].copy_(source[n])
                got = cases.run(state)
                got = [g.clone() for g in (got if isinstance(got, tuple) else [got])]
            torch.cuda.synchronize()
            assert all(torch.equal(g, w) for g, w in zip(got, want))
            del state, want, got
    finally:
        cases.own = False
        torch.cuda.set_stream(before)
