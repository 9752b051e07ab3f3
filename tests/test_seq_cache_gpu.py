"""Rotary positions, the paged 8-bit cache and the attention over it (sam3b200_rope_*, sam3b200_kv_*) against the
float64 oracle.

Tolerances.  Codes and scales are equal.  rope: the angle is off by at most 2^-24 turns' worth (2^-23 pi half turns
rounded once, 2^-24 pi) plus two roundings of cosine, sine and the two products, so 2^-21 of the pair's length, plus half
a step of the output's type.  attention: each softmax weight is rounded to f16 (2^-11) in the numerator, queries in
bf16 lose 2^-25 of the row's largest element, scores and sums are f32: 2^-10 of the largest cached magnitude of the
sequence's head covers the weights twice over; half a step of the output's type comes on top."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import seq_cache_oracle as sc  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": 0, "f16": 1, "bf16": 30}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def store(x, t):
    """float array -> the bytes of type t (round to nearest even)."""
    x = np.asarray(x, np.float32)
    if t == "f32":
        return x
    if t == "f16":
        return x.astype(np.float16)
    u = x.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def value(raw, t):
    return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if t == "bf16" else raw.astype(np.float64)


def dtype(t):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[t]


class Device:
    """A cache and its batches on the GPU, next to the oracle's copy."""

    def __init__(self, b200, be, cache, table):
        self.b200, self.be, self.host = b200, be, {k: v.copy() for k, v in cache.items()}
        self.buf = {k: be.upload(v) for k, v in cache.items()}
        pages, heads, P, D = cache["k_codes"].shape
        self.cache = b200.KVCache(*(self.buf[n].ptr for n in ("k_codes", "v_codes", "k_scale", "v_scale")), pages, heads, P, D)
        self.set_table(table)

    def set_table(self, table):
        self.table_host = np.ascontiguousarray(table, np.int32)
        self.table = self.be.upload(self.table_host)

    def batch(self, row_start, kv_len, n_rows=None, max_len=None):
        keep = [self.be.upload(np.asarray(row_start, np.int32)), self.be.upload(np.asarray(kv_len, np.int32))]
        b = self.b200.KVBatch(self.table.ptr, self.table_host.shape[1], keep[0].ptr, keep[1].ptr, len(kv_len),
                              int(row_start[-1]) if n_rows is None else n_rows,
                              int(max(np.diff(row_start), default=0)), int(max(kv_len, default=0)) if max_len is None else max_len)
        b._keep = keep
        return b

    def get(self):
        return {k: self.buf[k].get(v.shape, v.dtype) for k, v in self.host.items()}

    def write(self, k, v, t, row_start, kv_len, oracle=True):
        kb, vb = self.be.upload(store(k, t)), self.be.upload(store(v, t))
        self.be.kv_write(self.cache, self.batch(row_start, kv_len), TYPES[t], kb.ptr, vb.ptr)
        self.be.synchronize()
        if oracle:
            sc.write(self.host, value(store(k, t), t), value(store(v, t), t), self.table_host, row_start, kv_len)

    def same(self):
        got = self.get()
        for n, want in self.host.items():
            assert np.array_equal(got[n], want, equal_nan=want.dtype.kind == "f"), (n, np.argwhere(got[n] != want)[:5])


def pages_for(lens, P, spare=2, seed=0):
    used = [-(-n // P) for n in lens]
    order = np.random.default_rng(seed).permutation(sum(used) + spare)
    table = np.full((len(lens), max(used + [1]) + 1), 1 << 30, np.int32)  # entries that nothing may follow
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    return table, sum(used) + spare


# ---- rope ------------------------------------------------------------------------------------------------------


def run_rope(b200, be, x, pos, sections, t_in, t_out, x_nb=None, y_nb=None, in_place=False, inverse=False, offset=0, pos_stride=None,
             y_size=None, **kw):
    """x: raw array of type t_in holding the rows; returns the raw output buffer."""
    rows, heads, D = kw.pop("shape")
    n = x.size if y_size is None else y_size
    xb = be.upload(np.concatenate([np.zeros(offset, dtype(t_in)), x.reshape(-1)]))
    pb = be.upload(np.ascontiguousarray(pos, np.int32))
    yb = xb if in_place else be.upload(np.full(n + offset, 77, dtype(t_out)))
    r = be.rope(D, sections, **kw)
    at = lambda b, t: b.ptr + offset * np.dtype(dtype(t)).itemsize
    r.apply(at(xb, t_in), TYPES[t_in], pb.ptr, rows, heads, at(yb, t_out), TYPES[t_out], inverse=inverse, x_nb=x_nb, y_nb=y_nb,
            pos_stride=pos_stride)
    be.synchronize()
    r.free()
    return yb.get(n + offset, dtype(t_out))[offset:]


def check_rope(got, want, t_in_value, t_out, sections, neighbours):
    n = sum(sections)
    x = t_in_value
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if neighbours else (x[..., :n], x[..., n:2 * n])
    length = np.hypot(a, b)
    tol = np.zeros(want.shape)
    if neighbours:
        tol[..., 0:2 * n:2] = tol[..., 1:2 * n:2] = length
    else:
        tol[..., :n] = tol[..., n:2 * n] = length
    tol = tol * 2.0 ** -21 + np.abs(want) * HALF_STEP[t_out] * 1.01 + 2.0 ** -25 * (t_out == "f16")
    assert np.all(np.abs(got - want) <= tol), float(np.max(np.abs(got - want) - tol))


@pytest.mark.parametrize("t_in,t_out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("D,sections,kw", [(64, [16, 16], dict(neighbours=True, restart=True)), (128, [24, 20, 20], dict(deal=True, base=5e6)),
                                           (128, [0, 64], dict()), (64, [3, 5, 7, 9], dict(neighbours=True)), (96, [24], dict()),
                                           (20, [3, 4], dict(deal=True)), (256, [128], dict(pos_scale=0.25)), (2, [1], dict())])
def test_rope(b200, backend, t_in, t_out, D, sections, kw):
    rng = np.random.default_rng(D + len(sections))
    for rows, heads in ((1, 1), (7, 3), (130, 5)):
        x = store(rng.normal(size=(rows, heads, D)) * 3, t_in)
        pos = rng.integers(-50, 1 << rng.integers(3, 22), (len(sections), rows))
        want = sc.rope(value(x, t_in), pos, sections, **kw)
        got = value(run_rope(b200, backend, x, pos, sections, t_in, t_out, shape=(rows, heads, D), **kw), t_out).reshape(want.shape)
        check_rope(got, want, value(x, t_in), t_out, sections, kw.get("neighbours", False))


@pytest.mark.parametrize("offset", [0, 1])  # 16-byte aligned rows, and rows that are not
@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_rope_views_in_place_and_back(b200, backend, t, offset):
    """Heads inside a wider row (a fused projection's result), heads outside rows, in place, and the way back."""
    rng = np.random.default_rng(3)
    rows, heads, D, sections = 37, 3, 128, [20, 20, 16]
    wide = store(rng.normal(size=(rows, heads + 2, D)), t)
    pos = rng.integers(0, 5000, (3, rows + 4))
    x = value(wide, t)[:, :heads]
    want = sc.rope(x, pos[:, :rows], sections)
    kw = dict(shape=(rows, heads, D), pos_stride=rows + 4, offset=offset)
    nb = ((heads + 2) * D, D)
    got = run_rope(b200, backend, wide, pos, sections, t, t, x_nb=nb, in_place=True, y_nb=nb, **kw).reshape(wide.shape)
    check_rope(value(got, t)[:, :heads], want, x, t, sections, False)
    assert np.array_equal(got[:, heads:], wide[:, heads:])  # the rest of the rows is left alone
    got2 = run_rope(b200, backend, wide, pos, sections, t, t, x_nb=nb, y_nb=(D, rows * D), y_size=rows * heads * D, **kw)
    assert np.array_equal(got2.reshape(heads, rows, D).transpose(1, 0, 2), got[:, :heads])
    if t == "f32":  # the inverse is the transpose: <R x, z> = <x, R^-1 z>, the gradient
        z = rng.normal(size=(rows, heads, D)).astype(np.float32)
        back = run_rope(b200, backend, z, pos, sections, t, t, inverse=True, **kw).reshape(z.shape)
        check_rope(back, sc.rope(z, pos[:, :rows], sections, inverse=True), z.astype(np.float64), t, sections, False)
        assert abs((got[:, :heads].astype(np.float64) * z).sum() - (x * back).sum()) <= 2.0 ** -20 * np.abs(x).sum() * 4
        # differences of the rotation along a direction give the same gradient
        e, d = 2.0 ** -6, rng.normal(size=x.shape).astype(np.float32)
        up = run_rope(b200, backend, (x + e * d).astype(np.float32), pos, sections, t, t, **kw).reshape(z.shape).astype(np.float64)
        down = run_rope(b200, backend, (x - e * d).astype(np.float32), pos, sections, t, t, **kw).reshape(z.shape).astype(np.float64)
        slope = ((up - down) * z).sum() / (2 * e)
        assert abs(slope - (d.astype(np.float64) * back).sum()) <= 2.0 ** -21 / e * np.abs(z).sum() * 8


# ---- cache -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("P,D,H", [(16, 64, 1), (16, 128, 3), (32, 64, 2), (64, 128, 2), (128, 64, 1), (128, 128, 2)])
def test_write_and_read(b200, backend, t, P, D, H):
    """Ragged runs of tokens appended in several calls with growing and shrinking magnitudes; every code and scale of
    the cache, untouched pages included, equals the oracle's."""
    rng = np.random.default_rng(P + D + H)
    steps = [[0, 5, P, 3], [1, 0, 2 * P + 7, P - 3], [P, 1, 1, 1], [1, 1, 1, 1], [2 * P, 3, 0, P + 1]]
    lens = np.sum(steps, 0)
    table, n = pages_for(lens, P)
    dev = Device(b200, backend, sc.empty_cache(n, H, P, D), table)
    at = np.zeros(4, int)
    for i, new in enumerate(steps):
        at += new
        rows = np.concatenate([[0], np.cumsum(new)])
        k = rng.normal(size=(rows[-1], H, D)) * rng.choice([0.01, 1.0, 30.0], (rows[-1], 1, 1))
        v = rng.normal(size=(rows[-1], H, D)) * 2.0 ** i
        dev.write(k, v, t, rows, at)
        dev.same()
        before = dev.get()
        dev.write(k, v, t, rows, at)  # the same rows again change nothing
        assert all(np.array_equal(before[n], x, equal_nan=x.dtype.kind == "f") for n, x in dev.get().items())
    # read back: everything, and ragged ends, into packed rows and into heads outside rows
    for new in (lens, np.minimum(lens, [0, 1, P + 5, 9])):
        rows = np.concatenate([[0], np.cumsum(new)])
        want_k, want_v = sc.read(dev.host, table, rows, lens)
        N = rows[-1]
        kb, vb = (backend.upload(np.full(N * H * D + 8, 77, dtype(t))) for _ in range(2))
        backend.kv_read(dev.cache, dev.batch(rows, lens), TYPES[t], kb.ptr, vb.ptr, None, (D, N * D))
        backend.synchronize()
        got_k, got_v = kb.get(N * H * D + 8, dtype(t)), vb.get(N * H * D + 8, dtype(t))
        assert np.array_equal(got_k[:-8].reshape(N, H, D), store(want_k.astype(np.float32), t))
        assert np.array_equal(got_v[:-8].reshape(H, N, D).transpose(1, 0, 2), store(want_v.astype(np.float32), t))
        assert np.all(got_k[-8:] == 77) and np.all(got_v[-8:] == 77)


def test_write_rounds_the_exact_quotient(b200, backend):
    """Values on and next to the borders between two codes, NaN, infinities, zeros, subnormal and huge magnitudes."""
    rng = np.random.default_rng(5)
    P, D, H = 32, 128, 2
    for amax in (1.0, 127.0, 0.7300001, 3.1e38, 1e-29, 2.0 ** -100, 2.0 ** -101, 5e-41):
        s = np.float32(amax) / np.float32(127)
        half = (np.arange(P * D) % 253 - 126 + 0.5) * np.float64(s)
        k = half.astype(np.float32).reshape(P, 1, D).repeat(H, 1)
        u = k.view(np.int32)
        u[:, 1] += rng.integers(-2, 3, u[:, 1].shape)  # a few steps to either side
        k = u.view(np.float32).copy()
        k = np.clip(k, -np.float32(amax), np.float32(amax))
        k[0, :, 0] = amax
        v = (rng.normal(size=(P, H, D)) * amax / 4).clip(-amax, amax).astype(np.float32)
        v[3, 0, 5], v[4, 0, 6], v[5, 0, 7] = np.nan, np.inf, -np.inf
        v[:, 1] = [[np.nan]] if amax < 1 else [[np.inf]]
        dev = Device(b200, backend, sc.empty_cache(3, H, P, D), [[1]])
        dev.write(k, v, "f32", [0, P], [P])
        dev.same()


def test_write_from_views_and_broadcast_rows(b200, backend):
    """Keys and values inside one fused projection row, unaligned, and one row for all tokens."""
    rng = np.random.default_rng(6)
    P, D, H, N = 16, 64, 2, 41
    table, n = pages_for([N], P)
    for t, offset in (("bf16", 0), ("bf16", 3), ("f32", 1)):
        wide = store(rng.normal(size=(N * 6 * D + 8)), t)
        buf = backend.upload(wide)
        size = wide.itemsize
        dev = Device(b200, backend, sc.empty_cache(n, H, P, D), table)
        b = dev.batch([0, N], [N])
        backend.kv_write(dev.cache, b, TYPES[t], buf.ptr + offset * size, buf.ptr + (offset + 2 * D) * size, (6 * D, D), (6 * D, 2 * D))
        rows = value(wide, t)[offset:offset + N * 6 * D].reshape(N, 6, D)
        sc.write(dev.host, rows[:, :2], rows[:, 2::2][:, :2], table, [0, N], [N])
        backend.synchronize()
        dev.same()
        backend.kv_write(dev.cache, b, TYPES[t], buf.ptr, buf.ptr, (0, D), (0, 0))
        one = value(wide, t)[:2 * D].reshape(1, 2, D)
        sc.write(dev.host, one.repeat(N, 0), one[:, :1].repeat(N, 0).repeat(2, 1), table, [0, N], [N])
        backend.synchronize()
        dev.same()


def test_bad_tables_and_lengths_are_reported(b200, backend):
    """Entries outside the cache and arrays that contradict the sizes: an error at the next synchronize, nothing
    outside is touched, and the backend goes on."""
    P, D, H = 16, 64, 1
    host = sc.empty_cache(4, H, P, D)
    q = backend.upload(np.zeros((64, 2, D), np.float16))
    y = backend.upload(np.full((72, 2, D), 7, np.float16))
    rows = backend.upload(np.zeros((72, H, D), np.float16))
    att = backend.kv_attention()
    for table, row_start, kv_len, why in (([[9, 1]], [0, 20], [20], "page index"), ([[0, -1]], [0, 20], [20], "page index"),
                                          ([[0, 1]], [0, 20], [200], "contradicts"), ([[0, 1]], [0, 20], [-3], "contradicts"),
                                          ([[0, 1]], [-4, 20], [20], "contradicts"), ([[0, 1]], [0, 400], [20], "contradicts"),
                                          ([[0, 1], [2, 3]], [0, 20, 10], [20, 20], "contradicts")):
        for call in ("write", "read", "attend"):
            dev = Device(b200, backend, host, table)
            b = dev.batch(row_start, kv_len, n_rows=64, max_len=32)
            b.max_rows = 64
            if call == "write":
                backend.kv_write(dev.cache, b, b200.TYPE_F16, rows.ptr, rows.ptr)
            elif call == "read":
                backend.kv_read(dev.cache, b, b200.TYPE_F16, rows.ptr, rows.ptr + 36 * D * 2 * H)
            else:
                att.run(dev.cache, b, b200.TYPE_F16, q.ptr, 2, y.ptr, 0.1)
            with pytest.raises(b200.B200Error, match=why):
                backend.synchronize()
            backend.synchronize()
    assert np.all(y.get((72, 2, D), np.float16)[64:] == 7)
    att.free()


# ---- attention -------------------------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def attend(backend):
    h = backend.kv_attention()
    yield h
    h.free()


def filled(b200, backend, lens, P, D, H, seed=0, k_size=1.0, spread=0.0):
    """A cache with tokens of all sequences, written by the oracle, memory behind them holding anything."""
    rng = np.random.default_rng(seed)
    table, n = pages_for(lens, P, seed=seed)
    host = sc.empty_cache(n, H, P, D, seed)
    rows = np.concatenate([[0], np.cumsum(lens)])
    size = np.exp(spread * rng.normal(size=(rows[-1], 1, 1)))
    k, v = rng.normal(size=(rows[-1], H, D)) * k_size, rng.normal(size=(rows[-1], H, D)) * size
    sc.write(host, k, v, table, rows, lens)
    return Device(b200, backend, host, table)


def check_attention(dev, attend, q_raw, t, row_start, kv_len, n_heads, scale, causal=True, window=0, t_out=None, q_nb=None, y_nb=None,
                    n_rows=None, q=None, max_len=None):
    """Runs the call on packed or strided rows and compares every row of every sequence."""
    be, D = dev.be, dev.host["k_codes"].shape[3]
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
    want = sc.attention(dev.host, q, dev.table_host, row_start, kv_len, scale, causal, window)
    for i, length in enumerate(kv_len):
        r = slice(row_start[i], row_start[i + 1])
        v = np.abs(sc.tokens(dev.host, "v", dev.table_host[i], 0, length)).max((0, 2), initial=0.0)
        tol = 2.0 ** -10 * np.repeat(v, n_heads // len(v))[None, :, None] + np.abs(want[r]) * HALF_STEP[t_out] * 1.01
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


GROUPS = [(1, 1), (4, 1), (2, 8), (1, 16), (3, 5)]  # kv heads, query heads of each


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("P,D", [(16, 64), (16, 128), (32, 128), (64, 64), (64, 128), (128, 128)])
@pytest.mark.parametrize("H,G", GROUPS)
def test_attention_single_tokens(b200, backend, attend, t, P, D, H, G):
    rng = np.random.default_rng(P + D + H + G)
    lens = [1, 15, 16, 17, P, P + 1, 333, 700]
    dev = filled(b200, backend, lens, P, D, H)
    q = store(rng.normal(size=(len(lens), H * G, D)) * 2, t)
    check_attention(dev, attend, q, t, np.arange(len(lens) + 1), lens, H * G, D ** -0.5)
    check_attention(dev, attend, q, t, np.arange(len(lens) + 1), lens, H * G, D ** -0.5, window=40, t_out="f32")


@pytest.mark.parametrize("t,t_out", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("P,D", [(16, 64), (32, 128), (128, 64)])
@pytest.mark.parametrize("H,G", GROUPS)
def test_attention_several_rows(b200, backend, attend, t, t_out, P, D, H, G):
    """Drafted tokens, parts of prompts and whole prompts in one ragged batch, sequences without rows or tokens
    among them; causal, windowed and full."""
    rng = np.random.default_rng(P + D + H + G)
    rows, lens = [3, 0, 130, 7, 1, 40, 2], [90, 50, 130, 300, 1, 515, 0]
    start = np.concatenate([[0], np.cumsum(rows)])
    dev = filled(b200, backend, lens, P, D, H)
    q = store(rng.normal(size=(start[-1], H * G, D)) * 2, t)
    for kw in (dict(), dict(window=1), dict(window=37), dict(causal=False)):
        check_attention(dev, attend, q, t, start, lens, H * G, D ** -0.5, t_out=t_out, **kw)


@pytest.mark.parametrize("rows", [1, 4, 70, 300])
def test_attention_rows_without_keys_are_zero(b200, backend, attend, rows):
    """More rows than tokens: the first rows see nothing; an empty cache: none does."""
    dev = filled(b200, backend, [min(rows, 3) - 1, 0, 20], 16, 128, 2)
    lens = [min(rows, 3) - 1, 0, 20]
    q = store(np.random.default_rng(0).normal(size=(3 * rows, 4, 128)), "f16")
    got = check_attention(dev, attend, q, "f16", np.arange(4) * rows, lens, 4, 0.1)
    assert np.all(got[:rows - lens[0]] == 0) and np.all(got[rows:2 * rows] == 0)
    got = check_attention(dev, attend, q, "f16", np.arange(4) * rows, lens, 4, 0.1, causal=False)
    assert np.all(got[rows:2 * rows] == 0)


@pytest.mark.parametrize("rows", [1, 200])
def test_attention_long_contexts_in_parts(b200, backend, attend, rows):
    """Key ranges that are cut into parts, of lengths around the cuts; a length far below max_len."""
    lens = [20000, 4096, 4097, 63, 12345]
    dev = filled(b200, backend, lens, 64, 128, 1)
    start = np.arange(6) * rows
    q = store(np.random.default_rng(1).normal(size=(5 * rows, 4, 128)) * 3, "bf16")
    check_attention(dev, attend, q, "bf16", start, lens, 4, 128 ** -0.5)
    check_attention(dev, attend, q, "bf16", start, lens, 4, 128 ** -0.5, window=5000)
    # a bound far above every length, as a captured step has it, and one sequence alone under it
    for bound in (100000, 1 << 30):
        check_attention(dev, attend, q, "bf16", start, lens, 4, 128 ** -0.5, max_len=bound)
        check_attention(dev, attend, q[:rows], "bf16", start[:2], lens[:1], 4, 128 ** -0.5, max_len=bound)


@pytest.mark.parametrize("rows", [2, 150])
def test_attention_views_and_rows_outside_sequences(b200, backend, attend, rows):
    """Queries inside a fused projection's rows, outputs with heads outside, unaligned data; rows in front of the first
    and behind the last sequence are left as they were."""
    rng = np.random.default_rng(2)
    D, H, G, lens = 64, 2, 3, [300, rows, 77 + rows]
    dev = filled(b200, backend, lens, 32, D, H)
    start = 5 + np.arange(4) * rows
    N = start[-1] + 9
    wide = store(rng.normal(size=(N, 10, D)), "f16")
    q = value(wide, "f16")[:, :6]
    check_attention(dev, attend, wide, "f16", start, lens, 6, 0.2, q_nb=(10 * D, D), y_nb=(D, N * D), n_rows=N, q=q)
    odd = store(rng.normal(size=(N, 6 * D + 3)), "f16")
    q = value(odd, "f16")[:, :6 * D].reshape(N, 6, D)
    check_attention(dev, attend, odd, "f16", start, lens, 6, 0.2, q_nb=(6 * D + 3, D), y_nb=(6 * D + 1, D), n_rows=N, q=q)
    one = store(rng.normal(size=(1, D)), "f16")  # one query for all rows and heads
    q = np.broadcast_to(value(one, "f16"), (N, 6, D))
    check_attention(dev, attend, one, "f16", start, lens, 6, 0.2, q_nb=(0, 0), n_rows=N, q=q)


@pytest.mark.parametrize("rows", [1, 140])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_attention_extreme_values(b200, backend, attend, t, rows):
    """Pages of very different scales, pages of zeros, scores far apart, a NaN in one query, queries of huge and tiny
    size, a zero scale."""
    rng = np.random.default_rng(3)
    lens = [400 + rows, 64 + rows]
    dev = filled(b200, backend, lens, 16, 128, 1, spread=4.0)
    N = 2 * rows
    start = [0, rows, N]
    zero = dev.table_host[0][2]
    for n in ("k", "v"):
        dev.host[n + "_codes"][zero] = 0
        dev.host[n + "_scale"][zero] = 0
        dev.buf[n + "_codes"].set(dev.host[n + "_codes"])
        dev.buf[n + "_scale"].set(dev.host[n + "_scale"])
    x = rng.normal(size=(N, 2, 128))
    check_attention(dev, attend, store(x * 30, t), t, start, lens, 2, 0.3)
    check_attention(dev, attend, store(x, t), t, start, lens, 2, 0.0)
    x[0, 1, 7] = np.nan
    got = check_attention(dev, attend, store(x, t), t, start, lens, 2, 0.1)
    assert np.isnan(got[0, 1]).all() and not np.isnan(got[0, 0]).any()
    if t == "bf16":
        x = rng.normal(size=(N, 2, 128))
        check_attention(dev, attend, store(x * 1e30, t), t, start, lens, 2, 1e-30)
        check_attention(dev, attend, store(x * 1e-30, t), t, start, lens, 2, 1e30)


@pytest.mark.parametrize("rows", [1, 50])
def test_sequences_share_full_pages(b200, backend, attend, rows):
    """A common prompt's full pages stand in the tables of several sequences; each goes on in pages of its own."""
    P, D, H = 32, 64, 2
    table = np.array([[5, 2, 7, 0], [5, 2, 1, 3], [5, 2, 6, 4]])
    lens = [2 * P + rows, 2 * P + rows + 3, 2 * P + 40]
    dev = Device(b200, backend, sc.empty_cache(8, H, P, D), table)
    rng = np.random.default_rng(9)
    k, v = rng.normal(size=(2 * P, H, D)), rng.normal(size=(2 * P, H, D))
    dev.write(k, v, "f16", [0, 2 * P, 2 * P, 2 * P], [2 * P] * 3)  # the first sequence's rows; the others have none
    new = np.array(lens) - 2 * P
    start = np.concatenate([[0], np.cumsum(new)])
    dev.write(rng.normal(size=(start[-1], H, D)), rng.normal(size=(start[-1], H, D)), "f16", start, lens)
    dev.same()
    q = store(rng.normal(size=(3 * rows, 4, D)), "f16")
    check_attention(dev, attend, q, "f16", np.arange(4) * rows, lens, 4, 0.125)


def test_pages_behind_four_gigabytes(b200, backend, attend):
    """Codes whose offsets pass 32 bits: written, read and attended to as in a small cache, bit for bit."""
    P, D, H, lens = 128, 128, 8, [300, 1000]
    small_table, n = pages_for(lens, P)
    far = 33000  # pages of 128 KiB
    far_table = np.where(small_table < n, small_table + far, small_table).astype(np.int32)
    rng = np.random.default_rng(10)
    start = np.concatenate([[0], np.cumsum(lens)])
    k, v = (backend.upload(store(rng.normal(size=(start[-1], H, D)), "bf16")) for _ in range(2))
    q = {r: backend.upload(store(rng.normal(size=(2 * r, 16, D)), "bf16")) for r in (1, 40)}
    results = []
    for pages, table in ((n, small_table), (n + far, far_table)):
        codes, scales = [backend.alloc(pages * H * P * D) for _ in range(2)], [backend.alloc(pages * H * 4) for _ in range(2)]
        cache = b200.KVCache(codes[0].ptr, codes[1].ptr, scales[0].ptr, scales[1].ptr, pages, H, P, D)
        keep = [backend.upload(np.ascontiguousarray(x, np.int32)) for x in (table, start, lens)]
        batch = b200.KVBatch(keep[0].ptr, table.shape[1], keep[1].ptr, keep[2].ptr, 2, int(start[-1]), max(lens), max(lens))
        backend.kv_write(cache, batch, TYPES["bf16"], k.ptr, v.ptr)
        out = [backend.alloc(int(start[-1]) * H * D * 4) for _ in range(2)]
        backend.kv_read(cache, batch, TYPES["f32"], out[0].ptr, out[1].ptr)
        got = [o.get((start[-1], H, D), np.float32) for o in out]
        for r in q:
            at = backend.upload(np.array([0, r, 2 * r], np.int32))
            y = backend.alloc(2 * r * 16 * D * 2)
            b = b200.KVBatch(keep[0].ptr, table.shape[1], at.ptr, keep[2].ptr, 2, 2 * r, r, max(lens))
            attend.run(cache, b, TYPES["bf16"], q[r].ptr, 16, y.ptr, 0.09)
            backend.synchronize()
            got.append(y.get((2 * r, 16, D), np.uint16))
        backend.synchronize()
        results.append(got)
        for x in codes + scales:
            x.free()
    assert all(np.array_equal(a, b) for a, b in zip(*results))
    assert np.abs(results[0][0]).max() > 1


def test_results_repeat_bit_for_bit(b200, backend, attend):
    lens = [9000, 100, 5000]
    dev = filled(b200, backend, lens, 32, 128, 2)
    for rows in (1, 33):
        q = store(np.random.default_rng(4).normal(size=(3 * rows, 8, 128)), "f16")
        runs = [check_attention(dev, attend, q, "f16", np.arange(4) * rows, lens, 8, 0.1) for _ in range(3)]
        assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])


# ---- together --------------------------------------------------------------------------------------------------


def test_a_prompt_and_steps_of_generation(b200, backend, attend):
    """As a decoder layer uses them: fused projection rows, queries and keys turned by three-axis positions, keys and
    values into the cache, attention -- for a ragged prompt, then single tokens; against the oracle's own cache."""
    rng = np.random.default_rng(7)
    H, G, D, P, t = 2, 4, 128, 16, "bf16"
    width = H * G + 2 * H
    lens = np.zeros(3, int)
    total = np.array([60, 21, 33]) + 5
    table, n = pages_for(total, P)
    dev = Device(b200, backend, sc.empty_cache(n, H, P, D), table)
    rope = backend.rope(D, [24, 20, 20], deal=True, base=1e6)
    for new in [[60, 21, 33]] + [[1, 1, 1]] * 5:
        start = np.concatenate([[0], np.cumsum(new)])
        N = start[-1]
        proj = store(rng.normal(size=(N, width, D)), t)
        pos = np.concatenate([np.arange(l, l + m) for l, m in zip(lens, new)]) + rng.integers(0, 9, (3, 1))
        lens = lens + new
        pb, xb = backend.upload(pos.astype(np.int32)), backend.upload(proj)
        row = width * D
        rope.apply(xb.ptr, TYPES[t], pb.ptr, N, H * G + H, xb.ptr, TYPES[t], x_nb=(row, D), y_nb=(row, D))
        b = dev.batch(start, lens)
        at = lambda head: xb.ptr + head * D * 2
        yb = backend.alloc(N * H * G * D * 4)
        backend.kv_write(dev.cache, b, TYPES[t], at(H * G), at(H * G + H), (row, D), (row, D))
        attend.run(dev.cache, b, TYPES[t], at(0), H * G, yb.ptr, D ** -0.5, y_type=b200.TYPE_F32, q_nb=(row, D))
        backend.synchronize()
        turned = value(xb.get(proj.shape, np.uint16), t)
        x = value(proj, t)
        check_rope(turned[:, :H * G + H], sc.rope(x[:, :H * G + H], pos, [24, 20, 20], deal=True, base=1e6), x[:, :H * G + H], t, [24, 20, 20], False)
        sc.write(dev.host, turned[:, H * G:H * G + H], turned[:, H * G + H:], table, start, lens)
        dev.same()
        want = sc.attention(dev.host, turned[:, :H * G], table, start, lens, D ** -0.5)
        assert np.max(np.abs(yb.get(want.shape, np.float32) - want)) <= 2.0 ** -10 * np.abs(sc.tokens(dev.host, "v", table[0], 0, lens[0])).max() * 2
    rope.free()


def test_a_captured_step_replays_with_new_lengths(b200, backend):
    """One step (rotation, write, attention) captured from the backend's stream; replays read the new lengths, rows and
    pages from device memory and match direct calls bit for bit."""
    import torch
    rng = np.random.default_rng(8)
    H, G, D, P, S = 2, 2, 64, 16, 3
    table, n = pages_for([120] * S, P)
    host = sc.empty_cache(n, H, P, D)
    lens = np.array([31, 32, 95])
    first = np.concatenate([[0], np.cumsum(lens)])
    sc.write(host, rng.normal(size=(first[-1], H, D)), rng.normal(size=(first[-1], H, D)), table, first, lens)
    dev, twin = Device(b200, backend, host, table), Device(b200, backend, host, table)
    own, other = backend.kv_attention(), backend.kv_attention()
    rope = backend.rope(D, [32])
    rows = [np.arange(S + 1)]
    x, pos = backend.alloc(S * 8 * D * 2), backend.alloc(S * 4)
    y, y2 = backend.alloc(S * 4 * D * 2), backend.alloc(S * 4 * D * 2)
    t = b200.TYPE_F16

    def step(d, handle, batch, xp, yp):
        rope.apply(xp, t, pos.ptr, S, 6, xp, t, x_nb=(8 * D, D), y_nb=(8 * D, D))
        d.be.kv_write(d.cache, batch, t, xp + 4 * D * 2, xp + 6 * D * 2, (8 * D, D), (8 * D, D))
        handle.run(d.cache, batch, t, xp, 4, yp, 0.125, q_nb=(8 * D, D))

    batch = dev.batch(rows[0], lens, max_len=120)
    stream = torch.cuda.ExternalStream(backend.stream)
    graph = torch.cuda.CUDAGraph()
    x.set(np.zeros(S * 8 * D, np.float16))
    pos.set(np.zeros(S, np.int32))
    with torch.cuda.graph(graph, stream=stream):
        step(dev, own, batch, x.ptr, y.ptr)
    for i in range(20):
        lens = lens + 1
        rowsx = store(rng.normal(size=(S, 8, D)), "f16")
        batch._keep[1].set(lens.astype(np.int32))
        x.set(rowsx)
        pos.set((lens - 1).astype(np.int32))
        with torch.cuda.stream(stream):
            graph.replay()
        backend.synchronize()
        got = y.get((S, 4, D), np.float16)
        x.set(rowsx)
        step(twin, other, twin.batch(rows[0], lens, max_len=120), x.ptr, y2.ptr)
        backend.synchronize()
        assert np.array_equal(got, y2.get((S, 4, D), np.float16))
        a, b = dev.get(), twin.get()
        assert all(np.array_equal(a[k], b[k], equal_nan=a[k].dtype.kind == "f") for k in a)
    del graph
    for h in (own, other, rope):
        h.free()


@pytest.mark.parametrize("captured", [False, True])
def test_calls_wait_for_another_stream_and_are_waited_for(b200, backend, attend, captured):
    """Every call of a chain follows a kernel of its own stream and, by an event, slow work of another stream that makes
    its input; and the other stream's work over the results follows the chain.  Any call that started early, or any work
    that did not see a call's results, gives other numbers."""
    import torch
    rng = np.random.default_rng(9)
    H, G, D, P, S, L = 2, 2, 64, 16, 2, 200
    width, t = H * G + 2 * H, b200.TYPE_F16
    table, n = pages_for([L] * S, P)
    dev = Device(b200, backend, sc.empty_cache(n, H, P, D), table)
    rope = backend.rope(D, [32])
    src = torch.from_numpy(rng.normal(size=(S * L, width, D)).astype(np.float16)).cuda()
    pos = torch.arange(L, dtype=torch.int32, device="cuda").repeat(S)
    x, out = torch.zeros_like(src), torch.zeros((S * L, H * G, D), dtype=torch.float16, device="cuda")
    kept = torch.zeros((4, *out.shape), dtype=torch.float16, device="cuda")
    slow, pad = torch.zeros(1 << 26, device="cuda"), torch.zeros(D, dtype=torch.float16, device="cuda")
    batch = dev.batch([0, L, 2 * L], [L, L])
    own, side = torch.cuda.ExternalStream(backend.stream), torch.cuda.Stream()
    at = lambda head: x.data_ptr() + head * D * 2
    nb = (width * D, D)
    torch.cuda.synchronize()

    def work():
        for i in range(4):
            side.wait_stream(own)  # the side stream keeps the last results, then makes the next input, slowly
            with torch.cuda.stream(side):
                if i:
                    kept[i - 1].copy_(out)
                slow.add_(1.0)
                x.copy_(src).mul_(1.0 + i)
            if i % 2 == 0:
                rope.apply(pad.data_ptr(), t, pos.data_ptr(), 1, 1, pad.data_ptr(), t)  # a kernel in front, of no matter
            own.wait_stream(side)
            rope.apply(at(0), t, pos.data_ptr(), S * L, H * G + H, at(0), t, x_nb=nb, y_nb=nb)
            backend.kv_write(dev.cache, batch, t, at(H * G), at(H * G + H), nb, nb)
            attend.run(dev.cache, batch, t, at(0), H * G, out.data_ptr(), 0.125, q_nb=nb)
        side.wait_stream(own)
        with torch.cuda.stream(side):
            kept[3].copy_(out)
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
    # the values' scale is proportional to the input: outputs of step i are those of its own input, computed alone
    for i in range(4):
        x.copy_(src).mul_(1.0 + i)
        torch.cuda.synchronize()
        rope.apply(at(0), t, pos.data_ptr(), S * L, H * G + H, at(0), t, x_nb=nb, y_nb=nb)
        backend.synchronize()
        backend.kv_write(dev.cache, batch, t, at(H * G), at(H * G + H), nb, nb)
        backend.synchronize()
        attend.run(dev.cache, batch, t, at(0), H * G, out.data_ptr(), 0.125, q_nb=nb)
        backend.synchronize()
        assert np.array_equal(got[i], out.cpu().numpy())
    assert not np.array_equal(got[0], got[1])
    if captured:
        del graph
    rope.free()
