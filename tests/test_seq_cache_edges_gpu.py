"""Edges of the sequence-cache operators on the GPU: values far from 1, rows that see nothing beside them, queries that
are not numbers, windows beyond every length, errors of two
kinds at once, many sequences, results over the queries.

Tolerances are those of test_seq_cache_gpu.py; where a result has no rounding (zeros, NaN) it is asked for as it is.
bf16 queries that the tcgen05 kernel takes as they are (every 8 elements' largest in [2^-4, 2^15]) lose at most half of
f16's smallest step, 2^-25, that is 2^-21 of a row's largest element; scores stay below 64 here, so a weight moves by
less than 2^-12."""
import numpy as np
import pytest

import seq_cache_oracle as sc
from test_seq_cache_gpu import TYPES, Device, attend, check_attention, pages_for, store  # noqa: F401

pytestmark = pytest.mark.gpu


def sized(b200, backend, lens, P, D, H, size, seed=0):
    """A cache whose values are of the given size, keys near 1."""
    rng = np.random.default_rng(seed)
    table, n = pages_for(lens, P, seed=seed)
    host = sc.empty_cache(n, H, P, D, seed)
    rows = np.concatenate([[0], np.cumsum(lens)])
    sc.write(host, rng.normal(size=(rows[-1], H, D)), rng.normal(size=(rows[-1], H, D)) * size, table, rows, lens)
    return Device(b200, backend, host, table)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e30])
@pytest.mark.parametrize("length", [50, 64, 128])
def test_rows_without_keys_beside_large_values(b200, backend, attend, t, D, size, length):
    """Six rows more than tokens: the first six see nothing and are zero whatever the values' size, in both kernels and
    under bounds that cut long key ranges into parts."""
    for G, n in ((4, length + 6), (1, 8)):
        rows = [n, 3]
        lens = [n - 6, 3]
        dev = sized(b200, backend, lens, 16, D, 1, size)
        q = store(np.random.default_rng(1).normal(size=(n + 3, G, D)), t)
        for bound in (None, 100000):
            got = check_attention(dev, attend, q, t, np.concatenate([[0], np.cumsum(rows)]), lens, G, D ** -0.5, t_out="f32", max_len=bound)
            assert np.all(got[:6] == 0)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [4, 48])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_queries_that_are_not_numbers(b200, backend, attend, t, rows, bad):
    """One element of every other row: NaN makes the row NaN however few tokens it sees and wherever they lie, infinities
    what the definition makes of them."""
    dev = sized(b200, backend, [48 + rows], 16, 64, 1, 1.0)
    for codes in (dev.host["k_codes"], dev.host["v_codes"]):  # no zeros: the sums of infinities are the definition's
        codes[codes == 0] = 1
    for n in ("k_codes", "v_codes"):
        dev.buf[n].set(dev.host[n])
    x = np.random.default_rng(2).normal(size=(rows, 1, 64))
    x[::2, 0, 5] = bad
    for window in (1, 2, 4, 20, 0):
        got = check_attention(dev, attend, store(x, t), t, [0, rows], [48 + rows], 1, 0.125, window=window)
        if np.isnan(bad):
            assert np.isnan(got[::2]).all()
        assert not np.isnan(got[1::2]).any()


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("size", [1.0, 1e15, 1e20, 1e35])
@pytest.mark.parametrize("length", [65, 70, 97, 127])
def test_values_of_any_size_beside_unused_places(b200, backend, attend, rows, size, length):
    """Places of a key tile that no token fills weigh nothing, however small the weights 1 / scale of the others are."""
    for D in (64, 128):
        dev = sized(b200, backend, [length], 16, D, 1, size)
        q = store(np.random.default_rng(3).normal(size=(rows, 1, D)), "bf16")
        check_attention(dev, attend, q, "bf16", [0, rows], [length], 1, D ** -0.5, t_out="f32")
        check_attention(dev, attend, q, "bf16", [0, rows], [length], 1, D ** -0.5, t_out="f32", causal=False)


@pytest.mark.parametrize("rows,length", [(6, 3), (9, 2), (80, 20), (300, 290)])
@pytest.mark.parametrize("window", [1 << 30, (1 << 31) - 1, 1 << 31, 1 << 62])
def test_windows_beyond_every_length(b200, backend, attend, rows, length, window):
    """A window that no length reaches is no window, also where the first rows see nothing."""
    dev = sized(b200, backend, [length, 40], 16, 64, 1, 1.0)
    q = store(np.random.default_rng(4).normal(size=(2 * rows, 1, 64)), "f16")
    start, lens = [0, rows, 2 * rows], [length, 40]
    for bound in (None, 5000):
        got = check_attention(dev, attend, q, "f16", start, lens, 1, 0.125, window=window, max_len=bound)
        assert np.array_equal(got, check_attention(dev, attend, q, "f16", start, lens, 1, 0.125, max_len=bound))


def test_errors_of_two_kinds_are_both_named(b200, backend):
    """A wait that ran out and a bad page before one synchronize."""
    dev = Device(b200, backend, sc.empty_cache(2, 1, 16, 64), [[9]])
    rows = backend.upload(np.zeros((4, 1, 64), np.float16))
    batch = dev.batch([0, 4], [4])
    backend.debug_wait_timeout(2_000_000)
    backend.kv_write(dev.cache, batch, TYPES["f16"], rows.ptr, rows.ptr)
    with pytest.raises(b200.B200Error, match="page index") as e:
        backend.synchronize()
    assert "timed out" in str(e.value)
    backend.synchronize()


@pytest.mark.parametrize("seqs", [129, 700])
@pytest.mark.parametrize("new", [1, 40])
def test_more_sequences_than_a_block_has_threads(b200, backend, attend, seqs, new):
    """Sequences are found in several turns; some of them have no rows."""
    rng = np.random.default_rng(seqs + new)
    P, D, H, G = 16, 64, 1, 1
    rows = rng.integers(0, new + 1, seqs)
    rows[-1] = new
    lens = rows + rng.integers(0, 40, seqs)
    table, n = pages_for(lens, P)
    dev = Device(b200, backend, sc.empty_cache(n, H, P, D), table)
    every = np.concatenate([[0], np.cumsum(lens)])
    start = np.concatenate([[0], np.cumsum(rows)])
    k, v = rng.normal(size=(every[-1], H, D)), rng.normal(size=(every[-1], H, D))
    dev.write(k, v, "f16", every, lens)
    dev.same()
    out = [backend.alloc(int(start[-1]) * H * D * 4) for _ in range(2)]
    backend.kv_read(dev.cache, dev.batch(start, lens), TYPES["f32"], out[0].ptr, out[1].ptr)
    backend.synchronize()
    for got, want in zip(out, sc.read(dev.host, table, start, lens)):
        assert np.array_equal(got.get(want.shape, np.float32), want.astype(np.float32))
    q = store(rng.normal(size=(start[-1], H * G, D)), "f16")
    check_attention(dev, attend, q, "f16", start, lens, H * G, 0.125)
    check_attention(dev, attend, q, "f16", start, lens, H * G, 0.125, causal=False)


@pytest.mark.parametrize("rows,length", [(1, 5000), (5, 700), (60, 5000), (300, 300)])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_results_over_the_queries(b200, backend, attend, t, rows, length):
    """y may be q: every block reads its queries before any block of the same rows stores results."""
    dev = sized(b200, backend, [length, 100 + rows], 64, 128, 2, 1.0)
    start, lens = np.array([0, rows, 2 * rows]), [length, 100 + rows]
    q = store(np.random.default_rng(5).normal(size=(2 * rows, 8, 128)), t)
    apart = check_attention(dev, attend, q, t, start, lens, 8, 128 ** -0.5)
    buf = backend.upload(q)
    attend.run(dev.cache, dev.batch(start, lens), TYPES[t], buf.ptr, 8, buf.ptr, 128 ** -0.5)
    backend.synchronize()
    assert np.array_equal(store(apart, t), buf.get(q.shape, q.dtype))


@pytest.mark.parametrize("rows", [1, 48])
@pytest.mark.parametrize("sizes", [(0, 1e7), (1e7, 0), (0, 1e-25), (1e-25, 0), (1e-14, 1e14), (1e14, 1e-14)])
def test_pages_of_far_sizes_side_by_side(b200, backend, attend, rows, sizes):
    """Value scales at the ends of the range that the accuracy is stated for: their weights all stay in the sum."""
    P = 64
    table, n = pages_for([4 * P], P)
    dev = Device(b200, backend, sc.empty_cache(n, 1, P, 64), table)
    rng = np.random.default_rng(6)
    size = np.repeat(np.tile(sizes, 2), P)[:, None, None]
    dev.write(rng.normal(size=(4 * P, 1, 64)), rng.normal(size=(4 * P, 1, 64)) * size, "f32", [0, 4 * P], [4 * P])
    q = store(rng.normal(size=(rows, 1, 64)), "f16")
    check_attention(dev, attend, q, "f16", [0, rows], [4 * P], 1, 0.125, t_out="f32")


@pytest.mark.parametrize("rows", [1, 48])
@pytest.mark.parametrize("size", [1e-25, 1e35])
def test_long_contexts_of_far_sizes(b200, backend, attend, rows, size):
    """The sum of weights over value scales stays in f32 over a long context."""
    dev = sized(b200, backend, [100000], 128, 64, 1, size)
    q = store(np.random.default_rng(7).normal(size=(rows, 1, 64)), "bf16")
    check_attention(dev, attend, q, "bf16", [0, rows], [100000], 1, 0.125, t_out="f32")
