"""CPU checks of the sequence-cache entry points (sam3b200_rope_*, sam3b200_kv_*): what they refuse, and the oracle
they are compared with."""
import ctypes
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import seq_cache_oracle as sc  # noqa: E402

A = 1 << 20  # an address that no refused call touches


def _cache(b200, **kw):
    c = b200.KVCache(A, A, A, A, 8, 2, 64, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _batch(b200, **kw):
    b = b200.KVBatch(A, 4, A, A, 2, 6, 3, 200)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


BAD_CACHE = [(dict(k_codes=None), "null"), (dict(v_scale=None), "null"), (dict(n_pages=0), "unsupported cache"),
             (dict(n_kv_heads=0), "unsupported cache"), (dict(n_kv_heads=32768), "unsupported cache"), (dict(page_tokens=48), "unsupported cache"),
             (dict(page_tokens=256), "unsupported cache"), (dict(head_dim=96), "unsupported cache"),
             (dict(v_codes=A + 8), "16-byte"), (dict(k_scale=A + 2), "4-byte")]
BAD_BATCH = [(dict(table=None), "null"), (dict(row_start=None), "null"), (dict(kv_len=None), "null"),
             (dict(n_seqs=-1), "bad batch"), (dict(n_rows=-1), "bad batch"), (dict(max_rows=-1), "bad batch"),
             (dict(table_width=0), "bad batch"), (dict(max_len=-1), "bad batch"), (dict(max_len=(1 << 30) + 1), "bad batch"),
             (dict(n_rows=(1 << 27) + 1), "bad batch"), (dict(kv_len=A + 1), "4-byte")]


def _calls(b200):
    L = b200.lib()
    p = ctypes.addressof
    return {"kv_write": lambda c, b: L.sam3b200_kv_write(None, p(c), p(b), b200.TYPE_F16, A, None, A, None),
            "kv_read": lambda c, b: L.sam3b200_kv_read(None, p(c), p(b), b200.TYPE_F16, A, None, A, None),
            "kv_attention": lambda c, b: L.sam3b200_kv_attention_run(None, p(c), p(b), b200.TYPE_F16, A, None, 4, 0.1, 1, 0,
                                                                     b200.TYPE_F16, A, None)}


@pytest.mark.parametrize("op", ["kv_write", "kv_read", "kv_attention"])
def test_caches_and_batches_are_checked(b200, op):
    call = _calls(b200)[op]
    for change, why in BAD_CACHE:
        assert call(_cache(b200, **change), _batch(b200)) == b200.STATUS_FAILED
        assert why in b200.last_error() and op in b200.last_error(), (change, b200.last_error())
    for change, why in BAD_BATCH:
        assert call(_cache(b200), _batch(b200, **change)) == b200.STATUS_FAILED
        assert why in b200.last_error() and op in b200.last_error(), (change, b200.last_error())
    assert call(_cache(b200), _batch(b200)) == b200.STATUS_FAILED  # nothing wrong but the missing backend
    assert "null" in b200.last_error()


def test_rows_are_checked(b200):
    L, c, b = b200.lib(), _cache(b200), _batch(b200)
    c, b = ctypes.addressof(c), ctypes.addressof(b)
    keep = (_cache(b200), _batch(b200))
    c, b = ctypes.addressof(keep[0]), ctypes.addressof(keep[1])
    nb = lambda *x: (ctypes.c_int64 * 2)(*x)
    for fn, op in ((L.sam3b200_kv_write, "kv_write"), (L.sam3b200_kv_read, "kv_read")):
        for args, why in (((b200.TYPE_Q8_0, A, None, A, None), "unsupported type"), ((b200.TYPE_F32, A + 2, None, A, None), "unaligned"),
                          ((b200.TYPE_F16, None, None, A, None), "null"), ((b200.TYPE_F16, A, None, None, None), "null"),
                          ((b200.TYPE_F16, A, nb(-1, 128), A, None), "strides of k"),
                          ((b200.TYPE_F16, A, None, A, nb(256, -1)), "strides of v")):
            assert fn(None, c, b, *args) == b200.STATUS_FAILED
            assert why in b200.last_error() and op in b200.last_error(), (args, b200.last_error())
    # outputs that hold an element twice: rows, or heads, that overlap
    for s in (nb(128, 128), nb(0, 128), nb(256, 64), nb(200, 128)):
        assert L.sam3b200_kv_read(None, c, b, b200.TYPE_F16, A, s, A, None) == b200.STATUS_FAILED
        assert "strides of k" in b200.last_error()
    # heads outside, rows outside, and one row read many times, are fine up to the missing backend
    for s in (nb(128, 1024), nb(256, 128), nb(1024, 256)):
        assert L.sam3b200_kv_read(None, c, b, b200.TYPE_F16, A, s, A, None) == b200.STATUS_FAILED
        assert "null backend" in b200.last_error()
    assert L.sam3b200_kv_write(None, c, b, b200.TYPE_F16, A, nb(0, 0), A, None) == b200.STATUS_FAILED
    assert "null backend" in b200.last_error()


def test_attention_arguments_are_checked(b200):
    L, keep = b200.lib(), (_cache(b200), _batch(b200))
    c, b = ctypes.addressof(keep[0]), ctypes.addressof(keep[1])
    F16, F32, BF16 = b200.TYPE_F16, b200.TYPE_F32, b200.TYPE_BF16
    good = dict(type=F16, q=A, q_nb=None, heads=4, scale=0.1, causal=1, window=0, y_type=F16, y=A, y_nb=None)
    for change, why in ((dict(q=None), "null"), (dict(y=None), "null"), (dict(type=F32), "unsupported types"),
                        (dict(y_type=BF16), "unsupported types"), (dict(q=A + 1), "unaligned"), (dict(y_type=F32, y=A + 2), "unaligned"),
                        (dict(heads=3), "query heads"), (dict(heads=0), "query heads"), (dict(heads=-2), "query heads"),
                        (dict(scale=-1.0), "bad scale"), (dict(scale=float("nan")), "bad scale"), (dict(scale=float("inf")), "bad scale"), (dict(scale=3e38), "bad scale"),
                        (dict(window=-1), "window"), (dict(causal=0, window=5), "window"),
                        (dict(y_nb=(ctypes.c_int64 * 2)(128, 128)), "strides of y"), (dict(q_nb=(ctypes.c_int64 * 2)(-5, 128)), "strides of q"),
                        ({}, "null handle")):
        a = {**good, **change}
        assert L.sam3b200_kv_attention_run(None, c, b, a["type"], a["q"], a["q_nb"], a["heads"], a["scale"], a["causal"],
                                           a["window"], a["y_type"], a["y"], a["y_nb"]) == b200.STATUS_FAILED
        assert why in b200.last_error(), (change, b200.last_error())
    keep[1].n_rows = 1 << 27  # a kv head's rows are counted in 32 bits
    assert L.sam3b200_kv_attention_run(None, c, b, F16, A, None, 2 * 32, 0.1, 1, 0, F16, A, None) == b200.STATUS_FAILED
    assert "too many" in b200.last_error()
    assert not L.sam3b200_kv_attention_create(None)
    L.sam3b200_kv_attention_free(None)
    L.sam3b200_rope_free(None)


def test_rope_arguments_are_checked(b200):
    class NoBackend:  # a handle is a host table; only a launch looks at the backend
        h = ctypes.addressof(ctypes.create_string_buffer(4096))

    for kw in (dict(head_dim=0, sections=[1]), dict(head_dim=258, sections=[4]), dict(head_dim=64, sections=[0, 0]),
               dict(head_dim=64, sections=[20, 13]), dict(head_dim=64, sections=[-1, 8]), dict(head_dim=64, sections=[8], base=0.0),
               dict(head_dim=64, sections=[8], base=float("inf")), dict(head_dim=64, sections=[8], pos_scale=float("nan")),
               dict(head_dim=64, sections=[1] * 5), dict(head_dim=64, sections=[])):
        with pytest.raises(b200.B200Error, match="rope"):
            b200.Rope(NoBackend, **kw)
    with pytest.raises(b200.B200Error):
        b200.Rope(type("X", (), {"h": None}), 64, [8])
    r = b200.Rope(NoBackend, 64, [16, 16])
    F16, F32 = b200.TYPE_F16, b200.TYPE_F32
    good = dict(x=A, x_type=F16, pos=A, n_rows=4, n_heads=2, y=A + 4096, y_type=F16)
    for change, why in ((dict(x=None), "null"), (dict(y=None), "null"), (dict(pos=None), "null"), (dict(x_type=b200.TYPE_Q8_0), "types"),
                        (dict(y_type=b200.TYPE_I32), "types"), (dict(x=A + 1), "unaligned"), (dict(pos=A + 2), "unaligned"),
                        (dict(n_rows=-1), "shape"), (dict(n_heads=-1), "shape"), (dict(n_heads=1 << 20), "shape"),
                        (dict(pos_stride=3), "shape"), (dict(y_nb=(64, 64)), "strides of y"), (dict(x_nb=(-1, 64)), "strides of x"),
                        (dict(y=A, y_type=F32), "in place"), (dict(y=A, y_nb=(256, 64)), "in place")):
        with pytest.raises(b200.B200Error, match=why):
            r.apply(**{**good, **change})
    r.apply(**{**good, "n_rows": 0})  # nothing to do: nothing is touched
    r.apply(**{**good, "n_heads": 0})
    r.free()


def test_oracle_rope_is_a_rotation_by_the_position():
    r = np.random.default_rng(0)
    x, pos = r.normal(size=(5, 2, 24)), r.integers(0, 1000, (2, 5))
    for kw in (dict(), dict(neighbours=True), dict(deal=True), dict(restart=True)):
        y = sc.rope(x, pos, [5, 3], **kw)
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1))
        assert np.array_equal(y[..., 16:], x[..., 16:])
        assert np.allclose(sc.rope(y, pos, [5, 3], inverse=True, **kw), x)
        # scores depend on differences of positions alone
        z = sc.rope(x[:, ::-1], pos, [5, 3], **kw)
        assert np.allclose((y * z).sum(-1), (sc.rope(x, pos * 0 + 7, [5, 3], **kw) * sc.rope(x[:, ::-1], pos * 0 + 7, [5, 3], **kw)).sum(-1))


def test_oracle_attention_against_a_direct_sum():
    r = np.random.default_rng(1)
    cache = sc.empty_cache(3, 2, 16, 64)
    table, rows, lens = np.array([[2, 0]]), [0, 3], [20]
    sc.write(cache, r.normal(size=(20, 2, 64)), r.normal(size=(20, 2, 64)), table, [0, 20], lens)
    q = r.normal(size=(3, 4, 64))
    y = sc.attention(cache, q, table, rows, lens, 0.2, window=4)
    k, v = sc.read(cache, table, [0, 20], lens)
    for i in range(3):
        for h in range(4):
            keys = range(17 + i - 3, 17 + i + 1)
            w = np.array([np.exp(0.2 * q[i, h] @ k[t, h // 2]) for t in keys])
            assert np.allclose(y[i, h], sum(w[j] * v[t, h // 2] for j, t in enumerate(keys)) / w.sum())
