"""CPU checks of the entry points of a decoding step (sam3b200_rope_norm_run, sam3b200_kv4_*, sam3b200_mul_mat_vec): what
they refuse, and the oracle they are compared with."""
import ctypes

import numpy as np
import pytest

import decode_oracle as do
import seq_cache_oracle as sc
from test_seq_cache import BAD_BATCH, BAD_CACHE, _batch

A = 1 << 20  # an address that no refused call touches


class NoBackend:  # a rope handle is a host table; only a launch looks at the backend
    h = ctypes.addressof(ctypes.create_string_buffer(4096))


def _cache(b200, **kw):
    c = b200.KV4Cache(A, A, A, A, 8, 2, 64, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _calls(b200):
    L, p = b200.lib(), ctypes.addressof
    return {"kv4_write": lambda c, b: L.sam3b200_kv4_write(None, p(c), p(b), b200.TYPE_F16, A, None, A, None),
            "kv4_read": lambda c, b: L.sam3b200_kv4_read(None, p(c), p(b), b200.TYPE_F16, A, None, A, None),
            "kv4_attention": lambda c, b: L.sam3b200_kv4_attention_run(None, p(c), p(b), b200.TYPE_F16, A, None, 4, 0.1, 1, 0,
                                                                       b200.TYPE_F16, A, None)}


@pytest.mark.parametrize("op", ["kv4_write", "kv4_read", "kv4_attention"])
def test_caches_and_batches_are_checked(b200, op):
    call = _calls(b200)[op]
    for change, why in BAD_CACHE + [(dict(k_scale=A + 8), "16-byte"), (dict(v_scale=A + 4), "16-byte")]:
        if change == dict(k_scale=A + 2):
            why = "16-byte"
        assert call(_cache(b200, **change), _batch(b200)) == b200.STATUS_FAILED
        assert why in b200.last_error() and op in b200.last_error(), (change, b200.last_error())
    for change, why in BAD_BATCH:
        assert call(_cache(b200), _batch(b200, **change)) == b200.STATUS_FAILED
        assert why in b200.last_error() and op in b200.last_error(), (change, b200.last_error())
    assert call(_cache(b200), _batch(b200)) == b200.STATUS_FAILED  # nothing wrong but the missing backend
    assert "null" in b200.last_error()


def test_the_two_caches_are_told_apart(b200):
    """KVCache and KV4Cache have the same fields: the bindings refuse one in place of the other before the library sees it."""
    four, eight, batch = _cache(b200), b200.KVCache(A, A, A, A, 8, 2, 64, 128), _batch(b200)
    for op, cache in (("kv_write", four), ("kv_read", four), ("kv4_write", eight), ("kv4_read", eight)):
        with pytest.raises(b200.B200Error, match=f"{op}: a {type(cache).__name__} is another cache"):
            getattr(b200.Backend, op)(None, cache, batch, b200.TYPE_F16, A, A)


def test_rows_are_checked(b200):
    L, keep = b200.lib(), (_cache(b200), _batch(b200))
    c, b = ctypes.addressof(keep[0]), ctypes.addressof(keep[1])
    nb = lambda *x: (ctypes.c_int64 * 2)(*x)
    for fn, op in ((L.sam3b200_kv4_write, "kv4_write"), (L.sam3b200_kv4_read, "kv4_read")):
        for args, why in (((b200.TYPE_Q8_0, A, None, A, None), "unsupported type"), ((b200.TYPE_F32, A + 2, None, A, None), "unaligned"),
                          ((b200.TYPE_F16, None, None, A, None), "null"), ((b200.TYPE_F16, A, None, None, None), "null"),
                          ((b200.TYPE_F16, A, nb(-1, 128), A, None), "strides of k"),
                          ((b200.TYPE_F16, A, None, A, nb(256, -1)), "strides of v")):
            assert fn(None, c, b, *args) == b200.STATUS_FAILED
            assert why in b200.last_error() and op in b200.last_error(), (args, b200.last_error())
    for s in (nb(128, 128), nb(0, 128), nb(256, 64), nb(200, 128)):  # outputs that hold an element twice
        assert L.sam3b200_kv4_read(None, c, b, b200.TYPE_F16, A, s, A, None) == b200.STATUS_FAILED
        assert "strides of k" in b200.last_error()
    assert L.sam3b200_kv4_write(None, c, b, b200.TYPE_F16, A, nb(0, 0), A, None) == b200.STATUS_FAILED
    assert "null backend" in b200.last_error()


def test_attention_arguments_are_checked(b200):
    L, keep = b200.lib(), (_cache(b200), _batch(b200))
    c, b = ctypes.addressof(keep[0]), ctypes.addressof(keep[1])
    F16, F32, BF16 = b200.TYPE_F16, b200.TYPE_F32, b200.TYPE_BF16
    good = dict(type=F16, q=A, q_nb=None, heads=4, scale=0.1, causal=1, window=0, y_type=F16, y=A, y_nb=None)
    for change, why in ((dict(q=None), "null"), (dict(y=None), "null"), (dict(type=F32), "unsupported types"),
                        (dict(y_type=BF16), "unsupported types"), (dict(q=A + 1), "unaligned"), (dict(y_type=F32, y=A + 2), "unaligned"),
                        (dict(heads=3), "query heads"), (dict(heads=0), "query heads"), (dict(heads=65536), "query heads"),
                        (dict(scale=-1.0), "bad scale"), (dict(scale=float("nan")), "bad scale"), (dict(scale=3e38), "bad scale"),
                        (dict(window=-1), "window"), (dict(causal=0, window=5), "window"),
                        (dict(y_nb=(ctypes.c_int64 * 2)(128, 128)), "strides of y"), (dict(q_nb=(ctypes.c_int64 * 2)(-5, 128)), "strides of q"),
                        ({}, "null handle")):
        a = {**good, **change}
        assert L.sam3b200_kv4_attention_run(None, c, b, a["type"], a["q"], a["q_nb"], a["heads"], a["scale"], a["causal"],
                                            a["window"], a["y_type"], a["y"], a["y_nb"]) == b200.STATUS_FAILED
        assert why in b200.last_error() and "kv4_attention" in b200.last_error(), (change, b200.last_error())


def test_norm_arguments_are_checked(b200):
    r = b200.Rope(NoBackend, 64, [16, 16])
    F16, F32 = b200.TYPE_F16, b200.TYPE_F32
    H = b200.NormHeads
    good = dict(sets=[H(A, 2, A, A + 4096)], x_type=F16, pos=A, n_rows=4, y_type=F16)
    sets = lambda *a, **kw: dict(sets=[H(*a, **kw)])
    for change, why in ((sets(None, 2, A, A), "null"), (sets(A, 2, A, None), "null"), (dict(pos=None), "null"), (dict(x_type=b200.TYPE_Q8_0), "types"),
                        (dict(y_type=b200.TYPE_I32), "types"), (dict(w_type=b200.TYPE_Q4_0), "types"), (dict(pos=A + 2), "unaligned"),
                        (sets(A + 1, 2, A, A), "unaligned"), (sets(A, 2, A, A + 1), "unaligned"), (sets(A, 2, A + 2, A + 4096), "unaligned"),
                        (sets(A, 2, A, A + 4096, bias=A + 1), "unaligned"), (dict(sets=[]), "sets of heads"), (dict(sets=good["sets"] * 5), "sets of heads"),
                        (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
                        (dict(n_rows=-1), "shape"), (dict(n_rows=(1 << 27) + 1), "shape"), (dict(pos_stride=3), "shape"),
                        (sets(A, -1, A, A), "heads"), (sets(A, 65536, A, A + 4096), "heads"),
                        (sets(A, 2, A, A + 4096, y_nb=(64, 64)), "strides of y"), (sets(A, 2, A, A + 4096, x_nb=(-1, 64)), "strides of x"),
                        (dict(sets=[H(A, 2, A, A)], y_type=F32), "in place"), (sets(A, 2, A, A, y_nb=(256, 64)), "in place")):
        with pytest.raises(b200.B200Error, match=why):
            r.norm(**{**good, **change})
    r.norm(**{**good, "n_rows": 0})  # nothing to do: nothing is touched
    r.norm(**{**good, "sets": [H(None, 0, None, None)]})
    with pytest.raises(b200.B200Error, match="null"):
        r.h, keep = None, r.h
        r.norm(**good)
    r.h = keep
    r.free()


def test_vec_arguments_are_checked(b200):
    """A weight handle made up of zeros has type F32, which is refused after the null checks."""
    L = b200.lib()
    fake = ctypes.addressof(ctypes.create_string_buffer(4096))
    for args in ((None, fake, A, A), (fake, None, A, A), (fake, fake, None, A), (fake, fake, A, None)):
        assert L.sam3b200_mul_mat_vec(args[0], args[1], b200.TYPE_F32, args[2], 64, 1, None, b200.TYPE_F32, args[3], 8) == b200.STATUS_FAILED
        assert "mul_mat_vec: null" in b200.last_error()
    assert L.sam3b200_mul_mat_vec(fake, fake, b200.TYPE_F32, A, 64, 1, None, b200.TYPE_F32, A, 8) == b200.STATUS_FAILED
    assert "unsupported weight type" in b200.last_error()


def test_oracle_quantiser_against_ggml_blocks(oracle):
    """Where bf16 holds the scale exactly, the 4-bit cache's values lie within half a step of the numbers, and the largest
    one is kept."""
    r = np.random.default_rng(0)
    x = np.round(r.normal(size=(50, 4, 64)) * 16) / 16
    codes, bits = do.kv4_quantise(x)
    d = do.bf16_value(bits).repeat(32, -1)
    back = (codes - 8) * d
    y = x.reshape(50, 4, 2, 32)
    top = np.abs(y).max(-1, keepdims=True).repeat(32, -1).reshape(x.shape)
    fits = np.abs(x / np.where(d == 0, 1, d)) < 7.5
    assert np.all(np.abs(back - x)[fits] <= np.abs(d)[fits] / 2 + 1e-12)
    assert np.all(np.abs(back - x) <= np.abs(d) * 1.01)
    assert np.allclose(np.abs(back).reshape(y.shape).max(-1), top.reshape(y.shape)[..., 0], rtol=2.0 ** -8)


def test_oracle_attention_against_a_direct_sum():
    r = np.random.default_rng(1)
    cache = do.kv4_empty(3, 2, 16, 64)
    table, rows, lens = np.array([[2, 0]]), [0, 3], [20]
    do.kv4_write(cache, r.normal(size=(20, 2, 64)), r.normal(size=(20, 2, 64)), table, [0, 20], lens)
    q = r.normal(size=(3, 4, 64))
    y = do.kv4_attention(cache, q, table, rows, lens, 0.2, window=4)
    k, v = do.kv4_read(cache, table, [0, 20], lens)
    for i in range(3):
        for h in range(4):
            keys = range(17 + i - 3, 17 + i + 1)
            w = np.array([np.exp(0.2 * q[i, h] @ k[t, h // 2]) for t in keys])
            assert np.allclose(y[i, h], sum(w[j] * v[t, h // 2] for j, t in enumerate(keys)) / w.sum())


def test_oracle_weights_are_ggmls(oracle):
    """Blocks that ggml's quantiser makes stand for the numbers that its dequantiser gives."""
    r = np.random.default_rng(2)
    for kind, code in (("q4_0", 2), ("q4_1", 3)):
        raw = do.blocks(r, kind, 3, 96)
        got = do.weight(raw, kind, 3, 96)
        for n in range(3):
            for b in range(3):
                p = raw[n * 3 + b]
                d = p[:2].copy().view(np.float16)[0].astype(np.float64)
                m = p[2:4].copy().view(np.float16)[0].astype(np.float64) if kind == "q4_1" else -8 * d
                q = p[2 if kind == "q4_0" else 4:]
                for j in range(16):
                    assert np.isclose(got[n, 32 * b + j], d * (q[j] & 15) + m) and np.isclose(got[n, 32 * b + 16 + j], d * (q[j] >> 4) + m)


def test_oracle_norm():
    r = np.random.default_rng(3)
    x, pos = r.normal(size=(5, 2, 24)) + 1, np.zeros((1, 5))
    y = do.norm(x, None, None, 1e-12, True, pos, [8])
    assert np.allclose(y.mean(-1), 0) and np.allclose((y ** 2).mean(-1), 1)
    y = do.norm(x, np.full(24, 3.0), None, 1e-12, False, pos, [8])
    assert np.allclose((y ** 2).mean(-1), 9)
    assert np.allclose(do.norm(x, None, None, 1e-12, False, pos + 5, [12]), sc.rope(do.normalised(x, None, None, 1e-12, False), pos + 5, [12]))
