"""Refusals of the device operators (CPU: no call gets as far as a device) and
the host side of the rotary positions."""
import ctypes
import math

import numpy as np
import pytest

import codon_hip as ch
from codon_hip import _lib as C


class Fake:
    """An array that only looks like one: calls on it have to be refused."""

    def __init__(self, shape, dtype="float32", stride=None, at=1 << 20):
        self.shape, self.dtype, self._at = tuple(shape), dtype, at
        st, n = [], 1
        for d in reversed(self.shape):
            st.append(n)
            n *= d
        self._stride = stride or tuple(reversed(st))

    def data_ptr(self):
        return self._at

    def stride(self):
        return self._stride


def cache(pages=4, heads=2, d=64, **kw):
    dp = ch.Kv8Cache.dims(d)
    f = dict(k=Fake((pages, heads, 64, dp), "int8"), v=Fake((pages, heads, dp, 64), "int8"),
             scales=Fake((pages, heads, 2)), bad=Fake((pages, heads), "int64"))
    f.update(kw)
    return ch.Kv8Cache(f["k"], f["v"], f["scales"], f["bad"], d)


def batch(n_rows=3, max_rows=3, n_seq=2, **kw):
    f = dict(cu=Fake((n_seq + 1,), "int32"), lens=Fake((n_seq,), "int32"), table=Fake((n_seq, 5), "int32"), slots=None)
    f.update(kw)
    return ch.Kv8Batch(f["cu"], f["lens"], f["table"], n_rows, max_rows, f["slots"])


def code(fn, *a, **kw):
    with pytest.raises(ch.CihError) as e:
        fn(*a, **kw)
    return e.value.code


def test_cache_and_batch_refuse_other_arrays():
    for bad in (dict(k=Fake((4, 2, 64, 64), "uint8")), dict(v=Fake((4, 2, 64, 32), "int8")), dict(scales=Fake((4, 2))),
                dict(bad=Fake((4, 2), "int32")), dict(k=Fake((4, 2, 32, 64), "int8")),
                dict(k=Fake((4, 2, 64, 64), "int8", stride=(8192, 64, 128, 1)))):
        with pytest.raises((TypeError, ValueError)):
            cache(**bad)
    for bad in (dict(cu=Fake((2,), "int32")), dict(lens=Fake((2,), "int64")), dict(table=Fake((10,), "int32")),
                dict(table=Fake((2, 5), "int64")), dict(table=Fake((2, 5), "int32", stride=(1, 2))),
                dict(slots=Fake((3,), "int32"))):
        with pytest.raises((TypeError, ValueError)):
            batch(**bad)


def test_append_refusals():
    c, b = cache(), batch()
    row = lambda h=2, t="float32", **kw: Fake((3, h, 64), t, **kw)  # noqa: E731
    for a, kw in (((row(3), row()), {}), ((row(), row(t="float16")), {}), ((row(t="int8"), row()), {}),
                  ((row(), row()), dict(q=row(4), q_out=row(2))), ((row(), row()), dict(q=row(4, "float16"))),
                  ((row(stride=(128, 64, 2)), row()), {})):
        with pytest.raises((TypeError, ValueError)):
            c.append(b, *a, **kw)
    assert code(c.append, b, row(at=2), row()) == -1                     # unaligned
    assert code(c.append, b, row(at=0), row()) == -1                     # null
    assert code(c.append, b, row(), row(), q=row(3)) == -2               # heads that do not divide
    assert code(c.append, b, row(), row(), q=row(4), q_out=row(4, stride=(64, 64, 1))) == -2  # rows on each other
    assert code(c.append, b, row(), row(), q=row(4, stride=(512, 64, 1)), q_out=row(4)) == -1  # in place, other strides
    assert code(c.append, b, row(stride=(-128, 64, 1)), row()) == -2
    assert code(c.append, b, row(), row(), rope=ch.Rope(128)) == -2      # more rotary dims than the head has
    assert code(cache(k=Fake((4, 2, 64, 64), "int8", at=1 << 20 | 8)).append, b, row(), row()) == -1
    assert code(c.read, b, row(stride=(64, 64, 1)), row()) == -2
    assert code(cache(d=64, scales=Fake((4, 2, 2), at=4)).append, b, row(), row()) == -1
    assert code(batch_append, batch(table=Fake((1, 5), "int32"))) == -2  # fewer table rows than sequences
    assert code(batch_append, batch(max_rows=-1)) == -1
    assert code(batch_append, batch(table=Fake((2, 0), "int32"))) == -2
    with pytest.raises(ch.CihError):
        cache(d=48).append(b, Fake((3, 2, 48)), Fake((3, 2, 48)))
    # nothing to do: nothing is looked at
    c.append(batch(n_rows=0, max_rows=0), Fake((0, 2, 64), at=0), Fake((0, 2, 64), at=0))


def batch_append(b):
    cache().append(b, Fake((3, 2, 64)), Fake((3, 2, 64)))


def test_attention_refusals():
    c, b = cache(), batch()
    q = lambda h=4, t="float32", **kw: Fake((3, h, 64), t, **kw)  # noqa: E731
    ws = Fake((1 << 20,), "uint8")
    for a, kw in (((q(), q(2)), {}), ((q(), q(t="float16")), {}), ((q(), q()), dict(lse=Fake((3, 2)))),
                  ((q(), q()), dict(lse=Fake((3, 4), "float16"))), ((q(), q()), dict(workspace=Fake((8,), "float32")))):
        with pytest.raises((TypeError, ValueError)):
            c.attend(b, *a, **kw)
    assert code(c.attend, b, q(3), q(3), workspace=ws) == -2
    assert code(c.attend, b, q(), q(), window=-1, workspace=ws) == -1
    assert code(c.attend, b, q(), q(), scale=math.nan, workspace=ws) == -1
    assert code(c.attend, b, q(), q(at=1), workspace=ws) == -1
    assert code(c.attend, b, q(), q(stride=(64, 64, 1)), workspace=ws) == -2
    assert code(c.attend, b, q(), q(), lse=Fake((3, 4), at=2), workspace=ws) == -1
    long = batch(n_rows=1, max_rows=1, n_seq=1, table=Fake((1, 5000), "int32"))
    need = c.attend_workspace(long, 4)
    if need:
        one = Fake((1, 4, 64))
        assert code(c.attend, long, one, one, workspace=Fake((need - 1,), "uint8")) == -3
        assert code(c.attend, long, one, one) == -3
        assert code(c.attend, long, one, one, workspace=Fake((need,), "uint8", at=8)) == -3
    many = batch(n_rows=1 << 30, max_rows=1 << 30)  # 2^31 rows of a key/value head
    assert code(c.attend_workspace, many, 4) == -2
    assert code(c.attend, b, q(at=1 << 20), q(at=1 << 20, stride=(512, 64, 1)), workspace=ws) == -1  # in place, other strides
    lib = C.lib()
    assert lib.cih_kv8_attention(None, b._at, 0, 4, None, None, None, 1.0, 1, 0, None, 0, None) == -1
    assert lib.cih_kv8_attention(c._at, b._at, 7, 4, None, None, None, 1.0, 1, 0, None, 0, None) == -1
    assert lib.cih_kv8_attention(c._at, b._at, 0, 4, None, None, None, 1.0, 1, 0, None, 1 << 30, None) in (-1, -3)
    assert lib.cih_kv8_attention_workspace(c._at, b._at, 4, None) == -1


def test_logprobs_refusals():
    x, t, f = Fake((3, 100)), Fake((3,), "int32"), Fake((3,))
    ws = Fake((1 << 20,), "uint8")
    with pytest.raises(ValueError):
        ch.token_logprobs(x, None, f)
    with pytest.raises(ValueError):
        ch.token_logprobs(x, top_ids=Fake((3, 2), "int32"))
    with pytest.raises(ValueError):
        ch.token_logprobs(Fake((3, 100), stride=(1, 3)), t, f)
    with pytest.raises((TypeError, ValueError)):
        ch.token_logprobs(x, Fake((3,), "int64"), f)
    with pytest.raises((TypeError, ValueError)):
        ch.token_logprobs(x, t, Fake((4,)))
    with pytest.raises(TypeError):
        ch.token_logprobs(Fake((3, 100), "int32"), t, f)
    assert code(ch.token_logprobs, x, t, f, top_ids=Fake((3, 65), "int32"), top_logprobs=Fake((3, 65)), workspace=ws) == -2
    assert code(ch.token_logprobs, Fake((3, 100), stride=(99, 1)), t, f, workspace=ws) == -2
    assert code(ch.token_logprobs, Fake((3, 100), at=2), t, f, workspace=ws) == -1
    assert code(ch.token_logprobs, Fake((3, 100), at=0), t, f, workspace=ws) == -1
    assert code(ch.token_logprobs_workspace, 3, 0, 1) == -2
    assert code(ch.token_logprobs_workspace, -1, 10, 1) == -2
    assert code(ch.token_logprobs_workspace, (1 << 30) + 1, 10, 1) == -2
    need = ch.token_logprobs_workspace(1, 131072, 20)
    if need:
        assert code(ch.token_logprobs, Fake((1, 131072)), Fake((1,), "int32"), Fake((1,)), top_ids=Fake((1, 20), "int32"),
                    top_logprobs=Fake((1, 20)), workspace=Fake((need - 1,), "uint8")) == -3
    ch.token_logprobs(Fake((0, 100), at=0), Fake((0,), "int32", at=0), Fake((0,), at=0))


def test_rope_frequencies():
    """Each scaling's frequencies and gain from its formula."""
    base = [10000.0 ** (-2 * j / 32) for j in range(16)]
    assert np.allclose(ch.Rope(32).freq, base, rtol=1e-15) and ch.Rope(32).gain == 1
    assert np.allclose(ch.Rope(32, scaling="linear", factor=4).freq, np.array(base) / 4, rtol=1e-15)
    assert np.allclose(ch.Rope(32, scaling="ntk", factor=4).freq,
                       [(10000.0 * 4 ** (32 / 30)) ** (-2 * j / 32) for j in range(16)], rtol=1e-14)
    r = ch.Rope(32, scaling="yarn", factor=4, trained_len=2048)
    turns = 2048 * np.array(base) / (2 * math.pi)
    assert turns.max() > 32 and turns.min() < 1  # both ends and what is between
    g = np.clip((turns - 1) / 31, 0, 1)
    assert np.allclose(r.freq, np.array(base) * ((1 - g) / 4 + g), rtol=1e-14)
    assert r.gain == np.float32(0.1 * math.log(4) + 1)
    assert ch.Rope(32, scaling="yarn", factor=1).gain == 1


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=130), dict(base=0.0), dict(base=math.inf),
                                dict(scaling="linear", factor=0.5), dict(scaling="ntk", rot_dim=2, factor=2.0),
                                dict(scaling="yarn", factor=math.nan), dict(scaling="yarn", factor=2.0, trained_len=0)])
def test_rope_refusals(kw):
    args = dict(rot_dim=32)
    args.update(kw)
    with pytest.raises(ch.CihError):
        ch.Rope(**args)
    r = C.RopeStruct()
    assert C.lib().cih_rope_init(None, 32, 0, 1e4, 0, 1.0, 1) == -1
    assert C.lib().cih_rope_init(ctypes.addressof(r), 32, 0, 1e4, 9, 1.0, 1) == -1
    with pytest.raises(ValueError):
        ch.Rope(32, scaling="other")


def test_decoder_refusals_without_a_model():
    lib, out, r = C.lib(), ctypes.c_void_p(), C.RopeStruct()
    assert lib.cih_decoder_create_kv8(None, 1, 64, 8, 0, None, ctypes.byref(out)) == -1
    assert lib.cih_decoder_create_kv8(None, 1, 64, 8, 0, ctypes.addressof(r), None) == -1
    assert lib.cih_decoder_score(None, 1, None, None, None, 0, None, None, None, None) == -1
    assert lib.cih_decoder_read_cache(None, 0, 0, 0, 1, None, None) == -1


@pytest.mark.parametrize("field", ["gain", 0, 31])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_rope_not_finite(field, value):
    """Rotary positions that a caller filled: they would make every key NaN."""
    c, b, r = cache(), batch(), ch.Rope(64)
    row = Fake((3, 2, 64))
    if field == "gain":
        r.struct.gain = value
    else:
        r.struct.freq[field] = value
    assert code(c.append, b, row, row, rope=r) == -1
    # frequencies past the pairs that turn are not read
    part = ch.Rope(32)
    part.struct.freq[16] = value
    assert code(c.append, b, Fake((3, 2, 64), at=0), row, rope=part) == -1
    assert "rotary" not in C.lib().cih_last_error().decode()
