"""Refusals of attention with sinks, weighing, eviction, shifted appends and the
verification of drafts (CPU: no call gets as far as a device)."""
import ctypes
import math

import pytest

import codon_hip as ch
from codon_hip import _lib as C
from test_ops_args import Fake, batch, cache, code


def test_sinks_and_shifts_refusals():
    c, b, q = cache(), batch(), Fake((3, 4, 64))
    ws = Fake((1 << 20,), "uint8")
    assert code(c.attend, b, q, q, window=3, sinks=-1, workspace=ws) == -1
    assert code(c.attend, b, q, q, window=-3, sinks=1, workspace=ws) == -1
    row = Fake((3, 2, 64))
    for bad in (Fake((3,), "int32"), Fake((2,), "int64"), Fake((2,), "int32", stride=(2,))):
        with pytest.raises((TypeError, ValueError)):
            c.append(b, row, row, shifts=bad)
    assert code(c.append, b, row, row, shifts=Fake((2,), "int32", at=6)) == -1


def test_weigh_refusals():
    c, b = cache(), batch()
    q, lse, w = Fake((3, 4, 64)), Fake((3, 4)), Fake((4, 2, 64))
    for a in ((q, Fake((3, 2)), w), (q, lse, Fake((4, 2, 32))), (q, lse, Fake((4, 2, 64), "float16")), (Fake((3, 4, 64), "int8"), lse, w),
              (q, lse, Fake((4, 2, 64), stride=(256, 128, 2))), (Fake((2, 4, 64)), lse, w)):
        with pytest.raises((TypeError, ValueError)):
            c.weigh(b, *a)
    for keep in (-0.1, 1.1, math.nan):
        assert code(c.weigh, b, q, lse, w, keep=keep) == -1
    assert code(c.weigh, b, q, lse, w, window=-1) == -1
    assert code(c.weigh, b, q, lse, w, window=1, sinks=-1) == -1
    assert code(c.weigh, b, q, lse, w, scale=math.inf) == -1
    assert code(c.weigh, b, Fake((3, 3, 64)), Fake((3, 3)), w) == -2
    assert code(c.weigh, b, q, Fake((3, 4), at=0), w) == -1
    assert code(c.weigh, b, q, lse, Fake((4, 2, 64), at=0)) == -1
    assert code(c.weigh, b, q, Fake((3, 4), at=2), w) == -1
    assert code(c.weigh, b, Fake((3, 4, 64), at=2), lse, w) == -1
    c.weigh(batch(n_rows=0, max_rows=0), Fake((0, 4, 64), at=0), Fake((0, 4), at=0), w)  # nothing to do


def test_evict_refusals():
    c, b, w = cache(), batch(), Fake((4, 2, 64))
    need = c.evict_workspace(b, 100)
    assert need > 0
    ws = Fake((need,), "uint8")
    for kw in (dict(weights_out=Fake((4, 2, 63))), dict(lens_out=Fake((3,), "int32")), dict(lens_out=Fake((2,), "int64")),
               dict(shifts=Fake((1,), "int32")), dict(kept=Fake((2, 2, 99), "int32")), dict(kept=Fake((2, 1, 100), "int32")),
               dict(workspace=Fake((need,), "int8"))):
        with pytest.raises((TypeError, ValueError)):
            c.evict(b, w, 100, **{"workspace": ws, **kw})
    with pytest.raises((TypeError, ValueError)):
        c.evict(b, Fake((4, 2, 64), "float16"), 100, workspace=ws)
    assert code(c.evict, b, w, 0, workspace=ws) == -2
    assert code(c.evict, b, w, 100, first=60, recent=41, workspace=ws) == -1
    assert code(c.evict, b, w, 100, first=-1, workspace=ws) == -1
    assert code(c.evict, b, w, 100, recent=-1, workspace=ws) == -1
    assert code(c.evict, b, w, 100) == -3
    assert code(c.evict, b, w, 100, workspace=Fake((need - 1,), "uint8")) == -3
    assert code(c.evict, b, w, 100, workspace=Fake((need,), "uint8", at=8)) == -3
    assert code(c.evict, b, Fake((4, 2, 64), at=0), 100, workspace=ws) == -1
    assert code(c.evict, b, w, 100, shifts=Fake((2,), "int32", at=2), workspace=ws) == -1
    assert code(c.evict_workspace, b, 0) == -2
    # a table's room bounds what the largest budgets need
    assert c.evict_workspace(b, 1 << 30) == c.evict_workspace(b, 5 * 64)
    # the rows' offsets are not read
    b.struct.cu_rows = None
    assert code(c.evict, b, w, 100) == -3
    lib = C.lib()
    assert lib.cih_kv8_evict_workspace(c._at, b._at, 4, None) == -1
    assert lib.cih_kv8_evict(None, b._at, 4, 0, 0, None, None, None, None, None, None, 0, None) == -1
    none = batch(n_rows=0, max_rows=0, n_seq=0)
    c.evict(none, w, 100)  # nothing to do


def test_verify_refusals():
    x, a = Fake((5, 100)), Fake((3, 100))
    d, cu, n = Fake((3,), "int32"), Fake((3,), "int32"), Fake((2,), "int32")
    u, v, ws = Fake((3,)), Fake((2,)), Fake((1 << 22,), "uint8")

    def go(logits=x, drafts=d, offs=cu, acc=n, tok=n, **kw):
        kw = {"draft_logits": a, "accept_at": u, "sample_at": v, "workspace": ws, **kw}
        ch.verify_drafts(logits, drafts, offs, acc, tok, **kw)

    for kw in (dict(logits=Fake((4, 100))), dict(logits=Fake((5, 100), "int32")), dict(logits=Fake((5, 100), stride=(1, 5))),
               dict(draft_logits=Fake((2, 100))), dict(draft_logits=Fake((3, 99))), dict(draft_logits=Fake((3, 100), "float16")),
               dict(draft_logits=Fake((3, 100), stride=(1, 3))), dict(drafts=Fake((3,), "int64")), dict(offs=Fake((2,), "int32")),
               dict(acc=Fake((3,), "int32")), dict(tok=Fake((2,), "float32")), dict(accept_at=Fake((2,))), dict(sample_at=Fake((3,)))):
        with pytest.raises((TypeError, ValueError)):
            go(**kw)
    assert code(go, temperature=-1.0) == -1
    assert code(go, temperature=math.nan) == -1
    assert code(go, temperature=math.inf) == -1
    assert code(go, accept_at=None) == -1
    assert code(go, sample_at=None) == -1
    assert code(go, logits=Fake((5, 100), at=0)) == -1
    assert code(go, logits=Fake((5, 100), at=2)) == -1
    assert code(go, draft_logits=Fake((3, 100), at=2)) == -1
    assert code(go, logits=Fake((5, 100), stride=(99, 1))) == -2
    assert code(go, draft_logits=Fake((3, 100), stride=(99, 1))) == -2
    assert code(go, acc=Fake((2,), "int32", at=0)) == -1
    assert code(ch.verify_drafts_workspace, 1, 1, 0) == -2
    assert code(ch.verify_drafts_workspace, -1, 1, 5) == -2
    assert code(ch.verify_drafts_workspace, 1, -1, 5) == -2
    need = ch.verify_drafts_workspace(2, 3, 100)
    wide = ch.verify_drafts_workspace(2, 3, 100000)
    for size, logits, about in ((need, x, a), (wide, Fake((5, 100000)), Fake((3, 100000)))):
        if size:
            assert code(go, logits=logits, draft_logits=about, workspace=Fake((size - 1,), "uint8")) == -3
            assert code(go, logits=logits, draft_logits=about, workspace=None) == -3
            assert code(go, logits=logits, draft_logits=about, workspace=Fake((size,), "uint8", at=8)) == -3
    lib = C.lib()
    assert lib.cih_verify_drafts_workspace(1, 1, 5, None) == -1
    assert lib.cih_verify_drafts(9, None, 0, None, 0, 1, 1, 5, None, None, None, None, 1.0, None, None, None, 0, None) == -1
    ch.verify_drafts(Fake((0, 100), at=0), Fake((0,), "int32", at=0), Fake((1,), "int32"), Fake((0,), "int32", at=0),
                     Fake((0,), "int32", at=0), accept_at=Fake((0,)), sample_at=Fake((0,)))  # nothing to do
    size = ctypes.c_size_t()
    assert lib.cih_verify_drafts_workspace(0, 0, 1, ctypes.byref(size)) == 0
