"""Sizes and strides at the ends of the kv entry points' ranges: nothing here reaches a GPU."""
import ctypes as C

import qpack_amd as qa
from qpack_amd._lib import lib
from test_kv import P, attend, cache, refused, rows, write

TOP = 1 << 30


def test_sizes_past_63_bits_are_refused():
    b = C.c_int64(-5)
    for kind, bytes_of in ((qa.QPH_F16, lambda n, h, d, c: 4 * n * h * d * c), (qa.QPH_Q4, lambda n, h, d, c: n * h * -(-c // 8) * 9 * d)):
        for nseq, heads, hd, ctx in ((65535, 4096, 128, TOP), (65535, 4096, 64, TOP), (65535, 1024, 128, TOP), (65535, 512, 64, TOP), (65535, 4096, 128, 1 << 27), (3, 2, 64, 9)):
            want = bytes_of(nseq, heads, hd, ctx)
            status = lib().qph_kv_bytes(kind, nseq, heads, hd, ctx, C.byref(b))
            if want < 2 ** 63:
                assert status == 0 and b.value == want
            else:
                refused(status, "2^63")
                refused(write(cache(kind=kind, nseq=nseq, kv_heads=heads, head_dim=hd, ctx=ctx)), "2^63")
                refused(attend(cache(kind=kind, nseq=nseq, kv_heads=heads, head_dim=hd, ctx=ctx), heads=heads), "2^63")


def test_strides_past_63_bits_are_refused():
    f = lambda **k: cache(kind=qa.QPH_F16, v=2 * P, **k)   # noqa: E731
    for c in (f(ctx=TOP, row=1 << 40), f(row=1 << 62), f(nseq=3, seq=1 << 61), f(nseq=1, ctx=TOP, row=1 << 33)):
        refused(write(c), "2^63")
        refused(attend(c), "2^63")
    for c in (f(row=1 << 62, seq=128), f(ctx=TOP, row=1 << 33, seq=1 << 40)):   # a sequence's rows past 2^63, the sequences near
        refused(write(c), "overlap")
    far = rows(p=4 * P, seq=0, tok=0, head=0)
    for c in (f(nseq=1, seq=1 << 62), f(nseq=2, seq=1 << 60), f(nseq=1, ctx=1, row=1 << 62)):   # taken: the next check is what refuses
        refused(write(c, k=far, v=far, n=-1), "n must be")


def test_over_q_in_other_places_is_refused():
    """rows that are stored where other tokens' queries are still to be read"""
    for r in (rows(seq=3200), rows(tok=320), rows(tok=256), rows(head=128)):
        refused(attend(q=rows(), out=r), "q's strides")
    assert attend(q=rows(), out=rows(tok=320), n=0) == 0
    one = lambda **k: cache(ctx=4096, kv_heads=1, **k)   # noqa: E731
    for q, out, n, c in ((rows(), rows(), 3, one()), (rows(), rows(tok=7), 1, one()), (rows(), rows(seq=9), 3, one(nseq=1)), (rows(tok=0), rows(p=2 * P), 3, one())):
        refused(attend(c, q=q, out=out, n=n), "work")   # taken: the next check is what refuses


def test_cache_kinds_of_models_are_checked_first():
    m = C.c_void_p()
    for kind in (qa.QPH_F32, qa.QPH_Q8, qa.QPH_BF16, -1):
        refused(lib().qph_load_kv(b"/nonexistent", 0, kind, C.byref(m)), "cache: kind")
        assert m.value is None
    assert lib().qph_load_kv(b"/nonexistent", 0, qa.QPH_Q4, C.byref(m)) == -1 and "kind" not in lib().qph_last_error().decode()
