"""The kv entry points' refusals, and the sizes they report: nothing here reaches a GPU."""
import ctypes as C

import pytest

import qpack_amd as qa
from qpack_amd._lib import KvC, RowsC, lib

P = 1 << 20   # an address that is never read


def cache(kind=qa.QPH_Q4, nseq=2, kv_heads=2, head_dim=64, ctx=100, k=P, v=P, seq=0, row=0):
    return KvC(kind, nseq, kv_heads, head_dim, ctx, k, v, seq, row)


def rows(p=P, type=qa.QPH_F16, seq=6400, tok=640, head=64):
    return RowsC(p, type, seq, tok, head)


def refused(status, words):
    assert status == -1
    msg = lib().qph_last_error().decode()
    assert words in msg, msg


def write(c, k=None, v=None, n=3, pos=P, f="qph_kv_write"):
    k, v = k or rows(), v or rows()
    return getattr(lib(), f)(C.byref(c), C.byref(k), C.byref(v), n, pos, None, None)


def attend(c=None, q=None, out=None, heads=4, n=3, pos=P, window=0, sinks=0, scale=0.0, work=None, bytes=0):
    c, q, out = c or cache(), q or rows(), out or rows()
    return lib().qph_kv_attention(C.byref(c), C.byref(q), C.byref(out), heads, n, pos, None, window, sinks, scale, work, bytes, None)


@pytest.mark.parametrize("c,words", [
    (cache(kind=qa.QPH_Q8), "kind"), (cache(nseq=0), "nseq"), (cache(nseq=65536), "nseq"), (cache(kv_heads=0), "kv_heads"), (cache(kv_heads=4097), "kv_heads"),
    (cache(head_dim=96), "head_dim"), (cache(ctx=0), "ctx"), (cache(ctx=(1 << 30) + 1), "ctx"), (cache(k=None), "NULL"), (cache(k=P + 8), "aligned"),
    (cache(kind=qa.QPH_F16, v=None), "NULL"), (cache(kind=qa.QPH_F16, v=P + 2), "aligned"), (cache(kind=qa.QPH_F16, row=132), "multiples of 8"),
    (cache(kind=qa.QPH_F16, row=120), "overlap"), (cache(kind=qa.QPH_F16, seq=99 * 128), "overlap"),
])
def test_cache_refusals(c, words):
    refused(write(c), words)
    refused(write(c, f="qph_kv_read"), words)
    refused(attend(c), words)


@pytest.mark.parametrize("r,words", [(rows(p=None), "NULL"), (rows(type=qa.QPH_Q8), "type"), (rows(p=P + 1), "aligned"), (rows(seq=-64), "negative"), (rows(tok=-64), "negative")])
def test_rows_refusals(r, words):
    refused(write(cache(), k=r), words)
    refused(write(cache(), v=r), words)
    refused(attend(q=r), words)
    refused(attend(out=r), words)


def test_other_refusals():
    refused(write(cache(), v=rows(type=qa.QPH_BF16)), "same type")
    refused(write(cache(), n=-1), "n must be")
    refused(write(cache(), n=(1 << 20) + 1), "n must be")
    refused(write(cache(), pos=None), "pos is NULL")
    for r in (rows(tok=0), rows(head=32), rows(seq=0)):   # rows read may repeat, rows written may not
        refused(write(cache(), v=r, f="qph_kv_read"), "overlap")
        refused(attend(out=r), "overlap")
    refused(attend(heads=3), "multiple of kv_heads")
    refused(attend(heads=0), "multiple of kv_heads")
    refused(attend(n=1 << 20, heads=32), "n * heads")
    refused(attend(window=-1), "negative")
    refused(attend(sinks=-1), "negative")
    refused(attend(pos=None), "pos is NULL")
    for s in (-1.0, float("nan"), float("inf")):
        refused(attend(scale=s), "scale")
    refused(attend(out=rows(type=qa.QPH_F32)), "same type")
    refused(lib().qph_kv_write(None, C.byref(rows()), C.byref(rows()), 1, P, None, None), "cache is NULL")
    refused(lib().qph_kv_bytes(qa.QPH_Q4, 1, 1, 64, 1, None), "bytes is NULL")


def test_rows_that_would_be_written_twice_are_refused():
    """each stride alone is long enough, two of them together are not; nested in any order they are"""
    for r in (rows(tok=64, head=64), rows(tok=128, head=64), rows(seq=64 * 11, tok=64 * 4, head=64), rows(seq=64, tok=128, head=320), rows(seq=1 << 62, tok=1 << 62, head=64)):
        refused(attend(out=r), "overlap")
    for r in (rows(tok=64, head=192), rows(seq=64, tok=128, head=384), rows(seq=1 << 62, tok=256, head=64)):
        refused(attend(out=r, scale=-1.0), "scale")   # taken: the next check is what refuses
    refused(write(cache(), v=rows(p=P), f="qph_kv_read"), "k and v overlap")
    refused(write(cache(kind=qa.QPH_F16)), "k and v overlap")


def test_sizes_past_a_launch_are_refused():
    wide = cache(kind=qa.QPH_F16, nseq=1, kv_heads=4096, head_dim=128, v=2 * P)
    far = rows(p=4 * P, seq=0, tok=0, head=0)
    refused(write(wide, k=far, v=far, n=32769), "2^34")
    refused(attend(scale=3e38), "scale")


def test_no_tokens_is_no_call():
    assert write(cache(), n=0) == 0 and write(cache(), n=0, f="qph_kv_read") == 0 and attend(n=0) == 0


def test_sizes():
    b = C.c_int64()
    for ctx in (1, 8, 9, 1 << 30):
        assert lib().qph_kv_bytes(qa.QPH_Q4, 3, 2, 128, ctx, C.byref(b)) == 0 and b.value == 3 * 2 * -(-ctx // 8) * 1152
        assert lib().qph_kv_bytes(qa.QPH_F16, 3, 2, 64, ctx, C.byref(b)) == 0 and b.value == 3 * ctx * 2 * 64 * 4
    refused(lib().qph_kv_bytes(qa.QPH_Q4, 3, 2, 80, 10, C.byref(b)), "head_dim")


def test_work():
    """scratch only where a row is split, and the attention asks for all of it"""
    b, one = C.c_int64(), cache(nseq=1, kv_heads=1, ctx=4096)
    f = lib().qph_kv_attention_work
    assert f(C.byref(one), qa.QPH_F16, 4, 1, 0, 0, C.byref(b)) == 0 and b.value > 0 and b.value % (4 * 66 * 4) == 0
    refused(attend(one, n=1, work=None, bytes=b.value), "work")
    refused(attend(one, n=1, work=P, bytes=b.value - 1), "work")
    refused(attend(one, n=1, work=P + 4, bytes=b.value), "work")
    assert f(C.byref(cache(ctx=64)), qa.QPH_F16, 4, 1, 0, 0, C.byref(b)) == 0 and b.value == 0
    assert f(C.byref(one), qa.QPH_F16, 4, 0, 0, 0, C.byref(b)) == 0 and b.value == 0
    refused(f(C.byref(one), qa.QPH_Q4, 4, 1, 0, 0, C.byref(b)), "type")
    refused(f(C.byref(one), qa.QPH_F16, 4, 1, -1, 0, C.byref(b)), "negative")
