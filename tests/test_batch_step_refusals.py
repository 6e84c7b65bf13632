"""Refusals of append, copy, attention behind a prefix and logprobs, and the sizes they report: nothing here reaches a GPU."""
import ctypes as C

import pytest

import qpack_amd as qa
from qpack_amd._lib import KvC, RowsC, TurnC, lib

P = 1 << 24   # addresses that are never read


def cache(kind=qa.QPH_Q4, nseq=2, kv_heads=2, head_dim=64, ctx=100, k=P, v=2 * P, seq=0, row=0):
    return KvC(kind, nseq, kv_heads, head_dim, ctx, k, v, seq, row)


def rows(p=P, type=qa.QPH_F16, seq=6400, tok=640, head=64):
    return RowsC(p, type, seq, tok, head)


def turn(cos=P, sin=P, places=50, half=32, at=None, q_norm=None, k_norm=None, eps=1e-6):
    return TurnC(cos, sin, places, half, at, q_norm, k_norm, eps)


def refused(status, words):
    assert status == -1
    msg = lib().qph_last_error().decode()
    assert words in msg, msg


def append(c=None, q=None, k=None, v=None, out=None, heads=4, n=3, pos=P, t=None):
    c, q, k, v, out, t = c or cache(), q or rows(), k or rows(), v or rows(), out or rows(), t or turn()
    return lib().qph_kv_append(*(C.byref(x) for x in (c, q, k, v, out)), heads, n, pos, None, C.byref(t), None)


def copy(dst=None, src=None, index=P, stride=3, n=3, pos=P, apart=0, work=None, size=0):
    dst, src = dst or cache(), src or cache(k=P << 4)
    return lib().qph_kv_copy(C.byref(dst), C.byref(src), index, stride, n, pos, None, None, apart, work, size, None)


def attend(c=None, p=None, q=None, out=None, heads=4, n=3, pos=P, scale=0.0, work=P, size=1 << 40):
    c, p, q, out = c or cache(), p or cache(nseq=1), q or rows(), out or rows()
    return lib().qph_kv_attention_prefix(C.byref(c), C.byref(p), None, C.byref(q), C.byref(out), heads, n, pos, None, scale, work, size, None)


def logprobs(x=P, type=qa.QPH_F32, n=3, vocab=100, ld=100, tokens=P, top=0, logp=P, ti=None, tl=None, work=None, size=0):
    return lib().qph_logprobs(x, type, n, vocab, ld, tokens, top, logp, None, None, ti, tl, work, size, None)


@pytest.mark.parametrize("c,words", [(cache(kind=qa.QPH_Q8), "kind"), (cache(nseq=0), "nseq"), (cache(head_dim=96), "head_dim"), (cache(ctx=0), "ctx"), (cache(k=None), "NULL"), (cache(k=P + 8), "aligned"),
                                     (cache(kind=qa.QPH_F16, v=None), "NULL"), (cache(kind=qa.QPH_F16, row=132), "multiples of 8"), (cache(kind=qa.QPH_F16, row=120), "overlap")])
def test_caches(c, words):
    refused(append(c), words)
    refused(copy(c), words)
    refused(copy(cache(), c), words)
    refused(attend(c), words)
    refused(attend(p=c), words)


def test_append():
    for r, words in ((rows(p=None), "NULL"), (rows(type=qa.QPH_Q8), "type"), (rows(p=P + 1), "aligned"), (rows(seq=-64), "negative")):
        for name in ("q", "k", "v", "out"):
            refused(append(**{name: r}), words)
    refused(append(q=rows(type=qa.QPH_BF16)), "same type")
    refused(append(k=rows(type=qa.QPH_BF16)), "same type")
    refused(append(q=rows(type=qa.QPH_BF16), out=rows(type=qa.QPH_BF16)), "same type")
    refused(append(out=rows(tok=63)), "overlap")
    refused(append(out=rows(seq=12800)), "out over q")
    for heads in (0, 3, 65536):
        refused(append(heads=heads), "heads")
    refused(append(n=-1), "n must be")
    refused(append(c=cache(nseq=1, kv_heads=32), heads=64, n=1 << 20), "2^26")
    refused(append(pos=None), "pos is NULL")
    for half in (-8, 4, 40, 12):
        refused(append(t=turn(half=half)), "half the rotated")
    for places in (0, -1, (1 << 31) + 1):
        refused(append(t=turn(places=places)), "places")
    refused(append(t=turn(cos=None)), "cos is NULL")
    refused(append(t=turn(sin=None)), "sin is NULL")
    refused(append(t=turn(q_norm=P + 2)), "aligned")
    for eps in (-1.0, float("inf"), float("nan")):
        refused(append(t=turn(eps=eps)), "eps")
    assert append(n=0) == 0 and append(n=0, t=turn(cos=None, sin=None, half=0)) == 0


def size(f, *a):
    b = C.c_int64(-1)
    assert f(*a, C.byref(b)) == 0, lib().qph_last_error()
    return b.value


def test_copy():
    for src in (cache(kind=qa.QPH_F16, k=P << 4, v=P << 5), cache(kv_heads=1), cache(head_dim=128)):
        refused(copy(src=src), "same kind")
    refused(copy(n=-1), "n must be")
    refused(copy(n=(1 << 20) + 1), "n must be")
    wide = dict(kind=qa.QPH_F16, nseq=1, kv_heads=4096, head_dim=128, ctx=8, v=P << 5)
    refused(copy(cache(**wide), cache(**{**wide, "k": P << 4}), n=1 << 20), "2^34")   # more threads than a launch counts
    refused(copy(index=None), "index is NULL")
    refused(copy(pos=None), "pos is NULL")
    refused(copy(stride=-1), "negative stride")
    assert copy(n=0) == 0
    # scratch only where memory is shared: a 4-bit record of 8 positions is 9 head_dim bytes
    c, far = cache(), cache(k=P << 4)
    work = lambda d, s, n, apart=0: size(lib().qph_kv_copy_work, C.byref(d), C.byref(s), n, apart)   # noqa: E731
    assert work(c, far, 9) == 0 and work(c, c, 9, 1) == 0 and work(c, c, 0) == 0
    assert work(c, c, 9) == 2 * 2 * 2 * 9 * 64 and work(c, c, 8) == 2 * 2 * 9 * 64
    refused(copy(src=c), "qph_kv_copy_work")
    refused(copy(src=c, work=P, size=10), "qph_kv_copy_work")
    refused(copy(src=c, work=P + 8, size=1 << 30), "qph_kv_copy_work")
    # fp16: two sequences of one memory, a sequence's K against the other's V
    a, b = (cache(kind=qa.QPH_F16, nseq=1, k=P + i * 25600, v=2 * P + i * 25600) for i in (0, 1))
    assert work(a, b, 10) == 0 and work(a, a, 10) == 4 * 10 * 128
    assert work(a, cache(kind=qa.QPH_F16, nseq=1, k=P + 25600 - 16, v=4 * P), 10) == 4 * 10 * 128
    assert work(a, cache(kind=qa.QPH_F16, nseq=1, k=4 * P, v=P + 16), 10) == 4 * 10 * 128
    refused(lib().qph_kv_copy_work(C.byref(c), C.byref(c), 3, 0, None), "NULL")


def test_attention_prefix():
    for p in (cache(nseq=2), cache(nseq=1, kv_heads=1), cache(nseq=1, head_dim=128), cache(kind=qa.QPH_F16, nseq=1)):
        refused(attend(p=p), "prefix must be")
    refused(attend(heads=3), "multiple of kv_heads")
    refused(attend(n=-1), "n must be")
    refused(attend(cache(nseq=60000), n=100), "2^23")
    refused(attend(cache(nseq=1000, kv_heads=4000, ctx=8), cache(nseq=1, kv_heads=4000), heads=4000, n=1000), "2^30")
    refused(attend(pos=None), "pos is NULL")
    refused(attend(out=rows(type=qa.QPH_F32)), "same type")
    refused(attend(out=rows(seq=12800)), "out over q")
    for scale in (-1.0, float("inf"), float("nan"), 3e38):
        refused(attend(scale=scale), "scale")
    c, p = cache(), cache(nseq=1)
    assert size(lib().qph_kv_attention_prefix_work, C.byref(c), C.byref(p), qa.QPH_F16, 4, 3) == 0   # few positions: nothing to be joined
    p = cache(nseq=1, ctx=5000)
    need = size(lib().qph_kv_attention_prefix_work, C.byref(c), C.byref(p), qa.QPH_F16, 4, 3)
    assert need >= 2 * 3 * 4 * 2 * 66 * 4   # two sums of a row at least
    refused(attend(p=p, size=need - 1), "qph_kv_attention_prefix_work")
    refused(attend(p=p, work=None), "qph_kv_attention_prefix_work")
    refused(attend(p=p, work=P + 4), "qph_kv_attention_prefix_work")
    assert attend(n=0) == 0 and size(lib().qph_kv_attention_prefix_work, C.byref(c), C.byref(p), qa.QPH_F16, 4, 0) == 0
    refused(lib().qph_kv_attention_prefix_work(C.byref(c), C.byref(p), qa.QPH_Q8, 4, 3, C.byref(C.c_int64())), "type of q")


def test_logprobs():
    refused(logprobs(x=None), "NULL")
    refused(logprobs(type=qa.QPH_Q4), "type")
    refused(logprobs(x=P + 2), "aligned")
    for n in (-1, (1 << 23) + 1, 1 << 24, (1 << 24) + 1):
        refused(logprobs(n=n), "rows")
    for vocab in (0, (1 << 28) + 1):
        refused(logprobs(vocab=vocab), "vocab")
    for top, vocab in ((-1, 100), (65, 100), (8, 7)):
        refused(logprobs(top=top, vocab=vocab), "top")
    refused(logprobs(ld=-1), "negative stride")
    refused(logprobs(tokens=None), "need tokens")
    refused(logprobs(top=3), "top_index is NULL")
    refused(logprobs(top=3, ti=P), "top_logp is NULL")
    refused(logprobs(vocab=100000), "qph_logprobs_work")
    refused(logprobs(vocab=100000, work=P + 4, size=1 << 30), "qph_logprobs_work")
    work = lambda *a: size(lib().qph_logprobs_work, *a)   # noqa: E731
    assert work(qa.QPH_F32, 0, 100, 3) == 0 and work(qa.QPH_F32, 5000, 128256, 64) == 0 and work(qa.QPH_BF16, 1, 100, 64) == 0
    assert 0 < work(qa.QPH_F32, 1, 128256, 20) <= 64 * (16 + 8 * 20)
    assert logprobs(n=0) == 0


def test_bindings_refuse_gradients():
    torch = pytest.importorskip("torch")
    from qpack_amd.kvcache import _binding
    b = _binding()
    c = b.Cache(qa.QPH_Q4, 2, 2, 64, 40, 1 << 20, 0, 0, 0, 0, torch.zeros(1, dtype=torch.uint8))
    x, pos, g = torch.zeros(2, 3, 2, 64).half(), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, 2, 64, dtype=torch.float16, requires_grad=True)
    t = torch.zeros(9, 32)
    for f in (lambda a: c.append(a, x, x, x, pos, None, t, t, None, None, None, 1e-6), lambda a: c.attention_prefix(a, x, pos, None, 0.0, c, None), lambda a: b.logprobs(a[0, 0].float(), None, 0)):
        with pytest.raises(qa.QphError, match="requires a gradient"):
            f(g)
        with torch.no_grad(), pytest.raises(qa.QphError, match="device|GPU"):
            f(g)
    for other in (None, 3, "c"):
        with pytest.raises((TypeError, qa.QphError), match="must be|device"):
            c.copy(other, torch.zeros(2, 3, dtype=torch.int32), pos, None, None, False)
