"""HipLlama.score: what it says of a text against the model's own logits (prefill_all), in 64 bits.

In decode steps the logits are the same to the bit, and only logprobs' own error is left (test_gpu_logprobs: under 1e-4 at these vocabularies).  In batched products logits are
within 1e-2 of the decode step's, the bound that every prompt is held to; moved by at most e each, a log probability moves by at most 2 e, and the entropy by
at most 2 e (1 + the spread of p ln p), taken as 2 e ln V."""
import math

import numpy as np
import pytest

import qpack_amd as qa

pytestmark = pytest.mark.gpu


def plain(logits, targets):
    x = logits.astype(np.float64)
    y = x - x.max(1, keepdims=True)
    y -= np.log(np.exp(y).sum(1, keepdims=True))
    H = -(np.exp(y) * y).sum(1)
    n = len(targets)
    logp = np.array([y[i, targets[i]] if 0 <= targets[i] < x.shape[1] else math.nan for i in range(n)])
    return y, H, logp


def check(r, logits, targets, e, top):
    y, H, logp = plain(logits, targets)
    V = logits.shape[1]
    assert np.array_equal(np.isnan(r.logp), np.isnan(logp)) and np.nanmax(np.abs(r.logp - logp), initial=0) <= 2 * e + 1e-4
    assert np.abs(r.entropy - H).max() <= 2 * e * math.log(V) + 1e-4
    order = np.argsort(-logits, axis=1, kind="stable")[:, :top]
    if e == 0:
        assert np.array_equal(r.top_index, order)
        rank = [int((logits[i] > logits[i, t]).sum() + (logits[i, :t] == logits[i, t]).sum()) if 0 <= t < V else -1 for i, t in enumerate(targets)]
        assert r.rank.tolist() == rank
    for i in range(len(targets)):
        assert np.abs(r.top_logp[i] - y[i, r.top_index[i]]).max(initial=0) <= 2 * e + 1e-4
        assert np.abs(r.top_logp[i] - y[i, order[i]]).max(initial=0) <= 2 * e + 1e-4
        assert (r.rank[i] == -1) == (not 0 <= targets[i] < V)


@pytest.mark.parametrize("name", ["mini", "mini128", "mini_q4", "mini_q4m", "mini_odd", "mini_q1", "mini_q1m", "mini_q4h", "mini_r7h"])
@pytest.mark.parametrize("cache", ["f16", "q4"])
def test_score(synth, name, cache, monkeypatch):
    print(f"score {name} {cache}", flush=True)
    V = qa.CONFIGS[name].vocab
    toks = np.random.default_rng(5).integers(0, V, 50).astype(np.int32)
    with qa.HipLlama.load(synth(name), max_ctx=64, cache=cache) as m:
        logits = m.prefill_all(toks)
        m.reset()
        r = m.score(toks, top=5)
        assert m.pos() == 50
        nxt = np.append(toks[1:], -1)
        check(r, logits, nxt, 1e-2, 5)
        follow = m.step(int(toks[3]))   # the text goes on behind it
        m.reset()
        m.prefill(toks)
        assert np.abs(m.step(int(toks[3])) - follow).max() <= 1e-2
        # decode steps
        monkeypatch.setenv("QPH_PREFILL_STEPS", "1")
        m.reset()
        steps = np.stack([m.step(int(t)) for t in toks])
        m.reset()
        targets = toks[::-1].copy()
        targets[4], targets[7] = V, -5
        check(m.score(toks, targets, top=64), steps, targets, 0, 64)


def test_pieces_windows_and_the_reference_order(synth):
    toks = np.random.default_rng(6).integers(0, 2048, 60).astype(np.int32)
    with qa.HipLlama.load(synth("mini128"), max_ctx=64) as m:
        whole = m.score(toks, top=3)
        m.reset()
        parts = [m.score(toks[i:j], np.append(toks[i + 1:j], toks[j] if j < 60 else -1), top=3) for i, j in ((0, 1), (1, 2), (2, 19), (19, 60))]
        for k in (0, 1, 4):
            a, b = np.concatenate([p[k] for p in parts]), whole[k]
            assert np.nanmax(np.abs(a - b)) <= 2e-2 * math.log(2048)
        m.reset()
        m.set_window(7, 1)
        logits = m.prefill_all(toks)
        m.reset()
        check(m.score(toks, top=2), logits, np.append(toks[1:], -1), 1e-2, 2)
        m.reset()
        m.set_window(0)
        m.set_order(1)
        logits = m.prefill_all(toks)
        m.reset()
        check(m.score(toks, top=2), logits, np.append(toks[1:], -1), 0, 2)


def test_chunks_and_few_rows_at_a_time(synth, monkeypatch):
    """a prompt of several chunks, whose tokens' logits fill the buffer many times over"""
    monkeypatch.setenv("QPH_PF_CHUNK", "24")
    toks = np.random.default_rng(7).integers(0, 1000, 100).astype(np.int32)
    with qa.HipLlama.load(synth("mini"), max_ctx=128) as m:
        logits = m.prefill_all(toks)
        m.reset()
        r = m.score(toks, top=7)
        check(r, logits, np.append(toks[1:], -1), 1e-2, 7)
        m.reset()
        again = m.score(toks)
        assert again.top_index.shape == (100, 0) and np.array_equal(again.entropy, r.entropy) and np.array_equal(again.rank, r.rank)


def test_refusals(synth):
    with qa.HipLlama.load(synth("mini"), max_ctx=16) as m:
        for top in (-1, 65):
            with pytest.raises(qa.QphError, match="top"):
                m.score([1, 2], top=top)
        with pytest.raises(qa.QphError, match="out of range"):
            m.score([1, 1000])
        with pytest.raises(qa.QphError, match="context window full"):
            m.score([1] * 17)
        with pytest.raises(qa.QphError, match="as many"):
            m.score([1, 2], targets=[3])
        assert m.pos() == 0 and m.score([]).logp.shape == (0,)
        m.score([1] * 16)
        assert m.pos() == 16


def test_a_text_of_2_31_tokens_does_not_fit(synth):
    """its last position passes 32 bits: refused before any of its tokens is read"""
    import ctypes as C

    from qpack_amd._lib import lib
    with qa.HipLlama.load(synth("mini"), max_ctx=16) as m:
        m.prefill([1, 2, 3], 0)
        tokens, out = (C.c_int * 4)(1, 2, 3, 4), (C.c_float * 1)()
        at = C.cast(tokens, C.POINTER(C.c_int))
        for call in (lambda n: lib().qph_score(m._h, at, None, n, 0, None, None, None, None, None), lambda n: lib().qph_prefill(m._h, at, n, 0, None), lambda n: lib().qph_prefill_all(m._h, at, n, out)):
            for n in (2 ** 31 - 1, 2 ** 31 - 3, 14):
                assert call(n) == -1 and b"context window full" in lib().qph_last_error()
        assert m.pos() == 3
