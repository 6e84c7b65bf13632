"""HipLlama with a 4-bit cache and with a sliding window (set_cache, set_window) against a plain 64-bit forward of the same file.

Tolerance: the path's logit contract (max-abs 1e-2, relative 1e-3).  Its float orders and int16 activations stay far below that; a 4-bit
code moves by a step where the kernels' fp32 key and the 64-bit one lie on two sides of a border, which is one dim of one position among
the visible ones."""
import json
import math
import struct

import numpy as np
import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
ATOL, RTOL = 1e-2, 1e-3


def held(x):
    """what a 4-bit cache holds of rows [.., head_dim]"""
    y = x.unflatten(-1, (-1, 32))
    s = (y.abs().amax(-1, keepdim=True).clamp(max=65504.).float() / 7).to(torch.bfloat16).half().double()
    return torch.where(s > 0, (y / s).round().clamp(-7, 7) * s, 0.).flatten(-2)


class Plain:
    def __init__(self, path):
        raw = open(path, "rb").read()
        toc = {}
        for i in range(struct.unpack("<I", raw[8:12])[0]):
            e = raw[16 + 72 * i:88 + 72 * i]
            toc[e[:56].rstrip(b"\0").decode()] = struct.unpack("<QQ", e[56:72])
        blob = lambda n: raw[toc[n][0]:toc[n][0] + toc[n][1]]   # noqa: E731
        self.c = json.loads(blob("config.json"))
        self.w = {}
        for t in json.loads(blob("manifest.json"))["tensors"]:
            if t["kind"] == "q8":
                x = np.frombuffer(blob(t["blob"]), np.int8).reshape(t["shape"]) * np.frombuffer(blob(t["scale"]), np.float32).astype(np.float64)[:, None]
            else:
                assert t["kind"] == "f32"
                x = np.frombuffer(blob(t["blob"]), np.float32).astype(np.float64)
            self.w[t["name"]] = torch.from_numpy(np.ascontiguousarray(x))

    def logits(self, toks, kind="f16", window=0, sinks=0, cache=None):
        """[n, vocab]: every position's; cache: the (K, V) [n, kv_heads, head_dim] of each layer that the attention reads instead of the rounded
        rows, which are to lie within half a step (4-bit; the scale's 2^-9 of 7 steps more) of them, fp16's rounding (2^-11) and 2e-3 for the
        path's own error before it"""
        c, w, n = self.c, self.w, len(toks)
        H, G, D, eps = c["num_attention_heads"], c["num_key_value_heads"], c["head_dim"], c["rms_norm_eps"]
        norm = lambda x, g: x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * g   # noqa: E731
        ang = torch.arange(n).double()[:, None] / c["rope_theta"] ** (torch.arange(D // 2).double() * 2 / D)
        cs, sn = torch.cos(ang)[:, None], torch.sin(ang)[:, None]

        def rope(x):
            a, b = x[..., :D // 2], x[..., D // 2:]
            return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)
        P, p = torch.arange(n)[:, None], torch.arange(n)[None]
        seen = p <= P
        if window:
            seen &= (p > P - window) | (p < sinks)
        x = w["embed"][torch.from_numpy(np.asarray(toks)).long()]
        for i in range(c["num_hidden_layers"]):
            g = lambda s: w[f"layers.{i}.{s}"]   # noqa: E731
            y = norm(x, g("attn_norm"))
            q, k, v = (y @ g("w" + s).T + (g("b" + s) if c["qkv_bias"] else 0) for s in "qkv")
            q, k, v = rope(q.view(n, H, D)), rope(k.view(n, G, D)), v.view(n, G, D)
            if cache is not None:
                for mine, theirs in ((k, cache[i][0]), (v, cache[i][1])):
                    step = mine.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) / 7 if kind == "q4" else torch.zeros(1)
                    off = (theirs - mine).unflatten(-1, (-1, 32)).abs()
                    assert bool((off <= step * (0.5 + 2.0 ** -6) + 2e-3).all()), f"layer {i}: a cached row is {float((off - step / 2).max()):.3g} past half a step"
                k, v = cache[i]
            else:
                k, v = (held(k), held(v)) if kind == "q4" else (k.half().double(), v.half().double())
            a = torch.einsum("thd,shd->hts", q, k.repeat_interleave(H // G, 1)) / math.sqrt(D)
            a = torch.softmax(a.masked_fill(~seen, -math.inf), -1)
            x = x + torch.einsum("hts,shd->thd", a, v.repeat_interleave(H // G, 1)).reshape(n, H * D) @ g("wo").T
            y = norm(x, g("ffn_norm"))
            u = y @ g("w_gate").T
            x = x + (u * torch.sigmoid(u) * (y @ g("w_up").T)) @ g("w_down").T
        head = w["embed"] if c["tie_embeddings"] else w["lm_head"]
        return (norm(x, w["final_norm"]) @ head.T).numpy()


def cached(m, ref):
    """the model's cache as its snapshot gives it"""
    raw, L, G, D = bytes(m.snapshot()), ref.c["num_hidden_layers"], ref.c["num_key_value_heads"], ref.c["head_dim"]
    x = torch.from_numpy(np.frombuffer(raw[4:], np.float16).astype(np.float64)).view(L, 2, m.pos(), G, D)
    return [(x[i, 0], x[i, 1]) for i in range(L)]


def check(got, want, what):
    err = np.abs(got - want)
    assert np.all(err <= np.maximum(ATOL, RTOL * np.abs(want))), f"{what}: max|d| {err.max():.3g}"


MODES = [("q4", 0, 0), ("f16", 24, 4), ("q4", 33, 0), ("q4", 20, 9), ("f16", 1, 0)]


@pytest.mark.parametrize("cfg", ["mini", "mini128", "mini_r7"])
@pytest.mark.parametrize("kind,window,sinks", MODES)
def test_prompt_steps_and_greedy(cfg, kind, window, sinks, synth):
    path = synth(cfg)
    ref = Plain(path)
    rng = np.random.default_rng(5)
    V = ref.c["vocab_size"]
    toks = rng.integers(0, V, 90).astype(np.int32)
    with qa.HipLlama.load(path, max_ctx=256) as m:
        m.set_cache(kind)
        m.set_window(window, sinks)
        print(f"{cfg} {kind} window {window} sinks {sinks}", flush=True)
        want = ref.logits(toks, kind, window, sinks)
        plain = ref.logits(toks)
        assert np.abs(want - plain)[-1].max() > 3 * ATOL   # the mode shows in the logits
        check(m.prefill(toks[:70]), want[69], "prompt")
        check(m.prefill(toks[70:75]), want[74], "turn")
        for i in range(75, 90):
            check(m.step(int(toks[i])), want[i], f"step {i}")
        out = m.greedy_run(int(toks[0]), 12)
        seq = np.concatenate([toks, [toks[0]], out])
        want = ref.logits(seq, kind, window, sinks)
        for i, t in enumerate(out):
            row = want[90 + i]
            assert row[t] >= row.max() - 2 * ATOL, f"greedy {i}"
        m.reset()
        check(m.prefill(toks[:2]), ref.logits(toks[:2], kind, window, sinks)[1], "prompt of two")


@pytest.mark.parametrize("kind,window,sinks", [("q4", 0, 0), ("f16", 100, 4), ("q4", 150, 5)])
@pytest.mark.parametrize("few", ["", "0"])
def test_long_prompt_in_chunks(kind, window, sinks, few, synth, monkeypatch):
    path = synth("mini")
    monkeypatch.setenv("QPH_KV_FEW", few)   # 0: every call through the many-token kernel
    toks = np.random.default_rng(6).integers(0, 1000, 700).astype(np.int32)
    want = Plain(path).logits(toks, kind, window, sinks)
    for chunk in (0, 97):
        if chunk:
            monkeypatch.setenv("QPH_PF_CHUNK", str(chunk))
        with qa.HipLlama.load(path, max_ctx=800) as m:
            m.set_cache(kind)
            m.set_window(window, sinks)
            check(m.prefill(toks[:650]), want[649], f"chunk {chunk}")
            check(m.prefill(toks[650:]), want[699], f"chunk {chunk}, second")


@pytest.mark.parametrize("kind,window,sinks", [("q4", 0, 0), ("q4", 16, 2)])
def test_prefill_all_rewind_and_snapshots(kind, window, sinks, synth):
    path = synth("mini128")
    toks = np.random.default_rng(7).integers(0, 2048, 60).astype(np.int32)
    with qa.HipLlama.load(path, max_ctx=128) as m, qa.HipLlama.load(path, max_ctx=128) as r:
        for x in (m, r):
            x.set_cache(kind)
            x.set_window(window, sinks)
        m.prefill(toks[:50])
        steps = [m.step(int(t)) for t in toks[50:]]
        assert m.rewind(50)
        got = m.prefill_all(toks[50:])
        for a, b in zip(got, steps):
            np.testing.assert_array_equal(a, b)
        # a snapshot into another 4-bit model: the same cache
        s = m.snapshot()
        assert len(s) == 4 + 4 * 2 * 60 * 128
        r.restore(s)
        assert r.pos() == 60 and r.snapshot() == s
        np.testing.assert_array_equal(m.step(3), r.step(3))
        m.reset()
        assert len(m.snapshot()) == 4
        m.restore(np.int32(0).tobytes())
        assert m.pos() == 0
    # into an fp16 model, and an fp16 model's into a 4-bit one: layer 0's rows are what rounding makes of them
    with qa.HipLlama.load(path, max_ctx=128) as f, qa.HipLlama.load(path, max_ctx=128) as m:
        f.restore(s)
        assert f.snapshot() == s
        f.reset()
        f.prefill(toks)
        fs = f.snapshot()
        m.set_cache("q4")
        m.restore(fs)
        rows = torch.from_numpy(np.frombuffer(fs, np.float16, offset=4).copy()).view(2, 2, 60, 1, 128)
        got = torch.from_numpy(np.frombuffer(m.snapshot(), np.float16, offset=4).copy()).view(2, 2, 60, 1, 128)
        assert torch.equal(got.double(), held(rows.double()))
        want = Plain(path).logits(np.concatenate([toks, [9]]))[60]
        assert np.abs(m.step(9) - want).max() < 0.2 * np.abs(want).max()   # rounded rows, the model's own next token


def test_switching_back_leaves_the_default_as_it_was(synth):
    path = synth("mini")
    toks = np.random.default_rng(8).integers(0, 1000, 80).astype(np.int32)
    with qa.HipLlama.load(path, max_ctx=160) as a, qa.HipLlama.load(path, max_ctx=160) as b:
        b.set_cache("q4")
        b.prefill(toks)
        b.greedy_run(1, 4)
        with pytest.raises(qa.QphError, match="position 0"):
            b.set_cache("f16")
        b.reset()
        b.set_window(7, 1)
        b.set_cache("f16")
        b.prefill(toks)
        b.step(2)
        b.set_window(0)
        b.reset()
        np.testing.assert_array_equal(a.prefill(toks), b.prefill(toks))
        for t in (5, 6):
            np.testing.assert_array_equal(a.step(t), b.step(t))
        np.testing.assert_array_equal(a.greedy_run(3, 20), b.greedy_run(3, 20))
        np.testing.assert_array_equal(a.prefill_all(toks[:9]), b.prefill_all(toks[:9]))
        # the reference order too
        a.reset(), b.reset()
        a.set_order(1), b.set_order(1)
        np.testing.assert_array_equal(a.prefill(toks[:20]), b.prefill(toks[:20]))
        for f, words in ((lambda: b.set_window(5), "reference order"), (lambda: (b.reset(), b.set_cache("q4")), "reference order")):
            with pytest.raises(qa.QphError, match=words):
                f()


@pytest.mark.parametrize("chunk,few", [(24, ""), (7, "0"), (90, "100000")])
def test_modes_one_after_the_other(chunk, few, synth, monkeypatch):
    """each change finds scratch for its own kernels, whatever the modes before it needed"""
    monkeypatch.setenv("QPH_PF_CHUNK", str(chunk))
    monkeypatch.setenv("QPH_KV_FEW", few)
    path = synth("mini128")
    ref = Plain(path)
    toks = np.random.default_rng(13).integers(0, 2048, 100).astype(np.int32)
    with qa.HipLlama.load(path, max_ctx=3000) as m:
        for kind, window, sinks in (("q4", 0, 0), ("q4", 40, 3), ("f16", 40, 3), ("f16", 1000, 0), ("q4", 1000, 0), ("f16", 1000, 0), ("q4", 0, 0)):
            m.reset()
            m.set_cache(kind)
            m.set_window(window, sinks)
            got = m.prefill(toks[:98]), m.step(int(toks[98]))
            # over the cache's own values: of 100K rounded ones many lie next to a border of their codes, and a narrow window gives each weight
            want = ref.logits(toks[:99], kind, window, sinks, cached(m, ref))
            check(got[0], want[97], f"{kind} {window} prompt")
            check(got[1], want[98], f"{kind} {window} step")


def test_window_changes_during_a_conversation(synth):
    path = synth("mini")
    ref = Plain(path)
    toks = np.random.default_rng(9).integers(0, 1000, 64).astype(np.int32)
    with qa.HipLlama.load(path, max_ctx=128) as m:
        m.prefill(toks[:60])
        # one layer's window would not change what is in the cache; with two the rows of the layers above were made under the full view: only
        # a window that sees everything, and the way back, can be compared with the plain forward
        m.set_window(100, 0)
        check(m.step(int(toks[60])), ref.logits(toks[:61])[60], "wide window")
        m.set_window(0)
        check(m.step(int(toks[61])), ref.logits(toks[:62])[61], "no window")
        m.set_window(1 << 30, 1 << 30)
        check(m.step(int(toks[62])), ref.logits(toks[:63])[62], "widest window")


def test_refusals(synth):
    with qa.HipLlama.load(synth("mini"), max_ctx=64) as m:
        for f in (lambda: m.set_cache(qa.QPH_Q8), lambda: m.set_window(-1), lambda: m.set_window(4, -1)):
            with pytest.raises(qa.QphError):
                f()
        m.set_cache("q4")
        with pytest.raises(qa.QphError, match="fp16 cache"):
            m.set_order(1)
        with pytest.raises(qa.QphError, match="fused"):
            m.time_kernel(6, 1)
        m.prefill(np.arange(64, dtype=np.int32))
        with pytest.raises(qa.QphError, match="full"):
            m.step(1)
        ms, nbytes = m.time_kernel(5, 2)
        assert ms > 0 and nbytes == 9 / 8 * 65 * 128


def test_without_graphs(synth, monkeypatch):
    toks = np.random.default_rng(10).integers(0, 2048, 40).astype(np.int32)

    def run():
        with qa.HipLlama.load(synth("mini128"), max_ctx=64) as m:
            m.set_cache("q4")
            m.set_window(10, 2)
            return m.prefill(toks), m.step(4), m.greedy_run(5, 8)
    a = run()
    monkeypatch.setenv("QPH_NO_GRAPH", "1")
    for x, y in zip(a, run()):
        np.testing.assert_array_equal(x, y)
