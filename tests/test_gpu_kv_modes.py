"""HipLlama with a 4-bit cache or a window: what changes around it, and what does not."""
import numpy as np
import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv_model import ATOL, Plain, cached, check, held  # noqa: E402


@pytest.mark.parametrize("few", ["0", "100000"])
def test_the_environment_after_load_changes_nothing(few, synth, monkeypatch):
    """the kernels are chosen as the scratch was sized"""
    toks = np.random.default_rng(3).integers(0, 2048, 120).astype(np.int32)
    monkeypatch.delenv("QPH_KV_FEW", raising=False)
    with qa.HipLlama.load(synth("mini128"), max_ctx=4000) as m:
        m.set_cache("q4")
        want = [m.prefill(toks[:n]) for n in (1, 7, 112)] + [m.step(5)]
        m.reset()
        monkeypatch.setenv("QPH_KV_FEW", few)
        got = [m.prefill(toks[:n]) for n in (1, 7, 112)] + [m.step(5)]
        for a, b in zip(want, got):
            np.testing.assert_array_equal(a, b)


def free():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("pos", [1, 16383, 16384, 16385, 20003, 33000])
def test_snapshots_longer_than_a_slice(pos, synth):
    """mini128: 512 bytes a position and layer, slices of 8 MiB"""
    rows = torch.randn(2, 2, pos, 1, 128, generator=torch.Generator().manual_seed(pos)).half()
    s = np.int32(pos).tobytes() + rows.numpy().tobytes()
    with qa.HipLlama.load(synth("mini128"), max_ctx=33001) as m:
        m.set_cache("q4")
        m.restore(s)
        assert m.pos() == pos
        got = torch.from_numpy(np.frombuffer(m.snapshot(), np.float16, offset=4).copy()).view_as(rows)
        assert torch.equal(got.double(), held(rows.double()))
        m.step(3)


def test_a_4_bit_cache_takes_9_of_32_parts(synth):
    """and 8 MiB of rows for snapshots, the attention's scratch, and what the allocator rounds up"""
    ctx, mib = 1 << 18, 1 << 20
    f16 = 2 * 2 * ctx * 128 * 2
    with qa.HipLlama.load(synth("mini128"), max_ctx=ctx) as m:
        before = free()
        m.set_cache("q4")
        gained = free() - before
        assert gained >= f16 * 23 // 32 - 40 * mib, f"{gained / mib:.0f} MiB of {f16 / mib:.0f}"
        m.set_cache("f16")
        assert abs(free() - before) <= 40 * mib


def test_loaded_with_a_4_bit_cache(synth):
    """as set afterwards, without the fp16 cache's memory at any time"""
    ctx, mib, toks = 1 << 18, 1 << 20, np.random.default_rng(5).integers(0, 2048, 60).astype(np.int32)
    f16 = 2 * 2 * ctx * 128 * 2
    used = {}
    for kind in ("f16", "q4"):
        before = free()
        with qa.HipLlama.load(synth("mini128"), max_ctx=ctx, cache=kind) as m:
            used[kind] = before - free()
            if kind == "f16":
                m.set_cache("q4")
                want = m.prefill(toks), m.step(3), m.greedy_run(4, 9)
            else:
                for a, b in zip(want, (m.prefill(toks), m.step(3), m.greedy_run(4, 9))):
                    np.testing.assert_array_equal(a, b)
                m.reset()
                m.set_cache("f16")
                default = m.prefill(toks), m.step(3)
                m.set_order(1)
    assert used["f16"] - used["q4"] >= f16 * 23 // 32 - 40 * mib, {k: v // mib for k, v in used.items()}
    with qa.HipLlama.load(synth("mini128"), max_ctx=ctx) as m:
        for a, b in zip(default, (m.prefill(toks), m.step(3))):
            np.testing.assert_array_equal(a, b)


def forward(ref, toks, seen, kind, cache=None):
    """every position's logits in 64 bits, where row t of the mask `seen` is what token t attends to: what later tokens find of it in the cache
    depends on the mask in force when it ran.  cache: the values that the attention reads, each layer's (K, V), in place of the rounded rows: a
    4-bit code moves by a whole step where the path's fp32 key and the 64-bit one lie on two sides of a border, which a narrow window
    does not average out.  They are to lie within half a step of the rows (the scale's 2^-9 of 7 steps more) and 2e-3 for the path's own error"""
    c, w, n = ref.c, ref.w, len(toks)
    H, G, D = c["num_attention_heads"], c["num_key_value_heads"], c["head_dim"]
    norm = lambda x, g: x / torch.sqrt((x * x).mean(-1, keepdim=True) + c["rms_norm_eps"]) * g   # noqa: E731
    ang = torch.arange(n).double()[:, None] / c["rope_theta"] ** (torch.arange(D // 2).double() * 2 / D)
    cs, sn = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    rope = lambda x: torch.cat([x[..., :D // 2] * cs - x[..., D // 2:] * sn, x[..., D // 2:] * cs + x[..., :D // 2] * sn], -1)   # noqa: E731
    x = w["embed"][torch.from_numpy(np.asarray(toks)).long()]
    for i in range(c["num_hidden_layers"]):
        g = lambda s: w[f"layers.{i}.{s}"]   # noqa: E731
        y = norm(x, g("attn_norm"))
        q, k, v = (y @ g("w" + s).T + (g("b" + s) if c["qkv_bias"] else 0) for s in "qkv")
        q, k, v = rope(q.view(n, H, D)), rope(k.view(n, G, D)), v.view(n, G, D)
        if cache is not None:
            for mine, theirs in zip((k, v), cache[i]):
                step = mine.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) / 7
                assert bool(((theirs - mine).unflatten(-1, (-1, 32)).abs() <= step * (0.5 + 2.0 ** -6) + 2e-3).all()), f"layer {i}: a cached row"
            k, v = cache[i]
        else:
            k, v = (held(k), held(v)) if kind == "q4" else (k.half().double(), v.half().double())
        a = torch.matmul(q.transpose(0, 1), k.repeat_interleave(H // G, 1).permute(1, 2, 0)) / D ** 0.5
        a = torch.softmax(a.masked_fill(~seen, -torch.inf), -1)
        x = x + torch.matmul(a, v.repeat_interleave(H // G, 1).transpose(0, 1)).transpose(0, 1).reshape(n, H * D) @ g("wo").T
        y = norm(x, g("ffn_norm"))
        u = y @ g("w_gate").T
        x = x + (u * torch.sigmoid(u) * (y @ g("w_up").T)) @ g("w_down").T
    return (norm(x, w["final_norm"]) @ (w["embed"] if c["tie_embeddings"] else w["lm_head"]).T).numpy()


@pytest.mark.parametrize("cfg,kind", [("mini", "f16"), ("mini128", "f16"), ("mini", "q4")])
def test_narrowing_and_widening_a_window(cfg, kind, synth):
    """each change takes effect for the next call, in steps, greedy steps and prompts, and every position stays in the cache"""
    ref = Plain(synth(cfg))
    toks = np.random.default_rng(9).integers(0, 1000, 110).astype(np.int32)
    phases = [(60, 0, 0), (66, 9, 2), (70, 30, 0), (82, 5, 1), (86, 0, 0), (98, 12, 4), (104, 1, 0), (110, 0, 0)]   # up to which token, window, sinks
    P, p = torch.arange(110)[:, None], torch.arange(110)[None]
    seen, full = p <= P, p <= P
    at = 0
    for upto, window, sinks in phases:
        if window:
            seen[at:upto] &= (p > P[at:upto] - window) | (p < sinks)
        at = upto
    got, modes = {}, {}
    with qa.HipLlama.load(synth(cfg), max_ctx=128, cache=kind) as m:
        at = 0
        for upto, window, sinks in phases:
            m.set_window(window, sinks)
            if upto - at > 8:   # a prompt; the rest by steps
                got[upto - 1] = m.prefill(toks[at:upto])
            else:
                got.update((i, m.step(int(toks[i]))) for i in range(at, upto))
            modes.update((i, (window, sinks)) for i in range(at, upto))
            at = upto
        held_rows = cached(m, ref) if kind == "q4" else None
    want, plain = forward(ref, toks, seen, kind, held_rows), forward(ref, toks, full, kind)
    for i, row in got.items():
        check(row, want[i], f"token {i}, window and sinks {modes[i]}")
        if modes[i][0]:
            assert np.abs(want - plain)[i].max() > 3 * ATOL   # the window shows


def test_an_error_is_not_reported_again(synth):
    """a context whose cache no card holds (512 GiB): the load fails, and the next one's launches are not told of it"""
    toks = np.arange(40, dtype=np.int32)
    with qa.HipLlama.load(synth("mini128"), max_ctx=64) as m:
        want = m.prefill(toks)
        with pytest.raises(qa.QphError, match="memory"):
            qa.HipLlama.load(synth("mini128"), max_ctx=1 << 30)
        m.reset()
        np.testing.assert_array_equal(m.prefill(toks), want)
        with pytest.raises(qa.QphError, match="memory"):
            qa.HipLlama.load(synth("mini128"), max_ctx=1 << 30)
    with qa.HipLlama.load(synth("mini128"), max_ctx=64) as m:
        np.testing.assert_array_equal(m.prefill(toks), want)


def test_a_load_that_fails_gives_its_memory_back(synth):
    with qa.HipLlama.load(synth("mini128"), max_ctx=64) as m:
        m.prefill(np.arange(40, dtype=np.int32))
    before = free()
    for _ in range(8):
        with pytest.raises(qa.QphError, match="memory"):
            qa.HipLlama.load(synth("mini128"), max_ctx=1 << 30)
    assert before - free() <= 4 << 20
