"""HipLlama with a 4-bit cache or a window: what changes around it, and what does not."""
import numpy as np
import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv_model import held  # noqa: E402


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
