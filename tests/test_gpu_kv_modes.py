"""HipLlama with a 4-bit cache or a window: what changes around it, and what does not."""
import numpy as np
import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


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
