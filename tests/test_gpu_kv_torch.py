"""KvCache beside torch's autograd: what the calls write counts as changed, and only that."""
import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv import F16, i32  # noqa: E402


@pytest.mark.parametrize("kind", ["q4", "f16"])
def test_versions_of_what_is_written(kind):
    c = qa.KvCache(kind, 1, 2, 64, 40)
    data = [c.data] if kind == "q4" else list(c.data)
    k, v, q = (torch.randn(1, 3, h, 64, device="cuda", dtype=F16) for h in (2, 2, 4))
    out, rk, rv, pos, lens = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k), i32([0]), i32([3])
    every = data + [k, v, q, out, rk, rv, pos, lens]

    def changed(f):
        before = [t._version for t in every]
        f()
        return [i for i, t in enumerate(every) if t._version != before[i]]
    m = len(data)
    assert changed(lambda: c.write(k, v, pos, lens=lens)) == list(range(m))
    assert changed(lambda: c.read(pos, 3, lens=lens, out=(rk, rv))) == [m + 4, m + 5]
    assert changed(lambda: c.attention(q, pos, lens=lens, out=out)) == [m + 3]
    assert changed(lambda: c.attention(q, pos, out=q)) == [m + 2]
    with pytest.raises(qa.QphError):
        c.attention(q, pos, out=out, window=-1)
    with torch.inference_mode():   # tensors without versions
        x = torch.zeros_like(q)
        c.attention(q, pos, out=x)
        c.write(k, v, pos)
    assert torch.equal(x, c.attention(q, pos))


def test_a_saved_result_that_is_written_over_is_noticed():
    c = qa.KvCache("f16", 1, 2, 64, 40)
    k, q, pos = torch.randn(1, 3, 2, 64, device="cuda", dtype=F16), torch.randn(1, 3, 4, 64, device="cuda", dtype=F16), i32([0])
    c.write(k, k, pos)
    w = torch.ones(64, device="cuda", dtype=F16, requires_grad=True)
    out = c.attention(q, pos)
    loss = (out * w).sum()
    loss.backward()
    loss = (out * w).sum()
    c.attention(q * 2, pos, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    loss = (c.data[0] * w).sum()   # the cache's own memory
    c.write(k, k, pos)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
