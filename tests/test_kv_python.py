"""KvCache's checks that need no GPU: a cache over CPU tensors gets as far as the check of their device."""
import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")


def cache(k, v, nseq, kv_heads, head_dim, ctx):
    return qa.KvCache("f16", nseq, kv_heads, head_dim, ctx, data=(k, v))


def f16(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


def bound(nseq=2, kv_heads=2, head_dim=64, ctx=40):
    """the compiled half over an address that is never read: CPU tensors are refused before anything is launched"""
    from qpack_amd.kvcache import _binding
    return _binding().Cache(qa.QPH_Q4, nseq, kv_heads, head_dim, ctx, 1 << 20, 0, 0, 0, 0, torch.zeros(1, dtype=torch.uint8))


def test_gradients_are_refused():
    c, x, pos = bound(), torch.zeros(2, 3, 2, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    g = torch.zeros(2, 3, 2, 64, dtype=torch.float16, requires_grad=True)
    calls = [lambda a: c.write(a, x, pos, None), lambda a: c.attention(a, x, pos, None, 0, 0, 0.0), lambda a: c.read(a, x, pos, None)]
    for f in calls:
        for a in (g, g * 2, g[:, :2]):
            with pytest.raises(qa.QphError, match="requires a gradient"):
                f(a)
            with torch.no_grad(), pytest.raises(qa.QphError, match="device"):   # taken as far as that
                f(a)
        with pytest.raises(qa.QphError, match="device"):
            f(g.detach())
    with pytest.raises(qa.QphError, match="requires a gradient"):
        cache(f16(3, 40, 2, 64).requires_grad_(), f16(3, 40, 2, 64), 3, 2, 64, 40)
    with pytest.raises(qa.QphError, match="requires a gradient"):
        cache(f16(3, 40, 2, 64), f16(3, 40, 2, 64).requires_grad_(), 3, 2, 64, 40)


def test_expanded_caches_are_refused():
    """one prefix shared by all sequences, one position by all: the C ABI takes a stride of 0 for a cache without gaps"""
    for x in (f16(1, 40, 2, 64).expand(3, -1, -1, -1), f16(3, 1, 2, 64).expand(-1, 40, -1, -1)):
        for k, v in ((x, x.clone(memory_format=torch.preserve_format)), (x, x)):
            with pytest.raises(qa.QphError, match="share memory|equal strides"):
                cache(k, v, 3, 2, 64, 40)
        with pytest.raises(qa.QphError, match="share memory"):
            cache(x, x, 3, 2, 64, 40)


def test_strides_of_single_axes_mean_nothing():
    k = f16(40 * 2 * 64 + 64)
    for shape, strides, more in (((1, 40, 2, 64), (0, 128, 64, 1), (7, 128, 64, 1)), ((2, 1, 2, 64), (1280, 0, 64, 1), (1280, 5, 64, 1)),
                                 ((2, 20, 1, 64), (1280, 64, 3, 1), (1280, 64, 0, 1)), ((1, 1, 1, 64), (0, 0, 0, 1), (9, 9, 9, 1))):
        with pytest.raises(qa.QphError, match="on a GPU"):   # taken as far as that
            cache(k.as_strided(shape, strides), k.as_strided(shape, more), shape[0], shape[2], 64, shape[1])
    for shape, a, b in (((2, 20, 1, 64), (1280, 64, 1, 1), (1344, 64, 1, 1)), ((1, 20, 2, 64), (0, 128, 64, 1), (0, 128, 0, 1))):
        with pytest.raises(qa.QphError, match="equal strides"):
            cache(k.as_strided(shape, a), k.as_strided(shape, b), shape[0], shape[2], 64, shape[1])


def test_a_binding_that_is_not_built_is_named(monkeypatch):
    import sys

    from qpack_amd import kvcache
    monkeypatch.setattr(kvcache, "_bind", None)
    monkeypatch.setitem(sys.modules, "qpack_amd._kvbind", None)
    monkeypatch.delattr(qa, "_kvbind", raising=False)
    with pytest.raises(qa.QphError, match="was not built"):
        kvcache._binding()


def test_tangents_are_refused():
    """forward mode: of what is read, of what is written and of the cache's own memory; also where no gradients are recorded, which leaves forward mode on"""
    from qpack_amd.kvcache import _binding
    from torch.autograd import forward_ad
    c, x, pos, t = bound(), torch.zeros(2, 3, 2, 64), torch.zeros(2, dtype=torch.int32), torch.zeros(9, 32)
    calls = [lambda a: c.write(a, x, pos, None), lambda a: c.read(a, x, pos, None), lambda a: c.attention(a, x, pos, None, 0, 0, 0.0), lambda a: c.attention(a, a, pos, None, 0, 0, 0.0),
             lambda a: c.append(a, x, x, x, pos, None, t, t, None, None, None, 1e-6), lambda a: c.attention_prefix(a, x, pos, None, 0.0, c, None), lambda a: _binding().logprobs(a[0, 0], None, 0)]
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for f in calls:
            for a in (d, d * 2, d[:, :2]):
                with pytest.raises(qa.QphError, match="tangent"):
                    f(a)
                with torch.no_grad(), pytest.raises(qa.QphError, match="tangent"):
                    f(a)
            with pytest.raises(qa.QphError, match="device|GPU"):   # taken as far as that
                f(forward_ad.unpack_dual(d).primal)
        memory = forward_ad.make_dual(f16(3, 40, 2, 64), f16(3, 40, 2, 64))
        for k, v in ((f16(3, 40, 2, 64), memory), (memory, f16(3, 40, 2, 64))):
            with pytest.raises(qa.QphError, match="tangent"):
                cache(k, v, 3, 2, 64, 40)
    with pytest.raises(qa.QphError, match="device|GPU"):
        calls[0](d)
