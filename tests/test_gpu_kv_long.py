"""append, copy and attention behind a prefix in caches whose offsets pass 32 bits (in bytes and, fp16, in elements).  Tolerances: test_gpu_kv's, over the positions that are not zero."""
import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv import F32, check_rows, i32  # noqa: E402

G, D = 8, 128
CTX = {"f16": 2 ** 21 + 4096, "q4": 2 ** 22}   # K of a sequence: 4.3 GB; records of one: 4.8 GB


@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_append_and_copy_at_the_end(kind):
    ctx = CTX[kind]
    c = qa.KvCache(kind, 2, G, D, ctx)
    gen = torch.Generator(device="cuda").manual_seed(1)
    n = 21
    q, k, v = (torch.randn(2, n, h, D, generator=gen, device="cuda").half() for h in (16, G, G))
    P = [ctx - n - 3, ctx - n]
    none = torch.zeros(1, 0, device="cuda")
    angle = torch.rand(64, D // 2, generator=gen, device="cuda")
    small = qa.KvCache(kind, 2, G, D, 64)
    for tables in ((angle.cos(), angle.sin()), (none.expand(64, 0), none.expand(64, 0))):
        at = i32([7, 11])
        got = c.append(q, k, v, i32(P), *tables, at=at)
        want = small.append(q, k, v, i32([x % 8 for x in P]), *tables, at=at)
        assert torch.equal(got, want)
        for x, y in zip(c.read(i32(P), n, dtype=F32), small.read(i32([x % 8 for x in P]), n, dtype=F32)):
            assert torch.equal(x, y)
    # within the cache, from the end of one sequence to the other's, and to another's start and back
    index = torch.arange(n, device="cuda", dtype=torch.int32)
    index = torch.stack([P[1] + index.flip(0), P[0] + index])
    rows = c.read(i32(P), n, dtype=F32)
    c.copy(index, i32([ctx - 2 * n - 30, ctx - 2 * n - 29]), seqs=i32([1, 0]))
    new = c.read(i32([ctx - 2 * n - 30, ctx - 2 * n - 29]), n, dtype=F32)
    for x, y in zip(new, rows):
        assert torch.equal(x[0], y[1].flip(0)) and torch.equal(x[1], y[0])
    small.copy(index, i32([2, 5]), source=c, seqs=i32([1, 0]))
    for x, y in zip(small.read(i32([2, 5]), n, dtype=F32), rows):
        assert torch.equal(x[0], y[1].flip(0)) and torch.equal(x[1], y[0])
    c.copy(torch.arange(2, 2 + n, device="cuda", dtype=torch.int32).expand(2, n), i32([ctx - 100, ctx - 99]), source=small, seqs=i32([0, 0]))
    for x, y in zip(c.read(i32([ctx - 100, ctx - 99]), n, dtype=F32), rows):
        assert torch.equal(x[0], y[1].flip(0)) and torch.equal(x[1], y[1].flip(0))


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("S", [2, 40])
def test_prefix_of_millions(kind, S):
    """keys of zeros but for the last 300 positions of the prefix, which have nearly all of the weight"""
    ctx = CTX[kind]
    gen = torch.Generator(device="cuda").manual_seed(2)
    L, m = ctx - 5, 300
    p, c = qa.KvCache(kind, 1, G, D, ctx), qa.KvCache(kind, S, G, D, 8)
    k0, v0, k, v = (torch.randn(s, t, G, D, generator=gen, device="cuda").half() for s, t in ((1, m), (1, m), (S, 5), (S, 5)))
    u = torch.randn(G, D, generator=gen, device="cuda")
    u = u / u.norm(dim=-1, keepdim=True) * D ** 0.5   # (each head's keys there have a large part along u, as the queries do)
    p.write(k0 + 4 * u.half(), v0, i32([L - m]))
    c.write(k + 4 * u.half(), v, i32([0] * S))
    q = (0.25 * torch.randn(S, 1, 2 * G, D, generator=gen, device="cuda") + 2 * u.repeat_interleave(2, 0)).half()
    out = c.attention(q, i32([4] * S), prefix=p, prefix_len=i32([L]))
    K0, V0 = (x[0].double().cpu() for x in p.read(i32([L - m]), m, dtype=F32))
    K, V = (x.double().cpu() for x in c.read(i32([0] * S), 5, dtype=F32))
    # the zeros' share: 2^22 e^(0 - s) against m e^s', scores of 8 sqrt(D) = 90 and more
    for b in range(0, S, 13):
        check_rows(out[b], q[b], torch.cat([K0, K[b]]), torch.cat([V0, V[b]]), m + 4)
