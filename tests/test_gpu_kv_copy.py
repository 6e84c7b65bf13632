"""KvCache.copy: copied positions hold the source's values, and what the copy does not write its own, to the bit."""
import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv import F32, i32  # noqa: E402


def cache(kind, S, G, D, ctx, gen, gaps=False):
    data = None
    if gaps and kind == "f16":   # positions and sequences further apart than they have to be
        data = tuple(torch.zeros(S, ctx + 3, G * D + 8, dtype=torch.float16, device="cuda").as_strided((S, ctx, G, D), ((ctx + 3) * (G * D + 8), G * D + 8, D, 1)) for _ in range(2))
    c = qa.KvCache(kind, S, G, D, ctx, data=data)
    k, v = (torch.randn(S, ctx, G, D, generator=gen).cuda() for _ in range(2))
    c.write(k, v, i32([0] * S))
    return c


def values(c):
    return torch.stack(c.read(i32([0] * c.nseq), c.ctx, dtype=F32))   # [K / V][sequence][position][head][dim]


def wanted(dst, src, index, pos, n, lens=None, seqs=None):
    """what dst holds after the copy, all reads before all writes"""
    was, new = values(src), values(dst)
    for b in range(dst.nseq):
        for t in range(n if lens is None else max(0, min(n, lens[b]))):
            s, p, i = seqs[b] if seqs else b, pos[b] + t, int(index[b][t])
            if pos[b] >= 0 and p < dst.ctx and 0 <= s < src.nseq and 0 <= i < src.ctx:
                new[:, b, p] = was[:, s, i]
    return new


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("D,G", [(64, 1), (128, 3)])
@pytest.mark.parametrize("S,n,pos", [(1, 1, [0]), (1, 1, [13]), (2, 5, [6, 9]), (3, 17, [0, 7, 30]), (2, 64, [0, 8]), (4, 100, [3, 0, 64, 1])])
def test_between_caches(kind, D, G, S, n, pos):
    print(f"copy {kind} {D} {G} {S} {n}", flush=True)
    gen = torch.Generator().manual_seed(n + D)
    src, dst = cache(kind, S + 1, G, D, 130, gen, gaps=True), cache(kind, S, G, D, max(pos) + n + 3, gen)
    for index in (torch.randint(0, 130, (S, n), generator=gen), torch.stack([torch.arange(n) + 8 * (b % 3) + (b & 1) for b in range(S)]), torch.arange(n).repeat(S, 1),
                  torch.full((S, n), 77)):
        seqs = [(b * 3 + 1) % (S + 1) for b in range(S)]
        want = wanted(dst, src, index, pos, n, seqs=seqs)
        dst.copy(index.int().cuda(), i32(pos), seqs=i32(seqs), source=src)
        assert torch.equal(values(dst), want)


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("D", [64, 128])
def test_within_a_cache_all_is_read_first(kind, D):
    """beams that change places, positions dropped, shifted either way, reversed"""
    gen = torch.Generator().manual_seed(D)
    S, G, ctx = 4, 2, 101
    c = cache(kind, S, G, D, ctx, gen, gaps=True)
    every = torch.arange(ctx)
    for index, pos, seqs in ((every.repeat(S, 1), [0] * S, [1, 2, 3, 0]), (every.repeat(S, 1), [0] * S, [2, 2, 0, 0]), (every[1::2].repeat(S, 1), [0] * S, None),
                             (every[:80].repeat(S, 1), [5, 1, 8, 21], None), (every[7:].repeat(S, 1), [0, 3, 7, 6], None), (every.flip(0).repeat(S, 1), [0] * S, [0, 0, 3, 2])):
        want = wanted(c, c, index, pos, index.shape[1], seqs=seqs)
        c.copy(index.int().cuda(), i32(pos), seqs=i32(seqs) if seqs else None)
        assert torch.equal(values(c), want)
    # sequences of one cache as two caches over one memory
    if kind == "f16":
        k, v = c.data
        a, b = qa.KvCache(kind, 3, G, D, ctx, data=(k[:3], v[:3])), qa.KvCache(kind, 3, G, D, ctx, data=(k[1:], v[1:]))
        want = wanted(a, b, every.repeat(3, 1), [0] * 3, ctx)
        a.copy(every.repeat(3, 1).int().cuda(), i32([0] * 3), source=b)
        assert torch.equal(values(a), want)


@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_fork_apart(kind):
    """one sequence's first positions into the others', without scratch; an expanded row of indices; then places within one record"""
    gen = torch.Generator().manual_seed(5)
    S, G, D, ctx, n = 5, 2, 128, 90, 71
    c = cache(kind, S, G, D, ctx, gen)
    index = torch.arange(n, dtype=torch.int32, device="cuda").unsqueeze(0).expand(S, n)
    pos, seqs = [-1, 0, 0, 0, 0], [0] * S
    want = wanted(c, c, index.cpu(), pos, n, seqs=seqs)
    c.copy(index, i32(pos), seqs=i32(seqs), apart=True)
    assert torch.equal(values(c), want)
    index = torch.tensor([[24, 26, 28]] * S)   # to 25 .., of which none is read
    index[:, 1] = 30
    want = wanted(c, c, index, [25] * S, 3)
    c.copy(index.int().cuda(), i32([25] * S), apart=False)
    assert torch.equal(values(c), want)
    index = torch.tensor([[40, 41, 44]] * S)
    want = wanted(c, c, index, [45] * S, 3)
    c.copy(index.int().cuda(), i32([45] * S), apart=True)
    assert torch.equal(values(c), want)


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("shared", [False, True])
def test_what_takes_no_part(kind, shared):
    gen = torch.Generator().manual_seed(6)
    S, G, D, ctx, n = 6, 1, 64, 50, 12
    c = cache(kind, S, G, D, ctx, gen)
    src = c if shared else cache(kind, 4, G, D, 30, gen)
    index = torch.randint(0, 30, (S, n), generator=gen)
    index[0, 3], index[0, 5], index[1, 0], index[2, 7] = -1, src.ctx, 2 ** 31 - 1, -2 ** 31
    pos, lens, seqs = [3, 0, 45, -1, 50, 8], [n, n, n, n, n, 5], [1, 3, 0, 2, 1, -1]
    for seqs in (seqs, [1, 3, 0, 2, 1, 2], [src.nseq, 3, 0, 2, 1, 2 ** 31 - 1]):
        want = wanted(c, src, index, pos, n, lens=lens, seqs=seqs)
        c.copy(index.int().cuda(), i32(pos), lens=i32(lens), seqs=i32(seqs), source=src)
        assert torch.equal(values(c), want)
    want = values(c)
    c.copy(index.int().cuda()[:, :0], i32(pos), source=src)
    c.copy(index.int().cuda(), i32(pos), lens=i32([0, -3, 0, 0, 0, 0]), source=src)
    assert torch.equal(values(c), want)


@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_graph_replays(kind):
    gen = torch.Generator().manual_seed(8)
    S, G, D, ctx = 3, 2, 64, 64
    c, e = cache(kind, S, G, D, ctx, gen), None
    e = qa.KvCache(kind, S, G, D, ctx, data=tuple(x.clone() for x in c.data) if kind == "f16" else c.data.clone())
    index, pos, seqs = torch.arange(ctx, dtype=torch.int32, device="cuda").repeat(S, 1), i32([0] * S), i32([1, 2, 0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):   # (before the capture, on another stream)
        c.copy(index, pos, seqs=seqs)
    torch.cuda.current_stream().wait_stream(s)
    e.copy(index, pos, seqs=seqs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.copy(index, pos, seqs=seqs)
    for sq, shift in (([1, 2, 0], 0), ([0, 0, 1], 3), ([2, 1, 0], 9)):
        seqs.copy_(i32(sq))
        pos.copy_(i32([shift] * S))
        g.replay()
        e.copy(index, pos, seqs=seqs)
        torch.cuda.synchronize()
        assert torch.equal(values(c), values(e))


def test_refusals():
    c = qa.KvCache("q4", 2, 2, 64, 40)
    index, pos = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), i32([0, 1])
    for bad in (qa.KvCache("f16", 2, 2, 64, 40), qa.KvCache("q4", 2, 1, 64, 40), qa.KvCache("q4", 2, 2, 128, 40)):
        with pytest.raises(qa.QphError, match="same kind"):
            c.copy(index, pos, source=bad)
    for bad in (index.long(), index[:1], index[0], torch.zeros(2, 6, dtype=torch.int32, device="cuda")[:, ::2]):
        with pytest.raises(qa.QphError, match="index"):
            c.copy(bad, pos)
    with pytest.raises(qa.QphError, match="device"):
        c.copy(index.cpu(), pos)
    for bad in (pos.long(), pos[:1], None):
        with pytest.raises(qa.QphError, match="pos"):
            c.copy(index, bad)
        if bad is not None:
            with pytest.raises(qa.QphError, match="seqs"):
                c.copy(index, pos, seqs=bad)
            with pytest.raises(qa.QphError, match="lens"):
                c.copy(index, pos, lens=bad)


@pytest.mark.parametrize("D", [64, 128])
def test_records_of_many_sequences(D):
    """more records than a wave each: in order, picked, shifted, and back by way of scratch"""
    gen = torch.Generator().manual_seed(D + 1)
    S, G, ctx, n = 90, 8, 270, 250   # 90 x 8 x 32 records
    src, dst = cache("q4", S, G, D, ctx, gen), cache("q4", S, G, D, ctx, gen)
    was, new = values(src), values(dst)
    b = torch.arange(S)[:, None]
    for index, pos in ((torch.arange(n).repeat(S, 1), b[:, 0] % 9), (torch.randint(0, ctx, (S, n), generator=gen), b[:, 0] % 5), (torch.arange(n).repeat(S, 1) + b % 3, b[:, 0] % 2 * 8)):
        at = (pos[:, None] + torch.arange(n)).cuda()
        new[:, b.cuda(), at] = was[:, b.cuda(), index.cuda()]
        dst.copy(index.int().cuda(), pos.int().cuda(), source=src)
        assert torch.equal(values(dst), new)
        seqs = torch.randint(0, S, (S,), generator=gen)
        new[:, b.cuda(), at] = was[:, seqs[:, None].cuda(), index.cuda()]
        dst.copy(index.int().cuda(), pos.int().cuda(), seqs=seqs.int().cuda(), source=src)
        assert torch.equal(values(dst), new)
    new[:, b.cuda(), torch.arange(n, device="cuda") + 7] = new[:, b.cuda(), torch.arange(n, device="cuda")]
    dst.copy(torch.arange(n, dtype=torch.int32, device="cuda").expand(S, n), torch.full((S,), 7, dtype=torch.int32, device="cuda"))
    assert torch.equal(values(dst), new)
