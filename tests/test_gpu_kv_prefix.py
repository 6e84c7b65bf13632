"""KvCache.attention behind a common prefix, against plain 64-bit arithmetic over the prefix's positions and the sequence's own.  Tolerances: those of
test_gpu_kv, whose formula the prefix and own positions together are (their two sums are joined in fp32, as splits are)."""
import math

import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv import F16, F32, TYPES, check_rows, filled, i32, route  # noqa: E402, F401


def both(prefix, own, L, b):
    return torch.cat([prefix[0, :L], own[b]])


# kind, hd, kv heads, rep, n, prefix, pasts, lens
CASES = [
    ("f16", 128, 2, 4, 1, 1, [0], None), ("q4", 64, 1, 7, 1, 8, [3, 0], None), ("f16", 64, 2, 7, 1, 700, [90, 0, 31, 5], None), ("q4", 128, 1, 4, 1, 1500, [40, 100, 7], None),
    ("f16", 128, 1, 1, 1, 33, [2], None), ("q4", 128, 1, 8, 1, 4100, [0], None), ("f16", 64, 1, 16, 3, 65, [1100, 7], [3, 1]), ("q4", 64, 2, 2, 5, 257, [0, 9, 700], [5, 2, 4]),
    # many columns: 256 a workgroup, the last one ragged, tokens of several sequences in one
    ("f16", 128, 1, 4, 1, 900, [5] * 70, None), ("q4", 128, 2, 3, 1, 300, list(range(90)), None), ("f16", 64, 1, 5, 40, 130, [0, 300, 9], [40, 11, 25]), ("q4", 64, 1, 8, 66, 64, [513], None),
    ("f16", 128, 1, 2, 150, 1000, [0, 64], [150, 3]), ("q4", 128, 1, 7, 13, 63, [0] * 7, [13, 1, 2, 0, 13, 6, 7]),
    # own columns in several chunks of k_kv_few for each of many sequences
    ("q4", 64, 5, 2, 20, 200, list(range(40)), None), ("f16", 128, 3, 3, 17, 70, [11] * 64, [1 + i % 17 for i in range(64)]),
]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind,hd,G,rep,n,L,pasts,lens", CASES)
def test_prefix(kind, hd, G, rep, n, L, pasts, lens, type, route):
    print(f"prefix {kind} hd {hd} kv heads {G} rep {rep} n {n} prefix {L} sequences {len(pasts)} {type}", flush=True)
    gen = torch.Generator().manual_seed(n + L)
    S, ctx, live = len(pasts), max(pasts) + n + 3, lens or [n] * len(pasts)
    p, K0, V0 = filled(kind, 1, G, hd, L + 9, [L + 9], gen)   # (positions behind the prefix are another text's)
    c, K, V = filled(kind, S, G, hd, ctx, [a + m for a, m in zip(pasts, live)], gen)
    q = (torch.randn(S, n, G * rep, hd, generator=gen) * 1.5).to(TYPES[type]).cuda()
    out = torch.full_like(q, 55.)
    c.attention(q, i32(pasts), lens=i32(lens) if lens else None, prefix=p, prefix_len=i32([L]), out=out)
    for b in range(S):
        if live[b] and (S < 10 or b % 9 == 0):
            check_rows(out[b, :live[b]], q[b, :live[b]], both(K0, K, L, b), both(V0, V, L, b), L + pasts[b])
        assert bool((out[b, live[b]:] == 55).all())


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("n", [1, 30])
@pytest.mark.parametrize("ctx", [300, 1500])   # (of few positions a workgroup takes all, of more their sums are joined: here and below)
def test_lengths_of_the_prefix(kind, n, ctx, route):
    """none, negative (none), past the cache's end (all of it), not given (all of it); a length that changes between replays"""
    gen = torch.Generator().manual_seed(3)
    G, rep, D = 2, 4, 64
    p, K0, V0 = filled(kind, 1, G, D, ctx, [ctx], gen)
    c, K, V = filled(kind, 2, G, D, 100, [70, 70], gen)
    q, pos = torch.randn(2, n, G * rep, D, generator=gen).half().cuda(), i32([70 - n, 12])
    length, got = i32([5]), torch.zeros_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.attention(q, pos, prefix=p, prefix_len=length, out=got)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.attention(q, pos, prefix=p, prefix_len=length, out=got)
    for given, L in ((i32([0]), 0), (i32([-7]), 0), (i32([ctx + 1]), ctx), (i32([2 ** 31 - 1]), ctx), (None, ctx), (i32([17]), 17), (i32([256]), 256)):
        out = c.attention(q, pos, prefix=p, prefix_len=given)
        for b in range(2):
            check_rows(out[b], q[b], both(K0, K, L, b), both(V0, V, L, b), L + int(pos[b]))
        length.copy_(given if given is not None else i32([ctx]))
        got.fill_(9)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, out)


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 21])
@pytest.mark.parametrize("L", [400, 1100])
def test_strides_absent_sequences_over_q_and_padding(kind, type, n, L, route):
    gen = torch.Generator().manual_seed(8)
    S, G, rep, D = 6, 2, 4, 64
    ctx = 120
    pasts, lens = [100 - n, 7, -1, 40, ctx - n // 2, ctx], [n, max(1, n // 2), n, 0, n, n]
    T = [min(ctx, max(0, a) + m) if a >= 0 else 0 for a, m in zip(pasts, lens)]
    p, K0, V0 = filled(kind, 1, G, D, L, [L], gen)
    c, K, V = filled(kind, S, G, D, ctx, T, gen)
    x = torch.randn(S, G * rep, n, D + 3, generator=gen).cuda().to(TYPES[type])
    q = x[..., 3:].transpose(1, 2)
    base = torch.full((S, n, G * rep, D + 2), 55., device="cuda", dtype=TYPES[type])
    out = base[..., :D]
    c.attention(q, i32(pasts), lens=i32(lens), prefix=p, out=out)
    plain = q.contiguous()
    c.attention(plain, i32(pasts), lens=i32(lens), prefix=p, out=plain)
    live = [max(0, min(m, ctx - a)) if a >= 0 else 0 for a, m in zip(pasts, lens)]
    for b, m in enumerate(live):
        if m:
            check_rows(out[b, :m], q[b, :m], both(K0, K, L, b), both(V0, V, L, b), L + pasts[b])
        assert torch.equal(plain[b, :m], out[b, :m]) and torch.equal(plain[b, m:], q[b, m:])
        assert bool((out[b, m:] == 55).all())
    assert bool((base[..., D:] == 55).all())
    # what rows that take no part hold changes no bit
    for bad in (0., math.nan, math.inf, 6e4):
        y = q.contiguous()
        for b, m in enumerate(live):
            y[b, m:] = bad
        again = c.attention(y, i32(pasts), lens=i32(lens), prefix=p)
        for b, m in enumerate(live):
            assert torch.equal(again[b, :m], out[b, :m])


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("room", [200, 1300])
def test_unseen_memory_and_not_finite_values(kind, room, route):
    """NaN behind the prefix and behind the tokens changes nothing; one in the prefix reaches every sequence"""
    gen = torch.Generator().manual_seed(4)
    G, rep, D, L = 1, 4, 128, 77
    p, K0, V0 = filled(kind, 1, G, D, room, [L], gen)
    c, K, V = filled(kind, 3, G, D, 64, [20, 20, 20], gen)
    bad = torch.full((1, room - L, G, D), math.nan, device="cuda")
    p.write(bad, bad, i32([L]))
    bad = torch.full((3, 44, G, D), math.inf, device="cuda")
    c.write(bad, bad, i32([20] * 3))
    q, pos = torch.randn(3, 2, G * rep, D, generator=gen).half().cuda(), i32([18, 18, 5])
    out = c.attention(q, pos, prefix=p, prefix_len=i32([L]))
    for b in range(3):
        check_rows(out[b], q[b], both(K0, K, L, b), both(V0, V, L, b), L + int(pos[b]))
    k, v = p.read(i32([30]), 1, dtype=F32)
    v[..., 5] = math.nan
    p.write(k, v, i32([30]))
    out = c.attention(q, pos, prefix=p, prefix_len=i32([L]))
    dims = torch.zeros(D, dtype=torch.bool, device="cuda")
    dims[:32 if kind == "q4" else 0] = True
    dims[5] = True
    assert bool(torch.isnan(out[..., dims]).all()) and bool(torch.isfinite(out[..., ~dims]).all())


@pytest.mark.parametrize("room", [50, 1100])
def test_loud_prefix_and_loud_own_positions(room):
    """one part's scores far above the other's: its weights are all there is, and nothing overflows"""
    gen = torch.Generator().manual_seed(5)
    D, L = 64, 50
    for mine, theirs in ((40., 0.1), (0.1, 40.)):
        p, c = qa.KvCache("f16", 1, 1, D, room), qa.KvCache("f16", 1, 1, D, 10)
        k0, v0, k, v = (torch.randn(1, m, 1, D, generator=gen).half() for m in (L, L, 10, 10))
        k0, k = k0 * theirs, k * mine
        p.write(k0.cuda(), v0.cuda(), i32([0]))
        c.write(k.cuda(), v.cuda(), i32([0]))
        q = torch.randn(1, 1, 4, D, generator=gen).float().cuda()
        out = c.attention(q, i32([9]), prefix=p, prefix_len=i32([L]))
        check_rows(out[0], q[0], torch.cat([k0[0], k[0]]).double(), torch.cat([v0[0], v[0]]).double(), L + 9)


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("n,rep", [(1, 4), (30, 4)])
def test_scratch_streams_and_graphs(kind, n, rep):
    """scratch with anything in it; two graphs and an eager call at once, replayed several times"""
    import ctypes as C

    from qpack_amd._lib import KvC, RowsC, lib
    gen = torch.Generator().manual_seed(12)
    G, D, L, S = 2, 128, 1000, 3
    p, K0, V0 = filled(kind, 1, G, D, L, [L], gen)
    c, K, V = filled(kind, S, G, D, 90, [90] * S, gen)
    q, pos = torch.randn(S, n, G * rep, D, generator=gen).half().cuda(), i32([90 - n, 50, 3])
    want = c.attention(q, pos, prefix=p)
    for b in range(S):
        check_rows(want[b], q[b], both(K0, K, L, b), both(V0, V, L, b), L + int(pos[b]))

    def handle(x):
        t = (x.data, x.data) if kind == "q4" else x.data
        return KvC(x.kind, x.nseq, G, D, x.ctx, t[0].data_ptr(), t[1].data_ptr())
    kc, kp, r = handle(c), handle(p), RowsC(q.data_ptr(), qa.QPH_F16, q.stride(0), q.stride(1), q.stride(2))
    size = C.c_int64()
    qa._lib.check(lib().qph_kv_attention_prefix_work(C.byref(kc), C.byref(kp), qa.QPH_F16, G * rep, n, C.byref(size)))
    assert size.value > 0
    for fill in (255, 0, 127):
        work, o = torch.full((size.value + 64,), fill, dtype=torch.uint8, device="cuda"), torch.empty_like(q)
        qa._lib.check(lib().qph_kv_attention_prefix(C.byref(kc), C.byref(kp), None, C.byref(r), C.byref(RowsC(o.data_ptr(), qa.QPH_F16, q.stride(0), q.stride(1), q.stride(2))), G * rep, n,
                                                    pos.data_ptr(), None, 0.0, work.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert bool((work[size.value:] == fill).all()) and torch.equal(o, want)
    other = torch.randn(S, n, G * rep, D, generator=gen).half().cuda()
    want2 = c.attention(other, pos, prefix=p)
    torch.cuda.synchronize()
    outs, graphs = [torch.empty_like(q) for _ in range(2)], []
    for x, o in zip((q, other), outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.attention(x, pos, prefix=p, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for o in outs:
            o.fill_(9)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = c.attention(q, pos, prefix=p)
        torch.cuda.synchronize()
        assert torch.equal(eager, want) and torch.equal(outs[0], want) and torch.equal(outs[1], want2)


def test_refusals():
    c, p = qa.KvCache("f16", 2, 2, 64, 40), qa.KvCache("f16", 1, 2, 64, 30)
    q, pos = torch.zeros(2, 3, 4, 64, device="cuda", dtype=F16), i32([0, 1])
    for bad in (qa.KvCache("f16", 2, 2, 64, 30), qa.KvCache("f16", 1, 1, 64, 30), qa.KvCache("f16", 1, 2, 128, 30), qa.KvCache("q4", 1, 2, 64, 30)):
        with pytest.raises(qa.QphError, match="prefix must be"):
            c.attention(q, pos, prefix=bad)
    for window, sinks in ((5, 0), (5, 2), (0, 3)):
        with pytest.raises(qa.QphError, match="exclude"):
            c.attention(q, pos, prefix=p, window=window, sinks=sinks)
    for bad in (i32([1, 2]), i32([1]).long(), i32([1]).cpu(), 5):
        with pytest.raises(qa.QphError, match="prefix_len"):
            c.attention(q, pos, prefix=p, prefix_len=bad)
    with pytest.raises(qa.QphError, match="without a prefix"):
        c.attention(q, pos, prefix_len=i32([3]))
    with pytest.raises(qa.QphError, match="multiple of kv_heads"):
        c.attention(q[:, :, :3], pos, prefix=p)
    with pytest.raises(qa.QphError, match="same type"):
        c.attention(q, pos, prefix=p, out=q.float())
    assert c.attention(q[:, :0], pos, prefix=p).shape == (2, 0, 4, 64)


def test_more_rows_than_a_grid_is_wide():
    gen = torch.Generator().manual_seed(6)
    n, rep, D, L = 8200, 65, 128, 30   # 8 rows a workgroup, 65536 workgroups side by side
    p, K0, V0 = filled("f16", 1, 1, D, L, [L], gen)
    c, K, V = filled("f16", 1, 1, D, n, [n], gen)
    q = torch.randn(1, n, rep, D, generator=gen).half().cuda()
    out = c.attention(q, i32([0]), prefix=p)
    for t in (0, 4000, 8065, 8066, n - 1):
        check_rows(out[0, t:t + 1], q[0, t:t + 1], both(K0, K, L, 0)[:L + t + 1], both(V0, V, L, 0)[:L + t + 1], L + t)


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_many_sequences_of_one_token(kind, type):
    """more workgroups of few own columns than the launch with the prefix's many columns takes"""
    gen = torch.Generator().manual_seed(12)
    S, G, rep, D, L = 270, 4, 2, 64, 333
    pasts = [i % 37 for i in range(S)]
    p, K0, V0 = filled(kind, 1, G, D, L, [L], gen)
    c, K, V = filled(kind, S, G, D, 40, [a + 1 for a in pasts], gen)
    q = torch.randn(S, 1, G * rep, D, generator=gen).to(TYPES[type]).cuda()
    out = c.attention(q, i32(pasts), prefix=p)
    for b in range(0, S, 7):
        check_rows(out[b], q[b], both(K0, K, L, b), both(V0, V, L, b), L + pasts[b])


def test_more_workgroups_than_a_grid_is_wide(monkeypatch):
    monkeypatch.setenv("QPH_KV_FEW", "0")   # (of the kernel for many columns, whose workgroups are one for each sequence and kv head)
    gen = torch.Generator(device="cuda").manual_seed(13)
    S, G, D, L, ctx = 65535, 17, 64, 50, 2
    c, p = qa.KvCache("f16", S, G, D, ctx), qa.KvCache("f16", 1, G, D, L)
    k, v = (torch.randn(S, ctx, G, D, generator=gen, device="cuda").half() for _ in range(2))
    k0, v0 = (torch.randn(1, L, G, D, generator=gen, device="cuda").half() for _ in range(2))
    c.write(k, v, torch.zeros(S, dtype=torch.int32, device="cuda"))
    p.write(k0, v0, i32([0]))
    some = [0, 1, 61679, 61680, 61681, 61682, 65534]   # (2^20 / 17 = 61680.9)
    pos = torch.full((S,), -1, dtype=torch.int32, device="cuda")
    pos[some] = i32([1, 0, 1, 1, 0, 1, 1])
    q = torch.randn(S, 1, G, D, generator=gen, device="cuda").half()
    out = torch.full_like(q, 55.)
    c.attention(q, pos, prefix=p, out=out)
    for b in some:
        check_rows(out[b], q[b], torch.cat([k0[0], k[b]]).double().cpu(), torch.cat([v0[0], v[b]]).double().cpu(), L + int(pos[b]))
    others = torch.ones(S, dtype=torch.bool, device="cuda")
    others[some] = False
    assert bool((out[others] == 55).all())


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_few_positions_of_both(kind, type, hd):
    """up to and past the positions that a workgroup takes by itself: 32 tiles of 32 with 64 dims, 24 with 128"""
    gen = torch.Generator().manual_seed(hd)
    G, rep, n = 2, 3, 7
    most = (32 if hd == 64 else 24) * 32
    for L, ctx in ((1, 8), (31, 32), (33, 100), (most - 64, 33), (most - 33, 33), (most - 32, 33), (most - 200, 200)):
        pasts, lens = [ctx - n, 0, 3], [n, 2, min(5, ctx - 3)]
        p, K0, V0 = filled(kind, 1, G, hd, L, [L], gen)
        c, K, V = filled(kind, 3, G, hd, ctx, [a + m for a, m in zip(pasts, lens)], gen)
        q = torch.randn(3, n, G * rep, hd, generator=gen).to(TYPES[type]).cuda()
        out = torch.full_like(q, 55.)
        c.attention(q, i32(pasts), lens=i32(lens), prefix=p, out=out)
        for b, m in enumerate(lens):
            check_rows(out[b, :m], q[b, :m], both(K0, K, L, b), both(V0, V, L, b), L + pasts[b])
            assert bool((out[b, m:] == 55).all())
