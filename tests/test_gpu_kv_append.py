"""KvCache.append against 64-bit arithmetic.

Tolerances, in units u = 2^-24 of fp32's half step.  The mean of the squares: at most 16 squares one after the other and 6 additions across lanes, the product with 1 / head_dim
and + eps: 24 u; its root halves that and rounds, the quotient rounds: 14 u; two products with the row: 16 u.  The turn: o s rounds once, the sum once, each at most u of |x c| + |o s|, of
which 16 u are there before: 18 u (|x c| + |o s|), 20 taken.  Then the result's own rounding, eps / 2 of it (fp16 below 2^-14: 2^-25).  What a 4-bit cache makes of k is defined by
those fp32 values: it is compared to the bit wherever neither the scale nor the code has a border within 2^-18 of them."""
import math

import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv import BF16, F16, F32, TYPES, held, i32  # noqa: E402


def tables(places, half, gen=None):
    a = torch.arange(places, dtype=torch.float64).unsqueeze(1) * 10000.0 ** (-torch.arange(max(half, 1), dtype=torch.float64)[:half] / max(half, 1))
    return a.cos().float(), a.sin().float()


def turned(x, w, cos, sin, place, eps=1e-6):
    """x [n, heads, hd] (CPU) at places place .. -> (values, |x c| + |o s|) in 64 bits"""
    n, hd, half = x.shape[0], x.shape[-1], cos.shape[1]
    y = x.double()
    if w is not None:
        y = y / ((y * y).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    c, s = cos[place:place + n].double().unsqueeze(1), sin[place:place + n].double().unsqueeze(1)
    a, b = y[..., :half], y[..., half:2 * half]
    v = torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), y[..., 2 * half:].abs()], -1)
    return v, size


def check(got, want, size, t):
    floor = 2.0 ** -25 if t == F16 else 1e-40
    tol = 20 * 2.0 ** -24 * size + torch.finfo(t).eps / 2 * want.abs() * (1 + 2.0 ** -10) + floor
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"{int((~(err <= tol)).sum())} of {err.numel()} off, worst {float((err / tol).nan_to_num(1e9).max()):.2f} tolerances"


def check_held(got, want):
    """got: what a 4-bit cache reads back as (fp32), want: the rows in 64 bits"""
    g, y = got.double().cpu().unflatten(-1, (-1, 32)), want.unflatten(-1, (-1, 32))
    a = y.abs().amax(-1, keepdim=True)
    scale = lambda a: (a.clamp(max=65504.).float() / 7).to(BF16).to(F16).double()   # noqa: E731
    s = scale(a)
    sure = scale(a * (1 - 2.0 ** -18)) == scale(a * (1 + 2.0 ** -18))
    r = torch.where(s > 0, y / s, 0)
    code = lambda r: r.round().clamp(-7, 7)   # noqa: E731
    sure = sure & (code(r * (1 - 2.0 ** -18)) == code(r * (1 + 2.0 ** -18)))
    # (bf16's steps are 2^-8 of its values or less: a group's scale has a border within 2^-18 of it in one case of 2^8 or so; of the two groups of the smallest case one may)
    assert float(sure.double().mean()) >= 0.5
    assert torch.equal(torch.where(sure, g, 0), torch.where(sure, code(r) * s, 0))
    assert bool(((g - y).abs() <= (0.51 + 7 * 2.0 ** -7) * s + 1e-7).all())   # (elsewhere a step off at most, and a scale's step)


CASES = [   # hd, heads, kv heads, half, n, pos, lens, norm
    (128, 4, 1, 64, 1, [0], None, True), (64, 14, 2, 32, 1, [332], None, False), (128, 8, 8, 64, 1, [7, 0, 40], None, True), (64, 6, 3, 8, 1, [15, 16], [1, 1], True),
    (128, 28, 4, 32, 5, [3, 10], [5, 2], True), (64, 4, 2, 32, 17, [0, 6, 90], [17, 9, 1], False), (128, 2, 2, 16, 40, [13], None, True), (128, 3, 1, 48, 9, [1], None, False),
    (64, 2, 1, 24, 200, [5], None, True), (128, 32, 8, 64, 130, [0], None, True), (64, 8, 8, 0, 3, [2, 9], None, True),
]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("hd,H,G,half,n,pos,lens,norm", CASES)
def test_append(kind, hd, H, G, half, n, pos, lens, norm, type):
    print(f"append {kind} hd {hd} heads {H} / {G} half {half} n {n} {type}", flush=True)
    gen = torch.Generator().manual_seed(hd + n + half)
    t, S, ctx = TYPES[type], len(pos), max(pos) + n + 3
    live, behind = lens or [n] * len(pos), 11 if n % 2 else 0
    qkv = (torch.randn(S, n, H + 2 * G, hd, generator=gen) * (1 + 3 * (torch.rand(H + 2 * G, hd, generator=gen) < 0.06))).to(t)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + G], qkv[:, :, H + G:]
    w = [1 + 0.3 * torch.randn(hd, generator=gen) for _ in range(2)] if norm else [None, None]
    cos, sin = tables(behind + ctx, half)
    c, dev = qa.KvCache(kind, S, G, hd, ctx), qkv.cuda()
    out = torch.full((S, n, H, hd), 55., dtype=t, device="cuda")
    r = c.append(dev[:, :, :H], dev[:, :, H:H + G], dev[:, :, H + G:], i32(pos), cos.cuda(), sin.cuda(), q_weight=w[0].cuda() if norm else None, k_weight=w[1].cuda() if norm else None,
                 at=i32([p + behind for p in pos]) if behind else None, lens=i32(lens) if lens else None, out=out)
    assert r is out
    K, V = c.read(i32([0] * S), ctx, dtype=F32)
    for b in range(S):
        m, p = live[b], pos[b]
        check(out[b, :m], *turned(q[b, :m], w[0], cos, sin, p + behind), t)
        assert bool((out[b, m:] == 55).all())
        y, size = turned(k[b, :m], w[1], cos, sin, p + behind)
        if kind == "f16":
            check(K[b, p:p + m], y, size, F16)
            assert torch.equal(V[b, p:p + m].cpu(), v[b, :m].half().float())
        else:
            check_held(K[b, p:p + m], y)
            assert torch.equal(V[b, p:p + m].cpu(), held(v[b, :m]).float())
        for x in (K, V):
            assert not x[b, :p].any() and not x[b, p + m:].any()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_without_norm_and_turn_it_is_write(kind, type):
    gen = torch.Generator().manual_seed(2)
    S, n, H, G, D = 2, 9, 4, 2, 64
    q, k, v = (torch.randn(S, n, h, D, generator=gen).to(TYPES[type]).cuda() for h in (H, G, G))
    empty = torch.zeros(100, 0, device="cuda")
    for m in (n, 1):
        a, b = qa.KvCache(kind, S, G, D, 30), qa.KvCache(kind, S, G, D, 30)
        assert torch.equal(a.append(q[:, :m], k[:, :m], v[:, :m], i32([3, 20]), empty, empty), q[:, :m])
        b.write(k[:, :m], v[:, :m], i32([3, 20]))
        for x, y in zip(*((c.data if kind == "f16" else [c.data]) for c in (a, b))):
            assert torch.equal(x, y)


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("n", [1, 2, 11])
def test_what_takes_no_part(kind, n):
    """absent sequences, tokens behind lens, the cache's end, places outside the tables; over q; odd offsets and head-major rows"""
    gen = torch.Generator().manual_seed(6)
    S, H, G, D, ctx, places = 8, 4, 2, 64, 40, 30
    pos = [0, -1, ctx - 1, ctx, 9, 9, 9, 2]
    at = [0, 3, 5, 5, places - 1, -1, places, 2 ** 31 - 1]
    lens = [n, n, n, n, n, n, n, n - 1]
    live = [max(0, min(m, ctx - p, places - a)) if p >= 0 and a >= 0 else 0 for p, a, m in zip(pos, at, lens)]
    x = torch.randn(S, H + 2 * G, n, D + 3, generator=gen).half().cuda()[..., 3:].transpose(1, 2)
    q, k, v = x[:, :, :H], x[:, :, H:H + G], x[:, :, H + G:]
    cos, sin = tables(places, 32)
    w = torch.ones(D)
    c = qa.KvCache(kind, S, G, D, ctx)
    fill = torch.randn(S, ctx, G, D, generator=gen).half().cuda()
    c.write(fill, fill, i32([0] * S))
    was = c.read(i32([0] * S), ctx, dtype=F32)
    base = torch.full((S, n, H, D + 2), 55., device="cuda", dtype=F16)
    out = c.append(q, k, v, i32(pos), cos.cuda(), sin.cuda(), q_weight=w.cuda(), k_weight=w.cuda(), at=i32(at), lens=i32(lens), out=base[..., :D])
    now = c.read(i32([0] * S), ctx, dtype=F32)
    for b, m in enumerate(live):
        if m:
            check(out[b, :m], *turned(q[b, :m].cpu(), w, cos, sin, at[b]), F16)
            y, size = turned(k[b, :m].cpu(), w, cos, sin, at[b])
            if kind == "f16":
                check(now[0][b, pos[b]:pos[b] + m], y, size, F16)
            else:
                check_held(now[0][b, pos[b]:pos[b] + m], y)
        assert bool((out[b, m:] == 55).all())
        keep = torch.ones(ctx, dtype=torch.bool, device="cuda")
        keep[max(pos[b], 0):max(pos[b], 0) + m] = False
        for y, z in zip(was, now):
            assert torch.equal(y[b, keep], z[b, keep])
    assert bool((base[..., D:] == 55).all())
    over = q.contiguous()
    c.append(over, k, v, i32(pos), cos.cuda(), sin.cuda(), q_weight=w.cuda(), k_weight=w.cuda(), at=i32(at), lens=i32(lens), out=over)
    for b, m in enumerate(live):
        assert torch.equal(over[b, :m], out[b, :m]) and torch.equal(over[b, m:], q[b, m:])


@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_token_by_token_is_all_at_once(kind):
    gen = torch.Generator().manual_seed(7)
    S, n, H, G, D = 2, 21, 4, 2, 128
    q, k, v = (torch.randn(S, n, h, D, generator=gen).bfloat16().cuda() for h in (H, G, G))
    cos, sin = (x.cuda() for x in tables(60, 64))
    w = (1 + 0.2 * torch.randn(D, generator=gen)).cuda()
    pos = torch.tensor([3, 8], dtype=torch.int32, device="cuda")
    a, b = qa.KvCache(kind, S, G, D, 40), qa.KvCache(kind, S, G, D, 40)
    whole = a.append(q, k, v, pos, cos, sin, w, w)
    parts = [b.append(q[:, i:j], k[:, i:j], v[:, i:j], pos + i, cos, sin, w, w) for i, j in ((0, 1), (1, 2), (2, 9), (9, 20), (20, 21))]
    # (a mean of squares is summed in another order by the single token's 4-bit kernel: a query never is)
    assert torch.equal(torch.cat(parts, 1), whole)
    for x, y in zip(a.read(pos, n, dtype=F32), b.read(pos, n, dtype=F32)):
        if kind == "f16":
            assert torch.equal(x, y)
        else:
            assert float((x != y).double().mean()) < 1e-3


def test_rows_of_zeros_infinities_and_nan():
    D, w = 64, torch.ones(64, device="cuda")
    q = torch.zeros(1, 4, 1, D, device="cuda")
    q[0, 1, 0, 3], q[0, 2, 0, 40], q[0, 3, 0, 60] = math.inf, math.nan, 1e18
    cos, sin = (x.cuda() for x in tables(10, 16))
    c = qa.KvCache("f16", 1, 1, D, 10)
    out = c.append(q, q, q, i32([0]), cos, sin)
    assert not out[0, 0].any() and float(out[0, 3, 0, 60]) == float(q[0, 3, 0, 60])
    # without a norm only the pair of a dim turns not finite, and dims that are not turned stay as they are
    assert [i for i in range(D) if not math.isfinite(float(out[0, 1, 0, i]))] == [3, 19] and [i for i in range(D) if not math.isfinite(float(out[0, 2, 0, i]))] == [40]
    out = c.append(q, q, q, i32([0]), cos, sin, w, w, eps=1e-6)
    assert not out[0, 0].any() and bool(torch.isnan(out[0, 2]).all())
    assert abs(float(out[0, 3, 0, 60]) - 8) < 8 * 20 * 2.0 ** -24


@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("n", [1, 12])
def test_graph_and_other_stream(kind, n):
    gen = torch.Generator().manual_seed(9)
    S, H, G, D = 3, 8, 2, 128
    q, k, v = (torch.randn(S, n, h, D, generator=gen).half().cuda() for h in (H, G, G))
    cos, sin = (x.cuda() for x in tables(200, 64))
    w, pos = torch.ones(D, device="cuda"), i32([0, 5, 50])
    c, e = qa.KvCache(kind, S, G, D, 100), qa.KvCache(kind, S, G, D, 100)
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = e.append(q, k, v, pos, cos, sin, w, w)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(q, k, v, pos, cos, sin, w, w, out=out)
    for p in ([0, 5, 50], [8, 0, 31], [40, 41, 42]):
        pos.copy_(i32(p))
        out.fill_(3)
        g.replay()
        want = e.append(q, k, v, pos, cos, sin, w, w)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for x, y in zip(c.read(pos, n), e.read(pos, n)):
            assert torch.equal(x, y)
    assert first.shape == out.shape


def test_refusals():
    c = qa.KvCache("q4", 2, 2, 64, 40)
    q, k, pos = torch.zeros(2, 3, 4, 64, device="cuda", dtype=F16), torch.zeros(2, 3, 2, 64, device="cuda", dtype=F16), i32([0, 1])
    cos = torch.zeros(50, 32, device="cuda")
    ok = dict(q=q, k=k, v=k.clone(), pos=pos, cos=cos, sin=cos)
    c.append(**ok)

    def refused(words, **kw):
        with pytest.raises(qa.QphError, match=words):
            c.append(**{**ok, **kw})
    for name in ("q", "k", "v"):
        x = ok[name]
        refused("device", **{name: x.cpu()})
        refused("float32, float16 or bfloat16", **{name: x.double()})
        refused("must be", **{name: x[:1]})
        refused("same type", **{name: x.float()})
    refused("numbers of tokens", k=k[:, :2])
    refused("2 heads", k=q)
    refused("multiple of kv_heads", q=q[:, :, :3])
    refused("q's shape", out=q[:, :2])
    refused("same type", out=q.float())
    refused("overlap", out=torch.zeros(1, 3, 4, 64, device="cuda", dtype=F16).expand(2, 3, 4, 64))
    for bad in (cos.half(), cos[0], cos[:, ::2], cos.double()):
        refused("cos", cos=bad)
        refused("sin", sin=bad)
    refused("sin", sin=cos[:, :16])
    refused("same shape", sin=cos[:40])
    refused("device", cos=cos.cpu())
    for half in (4, 33, 40):
        refused("half the rotated", cos=torch.zeros(50, half, device="cuda"), sin=torch.zeros(50, half, device="cuda"))
    refused("places", cos=cos[:0], sin=cos[:0])
    for name in ("q_weight", "k_weight"):
        for bad in (torch.ones(32, device="cuda"), torch.ones(64, device="cuda").half(), torch.ones(2, 64, device="cuda")):
            refused(name, **{name: bad})
    refused("at", at=pos.long())
    refused("eps", eps=-1.0)
    refused("eps", eps=math.inf)
    refused("eps", eps=math.nan)
    assert c.append(**{**ok, "q": q[:, :0], "k": k[:, :0], "v": k[:, :0]}).shape == (2, 0, 4, 64)


def test_optional_tensors_without_memory_are_refused():
    """what may be left out and was given back (its storage resized to nothing) is not taken as left out: lens, at, norms' weights, a prefix's length, a copy's sequences"""
    def gone(x):
        x.untyped_storage().resize_(0)
        return x

    one, ones = lambda *s: torch.ones(*s, device="cuda"), lambda: gone(torch.ones(2, dtype=torch.int32, device="cuda"))   # noqa: E731
    c, prefix = qa.KvCache("f16", 2, 1, 64, 40), qa.KvCache("f16", 1, 1, 64, 8)
    x, pos, t = one(2, 1, 1, 64), i32([3, 4]), one(50, 32)
    index = i32([[0], [0]])
    for name, call in (("q_weight", lambda: c.append(x, x, x, pos, t, t, q_weight=gone(one(64)))), ("k_weight", lambda: c.append(x, x, x, pos, t, t, k_weight=gone(one(64)))),
                       ("at", lambda: c.append(x, x, x, pos, t, t, at=ones())), ("lens", lambda: c.append(x, x, x, pos, t, t, lens=ones())), ("pos", lambda: c.append(x, x, x, ones(), t, t)),
                       ("cos", lambda: c.append(x, x, x, pos, gone(one(50, 32)), t)), ("lens", lambda: c.attention(x, pos, lens=ones())), ("lens", lambda: c.write(x, x, pos, lens=ones())),
                       ("prefix_len", lambda: c.attention(x, pos, prefix=prefix, prefix_len=gone(torch.ones(1, dtype=torch.int32, device="cuda")))),
                       ("seqs", lambda: c.copy(index, pos, seqs=ones()))):
        with pytest.raises(qa.QphError, match=f"{name} has no memory"):
            call()
    assert not bool(c.data[0].any())
    empty = one(50, 0)
    assert torch.equal(c.append(x, x, x, pos, empty, empty), x)   # (nothing to turn: tables without elements are as good as any)
    assert torch.equal(c.data[0][0, 3, 0].float(), x[0, 0, 0])
