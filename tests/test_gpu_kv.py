"""KvCache (qph_kv_write / read / attention) on the GPU against plain 64-bit arithmetic on the CPU.

Tolerances.  The rows that a 4-bit cache holds are defined to the bit.  An attention output o = sum p v, A = sum p |v|, may be off
by its last rounding (eps / 2 |o|), by the rounding of the probabilities to the matrix cores' fp16 (2^-11 A; fp32 queries:
two halves, 2^-21), and by what moves a score s by ds, which moves o by at most 2 ds A: the queries' operand (2^-25, fp32 2^-22 of
the row's largest, times sum |k|), fp32 sums of head_dim products (head_dim 2^-24 sum |q k|), the exponent's own rounding (2^-24 times
its size, under 2 max |s| log2 e + 64 with the scores' power and bias) and the hardware exp2 (2^-22); the sum over T
positions in fp32 adds T 2^-24, in blocks of 8 and more log-like, taken as sqrt(T) 2^-22."""
import ctypes as C
import math

import numpy as np
import pytest

import qpack_amd as qa
from qpack_amd._lib import KvC, RowsC, lib

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}


def held(x):
    """what a 4-bit cache holds of rows x [.., head_dim], float64"""
    y = x.double().unflatten(-1, (-1, 32))
    a = y.abs().amax(-1, keepdim=True)
    s = (a.clamp(max=65504.).float() / 7).to(BF16).to(F16).double()
    c = torch.where(s > 0, (y / s).round().clamp(-7, 7), 0.)
    return torch.where(torch.isfinite(a), c * s, math.nan).flatten(-2)


@pytest.fixture(params=["", "0", "100000"], ids=["auto", "many", "few"])
def route(request, monkeypatch):
    """the call's own choice of kernel, and each of the two"""
    if request.param:
        monkeypatch.setenv("QPH_KV_FEW", request.param)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def reference(q, K, V, P0, window=0, sinks=0, scale=0.0):
    """q [n, heads, hd] at positions P0 .., K / V [ctx, kv_heads, hd] float64 -> (output, A, tolerance term ds) per row"""
    n, H, D = q.shape
    G = K.shape[1]
    scale = scale or 1 / math.sqrt(D)
    out = torch.empty(n, H, D, dtype=torch.float64)
    A = torch.empty_like(out)
    ds = torch.empty(n, H, 1, dtype=torch.float64)
    for t in range(n):
        P = P0 + t
        p = torch.arange(P + 1)
        if window:
            p = p[(p > P - window) | (p < sinks)]
        for g in range(G):
            k, v = K[p, g], V[p, g]
            qq = q[t, g * (H // G):(g + 1) * (H // G)]
            s = qq @ k.T * scale
            w = torch.softmax(s, -1)
            out[t, g * (H // G):(g + 1) * (H // G)] = w @ v
            A[t, g * (H // G):(g + 1) * (H // G)] = w @ v.abs()
            size = (qq.abs() @ k.abs().T).amax(-1) * scale
            first = qq.abs().amax(-1) * k.abs().sum(-1).amax() * scale
            ds[t, g * (H // G):(g + 1) * (H // G), 0] = D * 2.0 ** -24 * size + 2.0 ** -24 * (2 * size * 1.4427 + 64) + math.sqrt(len(p)) * 2.0 ** -22 + 2.0 ** -22
            ds[t, g * (H // G):(g + 1) * (H // G), 0] += first * (2.0 ** -22 if q.dtype == torch.float64 and getattr(reference, "two", False) else 2.0 ** -25)
    return out, A, ds


def check_rows(got, q, K, V, P0, **mask):
    """got, q [n, heads, hd] (GPU tensors of one type) of one sequence"""
    reference.two = q.dtype == F32
    o, A, ds = reference(q.double().cpu(), K, V, P0, **mask)
    tol = A * ((2.0 ** -21 if q.dtype == F32 else 2.0 ** -11) + 2 * ds) + torch.finfo(q.dtype).eps / 2 * o.abs() + 1e-30
    err = (got.double().cpu() - o).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).nan_to_num(1e9).max()):.2f} tolerances"


def filled(kind, S, G, D, ctx, T, gen, loud=True):
    """a cache with T[b] positions of random rows written, and the values it holds"""
    c = qa.KvCache(kind, S, G, D, ctx)
    k = torch.randn(S, max(T), G, D, generator=gen) * (1 + 3 * (torch.rand(G, D, generator=gen) < 0.06))
    v = torch.randn(S, max(T), G, D, generator=gen)
    k, v = k.half(), v.half()
    c.write(k.cuda(), v.cuda(), i32([0] * S), lens=i32(T))
    if kind == "q4":
        return c, held(k), held(v)
    return c, k.double(), v.double()


# ------------------------------------------------------------------ writing and reading
@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("S,G,n,pos", [(1, 1, 1, [0]), (1, 3, 1, [13]), (2, 2, 5, [6, 9]), (3, 1, 17, [0, 7, 30]), (1, 8, 200, [3])])
def test_write_read(kind, hd, type, S, G, n, pos):
    gen = torch.Generator().manual_seed(hd + n)
    t, ctx = TYPES[type], max(pos) + n + 3
    c = qa.KvCache(kind, S, G, hd, ctx)
    k, v = ((torch.randn(S, n, G, hd, generator=gen) * 10 ** torch.randn(S, n, G, 1, generator=gen)).to(t) for _ in range(2))
    c.write(k.cuda(), v.cuda(), i32(pos))
    for out_t in (F32, F16, BF16):
        rk, rv = c.read(i32(pos), n, dtype=out_t)
        for got, x in ((rk, k), (rv, v)):
            want = held(x) if kind == "q4" else x.to(F16)
            assert torch.equal(got.cpu(), want.to(out_t) if kind == "q4" else want.to(F32).to(out_t))
    whole = c.read(i32([0] * S), ctx, dtype=F32)
    for b in range(S):   # nothing but the call's positions was written
        for x in whole:
            assert not x[b, :pos[b]].any() and not x[b, pos[b] + n:].any()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["q4", "f16"])
def test_write_in_pieces_keeps_the_rest(kind, hd):
    gen = torch.Generator().manual_seed(5)
    G, ctx = 2, 45
    k, v = (torch.randn(1, ctx, G, hd, generator=gen) for _ in range(2))
    a, b = qa.KvCache(kind, 1, G, hd, ctx), qa.KvCache(kind, 1, G, hd, ctx)
    a.write(k.cuda(), v.cuda(), i32([0]))
    at = 0
    for n in (1, 1, 3, 8, 2, 17, 13):
        b.write(k[:, at:at + n].cuda(), v[:, at:at + n].cuda(), i32([at]))
        at += n
    assert at == ctx
    b.write(k[:, 20:23].cuda(), v[:, 20:23].cuda(), i32([20]))   # again: the same rows
    for x, y in zip(a.data if kind == "f16" else [a.data], b.data if kind == "f16" else [b.data]):
        assert torch.equal(x, y)


def test_q4_border_values():
    """ties go to the even code; zeros, the smallest scales, values past fp16, NaN and infinities"""
    x = torch.zeros(1, 10, 1, 64)
    x[0, 0, 0, :16] = torch.tensor([7, 0.5, 1.5, 2.5, 3.5, -0.5, -1.5, -2.5, 4.5, 5.5, 6.5, -6.5, -3.5, 0.49999997, 0.50000006, 6.4999995])
    x[0, 1, 0, :8] = torch.tensor([7e-8, 1e-8, 3e-8, 6e-8, -6e-8, 2e-38, 0, 4.2e-7])
    x[0, 2, 0, :4] = torch.tensor([1e-20, 1e-38, -1e-45, 1e-30])
    x[0, 3, 0, :5] = torch.tensor([65504., -65520., 1e30, 3.4e38, 4000.])
    x[0, 4, 0, 3] = math.nan
    x[0, 5, 0, 40] = math.inf
    x[0, 6, 0, 1], x[0, 6, 0, 2] = -math.inf, math.nan
    # next to a border: (k + 1/2) s and its neighbours, s of 8 bits
    r = np.random.default_rng(3)
    for row in (7, 8, 9):
        s = np.float32((128 + r.integers(0, 128)) * 2.0 ** r.integers(-12, 3))
        m = (r.integers(0, 7, 62) + 0.5).astype(np.float32) * s
        d = r.integers(-1, 2, 62)
        m = np.where(d < 0, np.nextafter(m, np.float32(0)), np.where(d > 0, np.nextafter(m, np.float32(np.inf)), m))
        x[0, row, 0, 2:] = torch.from_numpy(m.astype(np.float32) * r.choice([-1, 1], 62).astype(np.float32))
        x[0, row, 0, 0] = x[0, row, 0, 32] = float(7 * s)
    c = qa.KvCache("q4", 1, 1, 64, 10)
    c.write(x.cuda(), x.flip(-1).contiguous().cuda(), i32([0]))
    k, v = c.read(i32([0]), 10, dtype=F32)
    assert torch.equal(torch.nan_to_num(k.cpu(), nan=123.), torch.nan_to_num(held(x).float(), nan=123.))
    assert torch.equal(torch.nan_to_num(v.cpu(), nan=123.), torch.nan_to_num(held(x.flip(-1)).float(), nan=123.))
    # what was read back and is written again is the same
    again = qa.KvCache("q4", 1, 1, 64, 10)
    again.write(*c.read(i32([0]), 10, dtype=F16), i32([0]))
    k2, _ = again.read(i32([0]), 10, dtype=F32)
    assert torch.equal(torch.nan_to_num(k2, nan=123.), torch.nan_to_num(k, nan=123.))


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_q4_16_bit_rows_next_to_every_border(type):
    """every scale of 8 bits at a few sizes, the values of the type on and around the borders (k + 1/2) s, both signs"""
    t = TYPES[type]
    rows = []
    for e in (-22, -14, -7, 0, 5):
        for j in range(128, 256):
            s = j * 2.0 ** e
            edge = torch.tensor([(k + 0.5) * s for k in range(7)]).to(t)
            bits = edge.view(torch.int16)
            near = torch.cat([(bits + d).view(t).float() for d in (-1, 0, 1)])   # 21 values and their negatives
            g = torch.zeros(64)
            g[0] = g[32] = 7 * s
            g[1:22], g[33:54] = near, -near
            rows.append(g)
    x = torch.stack(rows).to(t).view(1, -1, 1, 64)
    n = x.shape[1]
    c = qa.KvCache("q4", 1, 1, 64, n)
    c.write(x.cuda(), x.flip(-1).contiguous().cuda(), i32([0]))
    k, v = c.read(i32([0]), n, dtype=F32)
    assert torch.equal(k.cpu(), held(x).float()) and torch.equal(v.cpu(), held(x.flip(-1)).float())
    for p in range(0, n, 37):   # the single token's kernel
        c.write(x[:, p:p + 1].cuda() * 0, x[:, p:p + 1].cuda() * 0, i32([p]))
        c.write(x[:, p:p + 1].cuda(), x.flip(-1)[:, p:p + 1].contiguous().cuda(), i32([p]))
    again = c.read(i32([0]), n, dtype=F32)
    assert torch.equal(again[0], k) and torch.equal(again[1], v)


@pytest.mark.parametrize("kind", ["q4", "f16"])
def test_write_read_strides_limits_and_absent_sequences(kind):
    gen = torch.Generator().manual_seed(9)
    S, n, G, D, ctx = 4, 6, 2, 64, 20
    # a head-major tensor, an odd offset, an expanded one
    k = torch.randn(S, G, n, D + 1, generator=gen).cuda().half()[..., 1:].transpose(1, 2)
    v = torch.randn(1, n, 1, D, generator=gen).cuda().half().expand(S, n, G, D)
    pos, lens = [0, -1, 17, 19], [6, 6, 6, 0]
    c = qa.KvCache(kind, S, G, D, ctx)
    c.write(k, v, i32(pos), lens=i32(lens))
    want = torch.zeros(2, S, ctx, G, D)
    for b in range(S):
        for t in range(min(n, lens[b])):
            if pos[b] >= 0 and pos[b] + t < ctx:
                for i, x in enumerate((k, v)):
                    r = x[b, t].cpu()
                    want[i, b, pos[b] + t] = held(r).float() if kind == "q4" else r.float()
    got = c.read(i32([0] * S), ctx, dtype=F32)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    base = torch.full((S, n, G, 2 * D), 77., device="cuda")
    ok, ov = base[..., :D], torch.full((S, n, G, D), 77., device="cuda")
    c.read(i32(pos), n, lens=i32(lens), out=(ok, ov))
    for b in range(S):
        for t in range(n):
            there = t < lens[b] and pos[b] >= 0 and pos[b] + t < ctx
            for i, x in enumerate((ok, ov)):
                assert torch.equal(x[b, t].cpu(), want[i, b, pos[b] + t] if there else torch.full((G, D), 77.))
    assert bool((base[..., D:] == 77).all())


# ------------------------------------------------------------------ attention
CASES = [   # kind, hd, kv heads, rep, n, pasts, window, sinks
    ("q4", 128, 2, 4, 1, [0], 0, 0), ("q4", 64, 2, 7, 1, [1, 40, 31], 0, 0), ("q4", 128, 1, 1, 1, [333], 0, 0), ("q4", 64, 1, 8, 1, [700, 5], 0, 0),
    ("q4", 128, 1, 4, 1, [2600], 0, 0), ("q4", 128, 1, 3, 5, [1000, 0], 0, 0), ("q4", 64, 2, 16, 2, [77], 0, 0), ("q4", 128, 1, 5, 3, [90], 20, 3),
    ("q4", 64, 1, 4, 1, [900, 3], 100, 4), ("q4", 128, 1, 7, 1, [1500], 301, 17), ("q4", 64, 2, 2, 1, [50], 1, 0), ("q4", 64, 1, 1, 4, [60], 8, 60),
    ("f16", 128, 2, 4, 1, [0, 300], 0, 0), ("f16", 64, 1, 7, 1, [1030], 0, 0), ("f16", 128, 1, 8, 1, [2000], 128, 4), ("f16", 64, 1, 3, 4, [500], 37, 9),
    ("f16", 128, 1, 2, 7, [55, 3], 16, 0), ("f16", 64, 2, 5, 1, [120], 1000, 4),
    # the prompt kernel: more than 64 columns
    ("q4", 128, 1, 4, 65, [0], 0, 0), ("q4", 64, 2, 7, 40, [3, 100], 0, 0), ("q4", 128, 1, 1, 300, [0], 0, 0), ("q4", 64, 1, 8, 130, [513], 0, 0),
    ("q4", 128, 2, 3, 33, [700], 0, 0), ("q4", 128, 1, 2, 150, [20], 48, 5), ("q4", 64, 1, 4, 90, [400], 100, 70), ("q4", 64, 1, 66, 2, [130], 0, 0),
    ("f16", 128, 1, 4, 70, [0, 9], 0, 0), ("f16", 64, 2, 7, 50, [130], 0, 0), ("f16", 128, 1, 2, 200, [64], 33, 4), ("f16", 64, 1, 3, 129, [300], 64, 0),
    ("f16", 128, 1, 1, 280, [0], 1, 1), ("f16", 128, 1, 8, 20, [1100], 0, 0),
]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind,hd,G,rep,n,pasts,window,sinks", CASES)
def test_attention(kind, hd, G, rep, n, pasts, window, sinks, type, route):
    print(f"attention {kind} hd {hd} kv heads {G} rep {rep} n {n} pasts {pasts} window {window} sinks {sinks} {type}", flush=True)
    gen = torch.Generator().manual_seed(n + sum(pasts))
    S, ctx = len(pasts), max(pasts) + n + 5
    c, K, V = filled(kind, S, G, hd, ctx, [p + n for p in pasts], gen)
    q = (torch.randn(S, n, G * rep, hd, generator=gen) * 1.5).to(TYPES[type]).cuda()
    out = c.attention(q, i32(pasts), window=window, sinks=sinks)
    for b in range(S):
        check_rows(out[b], q[b], K[b], V[b], pasts[b], window=window, sinks=sinks)


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_attention_unseen_memory_may_hold_anything(kind, n, route):
    """NaN and infinities in unwritten positions, behind the last token, and before the window change nothing"""
    gen = torch.Generator().manual_seed(4)
    G, rep, D, past, window, sinks = 2, 4, 128, 150, 60, 3
    c, K, V = filled(kind, 1, G, D, 256, [past + n], gen)
    q = torch.randn(1, n, G * rep, D, generator=gen).half().cuda()
    bad = torch.full((1, past - window - 20, G, D), math.nan, device="cuda")
    c.write(bad, bad, i32([sinks]))                       # sinks .. : every position there is before every token's window
    far = 256 - past - n
    c.write(torch.full((1, far, G, D), math.inf, device="cuda"), torch.full((1, far, G, D), math.nan, device="cuda"), i32([past + n]))
    if kind == "q4":
        c.data[:, :, (past + n + 7) // 8:] = 255          # codes and scales of all ones
    out = c.attention(q, i32([past]), window=window, sinks=sinks)
    check_rows(out[0], q[0], K[0], V[0], past, window=window, sinks=sinks)


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("n,rep,where", [(4, 4, 2), (5, 3, 4), (40, 4, 17), (100, 1, 99)])
def test_attention_nan_rows_stay_with_those_who_see_them(kind, n, rep, where, route):
    """a NaN in one token's V row, an infinity in another's K: earlier tokens don't see them, the window's later ones no more"""
    gen = torch.Generator().manual_seed(6)
    G, D, past, window = 1, 64, 30, 12
    c, K, V = filled(kind, 1, G, D, 256, [past + n], gen)
    k, v = c.read(i32([past + where]), 1, dtype=F32)
    v[..., 5] = math.nan
    c.write(k, v, i32([past + where]))
    q = torch.randn(1, n, rep, D, generator=gen).half().cuda()
    out = c.attention(q, i32([past]), window=window)
    seen = [t for t in range(n) if where <= t < where + window]
    clean = [t for t in range(n) if t not in seen]
    for t in clean:
        check_rows(out[0, t:t + 1], q[0, t:t + 1], K[0], V[0], past + t, window=window)
    dims = torch.zeros(D, dtype=torch.bool)
    dims[:32 if kind == "q4" else 0] = True   # the group's scale, or the value itself
    dims[5] = True
    for t in seen:
        assert bool(torch.isnan(out[0, t, :, dims.cuda()]).all()) and bool(torch.isfinite(out[0, t, :, ~dims.cuda()]).all())


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("hd,type", [(64, "f32"), (128, "f16"), (128, "bf16")])
@pytest.mark.parametrize("S,n,G,rep,pasts,lens", [(4, 47, 1, 33, [1400, 30, -1, 1453], [47, 47, 47, 5]), (16, 8, 2, 16, [1100] * 14 + [40, -1], [8] * 12 + [3, 0, 8, 8])])
def test_attention_many_split_rows(kind, hd, type, S, n, G, rep, pasts, lens, route):
    """thousands of rows whose splits are merged, beside short and absent sequences; a head of them behind n's end is left alone"""
    print(f"many split rows {kind} {hd} {type} S {S}", flush=True)
    gen = torch.Generator().manual_seed(S)
    ctx = max(pasts) + n
    c, K, V = filled(kind, S, G, hd, ctx, [p + m if p >= 0 else 0 for p, m in zip(pasts, lens)], gen)
    q = torch.randn(S, n, G * rep, hd, generator=gen).to(TYPES[type]).cuda()
    out = torch.full_like(q, 55.)
    c.attention(q, i32(pasts), lens=i32(lens), out=out)
    for b in range(S):
        m = lens[b] if pasts[b] >= 0 else 0
        if m and (S == 4 or b % 5 == 0 or b > 11):
            check_rows(out[b, :m], q[b, :m], K[b], V[b], pasts[b])
        assert bool((out[b, m:] == 55).all())


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("n", [1, 33])
def test_attention_strides_ragged_absent_and_in_place(kind, n, route):
    gen = torch.Generator().manual_seed(8)
    S, G, rep, D = 5, 2, 4, 64
    pasts, lens, ctx = [100, 7, -1, 40, 300 - n // 2], [n, max(1, n // 2), n, 0, n], 300
    T = [min(ctx, p + m) if p >= 0 else 0 for p, m in zip(pasts, lens)]
    c, K, V = filled(kind, S, G, D, ctx, T, gen)
    x = torch.randn(S, G * rep, n, D + 3, generator=gen).cuda().half()
    q = x[..., 3:].transpose(1, 2)                       # head-major, odd offset
    base = torch.full((S, n, G * rep, D + 2), 55., device="cuda", dtype=F16)
    out = base[..., :D]
    c.attention(q, i32(pasts), lens=i32(lens), out=out)
    plain = q.contiguous()
    c.attention(plain, i32(pasts), lens=i32(lens), out=plain)   # over q
    for b in range(S):
        m = max(0, min(lens[b], ctx - pasts[b])) if pasts[b] >= 0 else 0
        if m:
            check_rows(out[b, :m], q[b, :m], K[b], V[b], pasts[b])
        assert torch.equal(plain[b, :m], out[b, :m]) and torch.equal(plain[b, m:], q[b, m:])
        assert bool((out[b, m:] == 55).all())
    assert bool((base[..., D:] == 55).all())


@pytest.mark.parametrize("type,size", [("f32", 1e-6), ("f32", 3e4), ("bf16", 1e-30), ("bf16", 1e4), ("f16", 6e-8)])
def test_attention_query_range(type, size, route):
    """rows far from 1, with the softmax scale that brings the scores back"""
    gen = torch.Generator().manual_seed(2)
    c, K, V = filled("q4", 1, 1, 128, 200, [200], gen)
    for n in (1, 80):
        q = (torch.randn(1, n, 4, 128, generator=gen) * size).to(TYPES[type]).cuda()
        out = c.attention(q, i32([200 - n]), scale=0.05 / size)
        check_rows(out[0], q[0], K[0], V[0], 200 - n, scale=0.05 / size)


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_attention_vanishing_scores(kind, type, route):
    """the scale times a row's power is below fp32's range: the positions weigh alike, the masked ones nothing"""
    gen = torch.Generator().manual_seed(12)
    c, K, V = filled(kind, 1, 1, 64, 200, [200], gen)
    for n in (3, 80):
        q = (torch.randn(1, n, 4, 64, generator=gen) * 1e-37).to(TYPES[type]).cuda()
        out = c.attention(q, i32([200 - n]), scale=1e-9)
        check_rows(out[0], q[0], K[0], V[0], 200 - n, scale=1e-9)


@pytest.mark.parametrize("kind", ["q4", "f16"])
def test_attention_far_smaller_weights_count(kind, route):
    """one position far above thousands that share the rest of the weight"""
    D, T = 64, 4096
    k = torch.zeros(1, T, 1, D)
    k[0, 100, 0, 0] = 7
    v = torch.zeros(1, T, 1, D)
    v[0, :, 0, 1] = 7
    v[0, 100, 0, 1] = 0
    c = qa.KvCache(kind, 1, 1, D, T)
    c.write(k.cuda(), v.cuda(), i32([0]))
    q = torch.zeros(1, 1, 1, D, device="cuda", dtype=F16)
    q[..., 0] = 2 * math.log(2)   # score 14 ln 2 / .. : weight 2^-18 each with the scale below
    out = c.attention(q, i32([T - 1]), scale=18 / 14)
    check_rows(out[0], q[0], k[0].double(), v[0].double(), T - 1, scale=18 / 14)
    assert float(out[0, 0, 0, 1]) > 0.05


def test_cache_past_32_bit_offsets(route):
    """17M positions: record and row offsets past 2^31 bytes and elements"""
    G, D = 1, 128
    gen = torch.Generator().manual_seed(1)
    for kind, ctx in (("q4", 17 << 20), ("f16", (17 << 20) + 64)):
        c = qa.KvCache(kind, 1, G, D, ctx)
        past = ctx - 90
        k, v = torch.randn(1, 90, G, D, generator=gen).half(), torch.randn(1, 90, G, D, generator=gen).half()
        c.write(k.cuda(), v.cuda(), i32([past]))
        hk, hv = (held(k), held(v)) if kind == "q4" else (k.double(), v.double())
        assert torch.equal(c.read(i32([past]), 90)[1].cpu().double(), hv)
        for n in (1, 40):
            q = torch.randn(1, n, 4, D, generator=gen).half().cuda()
            out = c.attention(q, i32([ctx - n]), window=50, sinks=0)
            check_rows(out[0], q[0], hk[0], hv[0], 90 - n, window=50)
        del c


@pytest.mark.parametrize("kind", ["q4", "f16"])
def test_captured_steps(kind, route):
    """write and attention in a graph, replayed at other positions, eager work between"""
    gen = torch.Generator().manual_seed(3)
    S, G, rep, D, ctx = 2, 2, 4, 128, 2100
    T = [2000, 300]
    c, K, V = filled(kind, S, G, D, ctx, T, gen)
    pos = i32(T)
    k, v = torch.zeros(S, 1, G, D, device="cuda", dtype=F16), torch.zeros(S, 1, G, D, device="cuda", dtype=F16)
    q, out = torch.zeros(S, 1, G * rep, D, device="cuda", dtype=F16), torch.zeros(S, 1, G * rep, D, device="cuda", dtype=F16)

    def step():
        c.write(k, v, pos)
        c.attention(q, pos, out=out)
        pos.add_(1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):   # the first calls, outside the capture; their positions are written again below
        step()
    torch.cuda.synchronize()
    pos.copy_(i32(T))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    pos.copy_(i32(T))
    for i in range(4):
        nk, nv, nq = (torch.randn(S, 1, h, D, generator=gen).half() for h in (G, G, G * rep))
        k.copy_(nk), v.copy_(nv), q.copy_(nq)
        g.replay()
        torch.cuda.synchronize()
        hk, hv = (held(nk), held(nv)) if kind == "q4" else (nk.double(), nv.double())
        for b in range(S):
            P = T[b] + i
            if K.shape[1] <= P:
                K, V = (torch.cat([x, torch.zeros(S, P + 1 - x.shape[1], G, D, dtype=torch.float64)], 1) for x in (K, V))
            K[b, P], V[b, P] = hk[b, 0], hv[b, 0]
            check_rows(out[b], q[b], K[b], V[b], P)
        eager = c.attention(q, pos - 1)
        assert torch.equal(eager, out)


def test_two_graphs_and_an_eager_call_at_once():
    """each captured call has scratch of its own"""
    gen = torch.Generator().manual_seed(31)
    c, K, V = filled("q4", 2, 2, 128, 4000, [4000, 2600], gen)
    qs = [torch.randn(2, n, 8, 128, generator=gen).half().cuda() for n in (1, 2, 40)]
    pos = [i32([4000 - q.shape[1], 2600 - q.shape[1]]) for q in qs]
    want = [c.attention(q, p) for q, p in zip(qs, pos)]
    for q, p, w in zip(qs, pos, want):
        for b in range(2):
            check_rows(w[b], q[b], K[b], V[b], int(p[b]))
    outs, graphs = [torch.empty_like(q) for q in qs], []
    torch.cuda.synchronize()
    for q, p, o in zip(qs, pos, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.attention(q, p, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for o in outs:
            o.fill_(9)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = c.attention(qs[1], pos[1])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[1])
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_scratch_is_not_read_before_it_is_written_and_results_repeat(route):
    gen = torch.Generator().manual_seed(12)
    c, K, V = filled("q4", 1, 1, 128, 3000, [3000], gen)
    for n, rep in ((1, 4), (40, 4)):
        q = torch.randn(1, n, rep, 128, generator=gen).half().cuda()
        b = C.c_int64()
        kv = KvC(qa.QPH_Q4, 1, 1, 128, 3000, c.data.data_ptr())
        rows = lambda x: RowsC(x.data_ptr(), qa.QPH_F16, x.stride(0), x.stride(1), x.stride(2))   # noqa: E731
        qa._lib.check(lib().qph_kv_attention_work(C.byref(kv), qa.QPH_F16, rep, n, 0, 0, C.byref(b)))
        assert b.value > 0
        outs, pos = [], i32([3000 - n])
        for fill in (255, 0, 127):
            work = torch.full((b.value + 64,), fill, dtype=torch.uint8, device="cuda")
            o = torch.empty_like(q)
            qa._lib.check(lib().qph_kv_attention(C.byref(kv), C.byref(rows(q)), C.byref(rows(o)), rep, n, pos.data_ptr(), None, 0, 0, 0.0,
                                                 work.data_ptr(), b.value, torch.cuda.current_stream().cuda_stream))
            torch.cuda.synchronize()
            assert bool((work[b.value:] == fill).all())
            outs.append(o)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
        check_rows(outs[0][0], q[0], K[0], V[0], 3000 - n)


def test_two_streams_at_once(route):
    gen = torch.Generator().manual_seed(13)
    c, K, V = filled("q4", 1, 2, 64, 1500, [1500], gen)
    q = [torch.randn(1, n, 8, 64, generator=gen).half().cuda() for n in (1, 24)]
    pos = [i32([1499]), i32([1476])]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    outs = []
    for _ in range(3):
        for s, x, p in zip(streams, q, pos):
            with torch.cuda.stream(s):
                outs.append(c.attention(x, p))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, outs[i % 2])
        check_rows(o[0], q[i % 2][0], K[0], V[0], int(pos[i % 2]))


@pytest.mark.parametrize("kind", ["q4", "f16"])
def test_conversation(kind, route):
    """a prompt, steps, a turn of several tokens and steps over it, two sequences: as a server runs them"""
    gen = torch.Generator().manual_seed(21)
    S, G, rep, D, ctx, window, sinks = 2, 2, 4, 64, 400, 70, 4
    c = qa.KvCache(kind, S, G, D, ctx)
    K, V = torch.zeros(S, ctx, G, D, dtype=torch.float64), torch.zeros(S, ctx, G, D, dtype=torch.float64)
    at = [0, 0]
    for n, lens in ((120, [120, 77]), (1, [1, 1]), (1, [1, 0]), (30, [12, 30]), (1, [1, 1])):
        k, v, q = (torch.randn(S, n, h, D, generator=gen).to(BF16).cuda() for h in (G, G, G * rep))
        c.write(k, v, i32(at), lens=i32(lens))
        out = c.attention(q, i32(at), lens=i32(lens), window=window, sinks=sinks)
        for b in range(S):
            m = lens[b]
            hk, hv = (held(k[b, :m].cpu()), held(v[b, :m].cpu())) if kind == "q4" else (k[b, :m].cpu().half().double(), v[b, :m].cpu().half().double())
            K[b, at[b]:at[b] + m], V[b, at[b]:at[b] + m] = hk, hv
            if m:
                check_rows(out[b, :m], q[b, :m], K[b], V[b], at[b], window=window, sinks=sinks)
            assert not out[b, m:].any()
            at[b] += m


def test_python_refusals():
    c = qa.KvCache("q4", 2, 2, 64, 40)
    f = qa.KvCache("f16", 2, 2, 64, 40)
    k = torch.zeros(2, 3, 2, 64, device="cuda", dtype=F16)
    q, pos = torch.zeros(2, 3, 4, 64, device="cuda", dtype=F16), i32([0, 1])
    for cache in (c, f):
        for bad, words in ((k.cpu(), "device"), (k.double(), "float32, float16 or bfloat16"), (k[:1], "must be"), (k[0], "must be"), (k[..., :32], "must be"),
                           (torch.zeros(2, 3, 2, 128, device="cuda", dtype=F16)[..., ::2], "contiguous"), (k[:, :, :1], "heads")):
            with pytest.raises(qa.QphError, match=words):
                cache.write(bad, k, pos)
            with pytest.raises(qa.QphError, match=words):
                cache.write(k, bad, pos)
            with pytest.raises(qa.QphError):
                cache.read(pos, 3, out=(k, bad))
            if words != "heads":
                with pytest.raises(qa.QphError, match=words):
                    cache.attention(bad, pos, out=q)
        for bad in (None, 3, torch.nested.nested_tensor([k[0], k[1]])):
            with pytest.raises(qa.QphError, match="must be|plain"):
                cache.write(bad, k, pos)
            with pytest.raises(qa.QphError, match="must be|plain"):
                cache.attention(q, bad)
        for bad in (pos.long(), pos[:1], pos.cpu(), i32([0, 0, 1, 1])[::2]):
            with pytest.raises(qa.QphError, match="pos|device"):
                cache.attention(q, bad)
            with pytest.raises(qa.QphError, match="lens|device"):
                cache.attention(q, pos, lens=bad)
        with pytest.raises(qa.QphError, match="numbers of tokens"):
            cache.write(k, k[:, :2], pos)
        with pytest.raises(qa.QphError, match="q's shape"):
            cache.attention(q, pos, out=q[:, :2])
        with pytest.raises(qa.QphError, match="same type"):
            cache.attention(q, pos, out=q.float())
        with pytest.raises(qa.QphError, match="multiple of kv_heads"):
            cache.attention(q[:, :, :3], pos)
        with pytest.raises(qa.QphError, match="negative"):
            cache.attention(q, pos, window=-1)
        with pytest.raises(qa.QphError, match="scale"):
            cache.attention(q, pos, scale=1e-60)   # 0 as a float, which means the default
        with pytest.raises(qa.QphError, match="overlap"):
            cache.read(pos, 3, out=(k, k))
        with pytest.raises(qa.QphError, match="overlap"):
            cache.attention(q, pos, out=torch.zeros(1, 3, 4, 64, device="cuda", dtype=F16).expand(2, 3, 4, 64))
        cache.write(k[:, :0], k[:, :0], pos)
        assert cache.attention(q[:, :0], pos).shape == (2, 0, 4, 64)
    for bad in (torch.zeros(2, 2, 5, 575, device="cuda", dtype=torch.uint8), torch.zeros(2, 2, 5, 576, device="cuda")):
        with pytest.raises(qa.QphError, match="uint8"):
            qa.KvCache("q4", 2, 2, 64, 40, data=bad)
    with pytest.raises(qa.QphError, match="fp16"):
        qa.KvCache("f16", 2, 2, 64, 40, data=(k, k))
    with pytest.raises(qa.QphError, match="head_dim"):
        qa.KvCache("q4", 2, 2, 80, 40)
    with pytest.raises(qa.QphError, match="kind"):
        qa.KvCache("q8", 2, 2, 64, 40)
