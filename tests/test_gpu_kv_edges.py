"""KvCache.attention at its edges: rows that take no part beside rows that do, values at the ends of their types' ranges.  Where a call is
compared with another one of the same kernel over the same tokens, the two are to agree to the bit."""
import math

import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv import BF16, F16, F32, TYPES, filled, held, i32, reference, route  # noqa: E402, F401


def check_loud(got, q, K, V, P0, **mask):
    """test_gpu_kv's bound for rows whose softmax picks few positions: where their V is 0 an output is as small as the weights of the
    others, and fp16's last place is no longer relative.  Below 2^-14 it is 2^-24, so an fp16 output is rounded by up to 2^-25.  A weight is an
    fp16 operand with 2^8 in the place of the largest, or more: one below 2^-14 is rounded by up to 2^-25, which is 2^-33 of the largest, and
    the sum of weights that divides it is no smaller than the largest."""
    reference.two = q.dtype == F32
    o, A, ds = reference(q.double().cpu(), K, V, P0, **mask)
    rep = q.shape[1] // V.shape[1]
    floor = 2.0 ** -33 * V[:P0 + q.shape[0]].abs().sum(0).repeat_interleave(rep, 0)
    tol = A * ((2.0 ** -21 if q.dtype == F32 else 2.0 ** -11) + 2 * ds) + torch.finfo(q.dtype).eps / 2 * o.abs() + floor + (2.0 ** -25 if q.dtype == F16 else 0)
    err = (got.double().cpu() - o).abs()
    assert bool((err <= tol).all()), f"{int((~(err <= tol)).sum())} of {err.numel()} off, worst {float((err / tol).nan_to_num(1e9).max()):.2f} tolerances"


# ------------------------------------------------------------------ rows that take no part
# n * rep a multiple of neither 8, 16 nor 256: the last chunk has columns behind the last token
@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,rep,past,window", [(3, 7, 900, 0), (1, 5, 40, 0), (5, 3, 700, 90), (75, 7, 333, 0), (41, 7, 500, 64)])
def test_over_q_as_beside_it(kind, type, n, rep, past, window, route):
    """out = q: no workgroup reads another one's rows, whose results may be there already"""
    print(f"over q: {kind} {type} n {n} rep {rep} past {past} window {window}", flush=True)
    gen = torch.Generator().manual_seed(n + rep)
    S, G, D = 3, 2, 64
    c, K, V = filled(kind, S, G, D, past + n, [past + n] * S, gen)
    # loud rows: the maxima move often
    q = (torch.randn(S, n, G * rep, D, generator=gen) * 6).to(TYPES[type]).cuda()
    pos = i32([past, past // 2, past])
    want = c.attention(q, pos, window=window)
    for _ in range(8):
        x = q.clone()
        assert c.attention(x, pos, window=window, out=x) is x
        assert torch.equal(x, want)
    check_loud(want[0], q[0], K[0], V[0], past, window=window)


@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,lens,rep,past", [(6, [3, 6, 1], 7, 3000), (2, [1, 2, 0], 4, 600), (60, [7, 60, 33], 5, 1500)])
def test_padding_rows_change_no_bit(kind, type, n, lens, rep, past, route):
    """what rows at and past lens[b] hold: zeros, values that outgrow every maximum, NaN, infinities"""
    print(f"padding: {kind} {type} n {n} lens {lens} rep {rep} past {past}", flush=True)
    gen = torch.Generator().manual_seed(n + past)
    S, G, D = 3, 1, 128
    c, K, V = filled(kind, S, G, D, past + n, [past + n] * S, gen)
    q = (torch.randn(S, n, G * rep, D, generator=gen) * 3).to(TYPES[type]).cuda()
    outs = []
    for fill in (0.0, 300 * torch.randn(n, G * rep, D, generator=gen), math.nan, math.inf):
        x = q.clone()
        for b, m in enumerate(lens):
            x[b, m:] = fill if isinstance(fill, float) else fill[m:].to(x)
        out = torch.full_like(x, 55.)
        c.attention(x, i32([past] * S), lens=i32(lens), out=out)
        outs.append(out)
    for o in outs[1:]:
        assert torch.equal(o, outs[0])
    for b, m in enumerate(lens):
        if m:
            check_loud(outs[0][b, :m], q[b, :m], K[b], V[b], past)
        assert bool((outs[0][b, m:] == 55).all())


# ------------------------------------------------------------------ values at the ends of their ranges
@pytest.mark.parametrize("kind", ["q4", "f16"])
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2, 70])
def test_queries_of_the_largest_size(kind, type, n, route):
    """rows with magnitudes of 2^127 and above, and a softmax scale that brings the scores back"""
    gen = torch.Generator().manual_seed(17)
    c, K, V = filled(kind, 1, 1, 64, 200, [200], gen)
    q = torch.randn(1, n, 4, 64, generator=gen) * 2.0 ** 122
    q.scatter_(3, torch.randint(0, 64, (1, n, 4, 1), generator=gen), 2.0 ** 127 * (1 + 0.98 * torch.rand(1, n, 4, 1, generator=gen)))
    q = q.to(TYPES[type]).cuda()
    assert bool((q.abs().amax(-1) >= 2.0 ** 127).all()) and bool(torch.isfinite(q).all())
    out = c.attention(q, i32([200 - n]), scale=2.0 ** -125)
    check_loud(out[0], q[0], K[0], V[0], 200 - n, scale=2.0 ** -125)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 70])
def test_scores_of_zero_under_the_largest_factors(type, n, route):
    """the scale times the rows' magnitude passes fp32, the scores are 0: all positions weigh alike"""
    gen = torch.Generator().manual_seed(18)
    c, _, V = filled("f16", 1, 1, 64, 200, [200], gen)
    c.data[0].zero_()
    q = (torch.randn(1, n, 4, 64, generator=gen) * 2.0 ** 100).to(TYPES[type]).cuda()
    out = c.attention(q, i32([200 - n]), scale=1e20)
    check_loud(out[0], q[0], torch.zeros_like(V[0]), V[0], 200 - n, scale=1e20)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 70])
@pytest.mark.parametrize("hd", [64, 128])
def test_infinite_keys(type, n, hd, route):
    """an fp32 key past fp16's range is infinite in an fp16 cache: where its score is -inf the position has no weight, where it is +inf the
    row is NaN, as the formula has it"""
    gen = torch.Generator().manual_seed(19)
    past, at, rep = 190, 77, 4
    c, K, V = filled("f16", 1, 1, hd, past + n, [past + n], gen)
    k, v = c.read(i32([at]), 1, dtype=F32)
    q = (torch.randn(1, n, rep, hd, generator=gen) * 1.5).to(TYPES[type])
    # head 0: exact in fp16; the others: halves of either sign, or as the type has them; the last one on the side that is NaN
    q[:, :, 0, 5], q[:, :, 1, 5], q[:, :, 2, 5] = -1.0, -1.0001, -0.9999
    q[:, :, 3, 5] = 0.7
    q = q.cuda()
    rest = [p for p in range(past + n) if p != at]
    for key, sign in ((1e5, 1), (-1e5, -1)):
        k[..., 5] = key
        c.write(k, v, i32([at]))
        x = q * sign
        out = c.attention(x, i32([past]))
        assert bool(torch.isnan(out[0, :, 3]).all())
        check_loud(out[0, :, :3], x[0, :, :3], K[0][rest], V[0][rest], past - 1)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,where,window", [(5, 2, 0), (5, 1, 3), (90, 40, 0), (90, 20, 33), (1, 0, 0), (1, -20, 0), (5, -30, 0), (90, -40, 0), (300, -40, 0)])
def test_infinite_values(type, n, where, window, route):
    """an infinite V element of a position that some tokens see, or all: theirs is infinite, the others' as it was"""
    gen = torch.Generator().manual_seed(20)
    past, rep, D = 45, 4, 64
    c, K, V = filled("f16", 1, 1, D, past + n, [past + n], gen)
    k, v = c.read(i32([past + where]), 1, dtype=F32)
    v[..., 5], v[..., 9] = math.inf, -math.inf
    c.write(k, v, i32([past + where]))
    q = torch.randn(1, n, rep, D, generator=gen).to(TYPES[type]).cuda()
    out = c.attention(q, i32([past]), window=window)
    for t in range(n):
        got, W = out[0, t:t + 1].clone(), V[0].clone()
        if t >= where and (not window or t < where + window):
            assert bool((got[..., 5] == math.inf).all()) and bool((got[..., 9] == -math.inf).all())
            got[..., [5, 9]] = 0
            W[..., [5, 9]] = 0
        check_loud(got, q[0, t:t + 1], K[0], W, past + t, window=window)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_rows_written_again_from_the_smallest_scales_on(type):
    """scales of a few of fp16's least steps are rounded anew, from 7 of them on rows stay as they are"""
    step = 2.0 ** -24
    tops = torch.cat([torch.arange(1, 64 * 60) / 64, torch.arange(60, 4000, 7).float()])   # groups' largest values in steps
    x = torch.zeros(1, len(tops), 1, 64)
    x[0, :, 0, 3], x[0, :, 0, 40] = tops * step, -tops * step
    x[0, :, 0, 9], x[0, :, 0, 50] = tops * step * 0.4, tops * step * 0.7
    x = x.to(TYPES[type])
    n, pos = x.shape[1], i32([0])
    a, b = qa.KvCache("q4", 1, 1, 64, n), qa.KvCache("q4", 1, 1, 64, n)
    a.write(x.cuda(), x.cuda(), pos)
    once = a.read(pos, n, dtype=F32)
    assert all(torch.equal(r.cpu(), held(x).float()) for r in once)
    b.write(*(r.to(TYPES[type]) if type != "bf16" else r for r in once), pos)
    again = b.read(pos, n, dtype=F32)
    assert all(torch.equal(r.cpu(), held(once[0].cpu()).float()) for r in again)
    s = (x.float().abs().amax(-1) / 7).to(BF16).half().float()[0, :, 0] / step   # both groups' scales
    same = (once[0] == again[0]).all(-1).cpu()[0, :, 0]
    assert bool(same[s >= 7].all())
    assert set(s[~same].tolist()) <= {2.0, 4.0, 5.0, 6.0} and (type == "bf16" or not bool(same.all()))
    if type == "f32":   # a largest of 10.7 steps: 2 x 5, then 1 x 7
        x = torch.full((1, 1, 1, 64), 10.7 * step)
        a.write(x.cuda(), x.cuda(), pos)
        r = a.read(pos, 1, dtype=F32)
        assert bool((r[0] == 10 * step).all())
        a.write(*r, pos)
        assert bool((a.read(pos, 1, dtype=F32)[0] == 7 * step).all())


def test_single_axes_with_strides_of_no_meaning():
    gen = torch.Generator().manual_seed(23)
    k = torch.randn(1, 40, 2, 64, generator=gen).half().cuda()
    data = [x.as_strided((1, 40, 2, 64), st) for x, st in ((k.clone(), (3, 128, 64, 1)), (k.flip(1).contiguous(), (0, 128, 64, 1)))]
    c = qa.KvCache("f16", 1, 2, 64, 40, data=data)
    q = torch.randn(1, 5, 4, 64, generator=gen).half().cuda()
    check_loud(c.attention(q, i32([35]))[0], q[0], data[0][0].cpu().double(), data[1][0].cpu().double(), 35)
    one = qa.KvCache("f16", 3, 1, 64, 1)
    x = torch.randn(3, 1, 1, 64, generator=gen).half().cuda()
    one.write(x, x * 2, i32([0, 0, 0]))
    assert torch.equal(one.attention(x, i32([0, 0, 0])), x * 2)
