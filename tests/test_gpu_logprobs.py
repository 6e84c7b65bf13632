"""qpack_amd.logprobs against 64-bit arithmetic.

Tolerances.  With d = x - m (m within 6 of the maximum of what has been seen) an e^d is off by 2^-24 (2 |d| + 6) of itself: the difference's and the product's rounding, and two last places of the
exponential.  A thread sums V / 256 values or fewer, taken as sqrt(V / 256) 2^-23, and the tree adds 2^-21.  So ln s is off by ds = 2^-24 (2 sum p |d| + 6) + sqrt(V / 256) 2^-23 + 2^-21, with sum p |d| at most
the entropy plus 14; a log probability by that and by the roundings of x - m, of ln s and of their difference, 2^-23 (|logp| + 20); the entropy by ds (2 + its size) and 2^-22 (its size + 7)."""
import math

import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def check(r, x, tokens, K):
    x = x.double().cpu()
    R, V = x.shape
    y = torch.log_softmax(x, -1)
    H = -torch.special.xlogy(y.exp(), y.exp()).sum(-1)
    ds = 2.0 ** -24 * (2 * (H + 14) + 6) + math.sqrt(V / 256) * 2.0 ** -23 + 2.0 ** -21
    assert bool(((r.entropy.cpu() - H).abs() <= ds * (2 + H) + 2.0 ** -22 * (H + 7)).all()), float((r.entropy.cpu() - H).abs().max())
    order = x.sort(dim=-1, descending=True, stable=True).indices
    if tokens is not None:
        for i, t in enumerate(tokens.tolist()):
            if not 0 <= t < V:
                assert math.isnan(r.logp[i]) and int(r.rank[i]) == -1
                continue
            want, got = float(y[i, t]), float(r.logp[i])
            assert want == got or abs(got - want) <= ds[i] + 2.0 ** -23 * (abs(want) + 20), (i, t, got, want)
            assert int(r.rank[i]) == int((x[i] > x[i, t]).sum() + (x[i, :t] == x[i, t]).sum())
    assert torch.equal(r.top_index.cpu().long(), order[:, :K])
    want = y.gather(1, order[:, :K])
    err = (r.top_logp.cpu() - want).abs().nan_to_num(0, posinf=0)   # (-inf of -inf)
    assert bool((err <= ds.unsqueeze(1) + 2.0 ** -23 * (want.abs().nan_to_num(posinf=0) + 20)).all())
    assert torch.equal(torch.isinf(r.top_logp.cpu()), torch.isinf(want))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 1), (3, 7, 7), (1, 63, 63), (5, 64, 64), (2, 255, 0), (7, 256, 20), (1, 257, 5), (4, 511, 64), (2, 513, 64), (33, 1000, 1), (1, 1025, 64),
                                            (3, 2047, 10), (2, 2049, 64), (1, 5000, 64), (64, 8191, 3), (2, 32000, 20), (1, 128256, 64), (3, 151936, 20), (300, 999, 2), (1100, 4097, 1)])
def test_logprobs(type, rows, vocab, top):
    print(f"logprobs {type} {rows} x {vocab} top {top}", flush=True)
    gen = torch.Generator().manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=gen) * 3).to(TYPES[type])   # (16 bits: many equal ones)
    x[0, vocab // 2:] = float(x[0, vocab // 2])
    tokens = torch.randint(0, vocab, (rows,), generator=gen)
    tokens[0] = vocab - 1
    if rows > 2:
        tokens[1], tokens[2] = -1, vocab
    check(qa.logprobs(x.cuda(), tokens.int().cuda(), top), x, tokens, top)


@pytest.mark.parametrize("rows", [1, 5, 1500])
def test_orders_that_insert_often(rows):
    """rising and falling rows, plateaus, the largest at either end, the smallest steps of a type"""
    V = 6007
    up = torch.arange(V).float() / 100
    x = torch.stack([up, up.flip(0), (up / 7).floor(), torch.zeros(V), -up, up.neg().exp(), torch.where(up > 30, up, -up), up % 3])
    x = x.repeat((rows + 7) // 8, 1)[:rows]
    tokens = torch.arange(rows) * 977 % V
    check(qa.logprobs(x.cuda(), tokens.int().cuda(), 64), x, tokens, 64)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V", [(1, 9001), (1030, 3001)])
def test_masked_logits(type, rows, V):
    """-inf entries: a few, all but a few (fewer than top), all but one; at the ends of shares"""
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(rows, V, generator=gen).to(TYPES[type])
    tokens = torch.randint(0, V, (rows,), generator=gen)
    base = x.clone()
    for keep in ([range(0, V, 2)], [[5, 700, 2999]], [[V - 1]], [[0]], [range(256, 300)]):
        x.fill_(-math.inf)
        for i in keep:
            x[:, list(i)] = base[:, list(i)]
        tokens[0] = list(keep[0])[-1]
        check(qa.logprobs(x.cuda(), tokens.int().cuda(), 10), x, tokens, 10)
    x.fill_(float(torch.finfo(TYPES[type]).min))   # a mask of the type's lowest value
    x[:, 17], x[:, V - 2] = 3., 2.
    check(qa.logprobs(x.cuda(), tokens.int().cuda(), 4), x, tokens, 4)


def test_values_far_from_zero_and_zeros_of_both_signs():
    V = 3000
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(6, V, generator=gen)
    x[0] += 1e4
    x[1] -= 1e4
    x[2] = torch.where(torch.arange(V) % 2 == 0, 0., -0.)
    x[3] *= 50
    x[4, 1234] = 200.
    x[5] *= 1e-30
    tokens = torch.tensor([5, 6, 2999, 8, 1234, 9])
    r = qa.logprobs(x.cuda(), tokens.int().cuda(), 20)
    y = x.clone()
    y[2] = 0.   # (as equal as they compare)
    # the spacing of values near 1e4 is 2^-10: exact in fp32, and in the differences
    check(r, y, tokens, 20)


def test_not_finite_rows():
    x = torch.randn(5, 2500, device="cuda")
    x[0, 77] = math.nan
    x[1, 2000] = math.inf
    x[2] = -math.inf
    r = qa.logprobs(x, torch.zeros(5, dtype=torch.int32, device="cuda"), 5)
    for i in range(3):
        assert math.isnan(r.logp[i]) and math.isnan(r.entropy[i]) and bool(torch.isnan(r.top_logp[i]).all())
        assert bool(((r.top_index[i] >= -1) & (r.top_index[i] < 2500)).all())
    assert torch.equal(r.top_index[2].cpu(), torch.arange(5, dtype=torch.int32))
    check(qa.LogProbs(*(y[3:] for y in r)), x[3:], torch.zeros(2, dtype=torch.int64), 5)
    full = torch.full((2, 600), math.nan, device="cuda")
    r = qa.logprobs(full, torch.zeros(2, dtype=torch.int32, device="cuda"), 5)
    assert bool(torch.isnan(r.logp).all()) and bool((r.top_index < 600).all())


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top", [1, 64])
def test_nan_before_what_rises(type, top):
    # each wave's first load is NaN and every later one passes its bound: what it keeps stays within its room, and the row beside it is right
    V = 40000
    x = torch.linspace(-20, 20, V).repeat(3, 1)
    x[0, :4096] = math.nan
    x[1, torch.randperm(V, generator=torch.Generator().manual_seed(top))[: V // 2]] = math.nan
    x = x.to(dict(f32=torch.float32, f16=torch.float16, bf16=torch.bfloat16)[type]).cuda()
    r = qa.logprobs(x.repeat(400, 1), torch.zeros(1200, dtype=torch.int32, device="cuda"), top)
    nan = torch.arange(1200, device="cuda") % 3 < 2
    assert bool(torch.isnan(r.logp[nan]).all()) and bool(torch.isnan(r.entropy[nan]).all()) and bool(torch.isnan(r.top_logp[nan]).all())
    assert bool(((r.top_index >= -1) & (r.top_index < V)).all())
    one = qa.logprobs(x[2:], torch.zeros(1, dtype=torch.int32, device="cuda"), top)
    assert bool((r.top_index[~nan] == one.top_index).all()) and bool((r.rank[~nan] == one.rank).all())


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_strides_alignment_and_no_tokens(type):
    gen = torch.Generator().manual_seed(4)
    base = (torch.randn(9, 4003, generator=gen) * 2).to(TYPES[type]).cuda()
    for x in (base[::2, 1:], base[1:, 3:3001], base[:, :1], base[:1].expand(4, -1), base.t().contiguous().t()[:1]):
        if x.stride(1) != 1 and x.shape[1] > 1:
            with pytest.raises(qa.QphError, match="contiguous rows"):
                qa.logprobs(x)
            continue
        K = min(6, x.shape[1])
        r = qa.logprobs(x, top=K)
        assert r.logp is None and r.rank is None
        check(r, x, None, K)
    r = qa.logprobs(base)
    assert r.top_index.shape == (9, 0) and r.top_logp.shape == (9, 0)
    r = qa.logprobs(base[:0], torch.zeros(0, dtype=torch.int32, device="cuda"), 3)
    assert r.logp.shape == (0,) and r.top_index.shape == (0, 3)


def test_row_by_row_is_all_at_once_in_indices_and_close_in_values():
    gen = torch.Generator().manual_seed(5)
    x = (torch.randn(40, 30001, generator=gen) * 3).half().cuda()
    t = torch.arange(40, dtype=torch.int32, device="cuda")
    whole = qa.logprobs(x, t, 8)
    again = qa.logprobs(x, t, 8)
    for a, b in zip(whole, again):
        assert torch.equal(a, b)
    for i in range(0, 40, 7):
        one = qa.logprobs(x[i:i + 1], t[i:i + 1], 8)
        check(one, x[i:i + 1], t[i:i + 1].cpu(), 8)
        assert torch.equal(one.top_index[0], whole.top_index[i]) and int(one.rank) == int(whole.rank[i])


@pytest.mark.parametrize("rows,vocab", [(1, 50000), (1200, 2001)])
def test_graph_and_other_stream(rows, vocab):
    gen = torch.Generator().manual_seed(6)
    x, t = torch.randn(rows, vocab, generator=gen).cuda(), torch.zeros(rows, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = qa.logprobs(x, t, 5)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = qa.logprobs(x, t, 5)
    for k in range(4):
        if k:
            x.copy_(torch.randn(rows, vocab, generator=gen))
            t.fill_(7 * k)
        g.replay()
        want = qa.logprobs(x, t, 5)
        torch.cuda.synchronize()
        for a, b in zip(r, want):
            assert torch.equal(a, b)
        if not k:
            for a, b in zip(other, want):
                assert torch.equal(a, b)


def test_refusals():
    x, t = torch.zeros(2, 100, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad, words in ((x.double(), "float32, float16"), (x[0], "rows, vocab"), (x.cpu(), "GPU"), (None, "tensor"), (torch.zeros(2, 0, device="cuda"), "vocab")):
        with pytest.raises(qa.QphError, match=words):
            qa.logprobs(bad, t if words != "GPU" else None)
    for bad in (t.long(), t[:1], t.unsqueeze(0), t.cpu(), torch.zeros(4, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(qa.QphError, match="tokens"):
            qa.logprobs(x, bad)
    for top in (-1, 65, 101, 2 ** 40):
        with pytest.raises(qa.QphError, match="top"):
            qa.logprobs(x, t, top)
    with pytest.raises(qa.QphError, match="top"):
        qa.logprobs(x[:, :5], t, 6)
    g = torch.zeros(2, 100, device="cuda", requires_grad=True)
    with pytest.raises(qa.QphError, match="requires a gradient"):
        qa.logprobs(g, t)
    with torch.no_grad():
        assert qa.logprobs(g, t).logp.shape == (2,)


def test_the_most_rows():
    R = 1 << 23
    x = (torch.arange(2 * R, device="cuda", dtype=torch.int32) % 777).half().view(R, 2)
    r = qa.logprobs(x, (torch.arange(R, device="cuda") % 2).int(), 1)
    d = (x[:, 1] - x[:, 0]).float()
    assert torch.equal(r.top_index[:, 0].bool(), d > 0)
    # differences of whole numbers are exact; the sum 1 + e^-d is off by 2^-24 (2 d e^-d + 6) or less, its logarithm by another 2^-23, the result's rounding is 2^-24 of it
    want = -torch.nn.functional.softplus(torch.where(torch.arange(R, device="cuda") % 2 == 0, d, -d).double())
    assert bool(((r.logp - want).abs() <= 2.0 ** -20 * (1 + want.abs())).all())


def test_results_are_tensors_of_their_own():
    x, tokens = torch.randn(5, 900, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda")
    r, again = qa.logprobs(x, tokens, 3), qa.logprobs(x, tokens, 3)
    with torch.inference_mode():
        inside = qa.logprobs(x, tokens, 3)
    for i, y in enumerate(r):   # one changed, the others stay
        assert torch.equal(y, inside[i])
        assert y.is_contiguous() and y.device == x.device and not y.requires_grad and y.data_ptr() % 64 == 0
        y.fill_(7)
        for j in range(i + 1, 5):
            assert torch.equal(r[j], again[j])
    w = torch.ones(5, device="cuda", requires_grad=True)
    (again.logp * w).sum().backward()   # (as constants of a graph)
    assert torch.equal(w.grad, again.logp)
    none = qa.logprobs(x[:0], tokens[:0], 3)
    assert none.logp.shape == (0,) and none.top_index.shape == (0, 3)
    only = qa.logprobs(x)
    assert only.logp is None and only.rank is None and only.top_index.shape == (5, 0) and torch.equal(only.entropy, inside.entropy)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top", [1, 5, 64])
def test_what_reaches_the_first_bound_lies_in_the_second_load(type, top):
    # a wave's loads are 256 or 512 logits, 1024 or 2048 apart
    V = 24000
    gen = torch.Generator().manual_seed(top)
    x = torch.randn(6, V, generator=gen)
    i = torch.arange(V)
    x[0] = torch.where(i % 4096 >= 1024, x[0], -math.inf)
    x[1] = torch.where((i >= 1024) & (i < 1024 + top // 2 + 1), x[1], -math.inf)
    x[2] = torch.where(i >= 2048, x[2] + 9, x[2] - 9)
    x[3] = torch.where(i % 2048 < 1024, 3., 2.)
    x[4] = 3.
    x[5] = torch.where((i >= 2048) & (i < 4096), 5., x[5].clamp(max=4))
    x = x.to(TYPES[type])
    tokens = torch.tensor([1024, 0, 3000, 23999, 17, 2048])
    r = qa.logprobs(x.repeat(100, 1).cuda(), tokens.repeat(100).int().cuda(), top)   # (whole rows and shares of them)
    few = qa.logprobs(x.cuda(), tokens.int().cuda(), top)
    for y in (qa.LogProbs(*(z[:6] for z in r)), qa.LogProbs(*(z[594:] for z in r)), few):
        check(y, x, tokens, top)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("rows,top", [(1, 64), (9, 40), (1100, 64)])
def test_four_lists_of_many(type, rows, top):
    # every wave of a workgroup has more than a quarter of 128 of what reaches the common bound: all logits equal, or two values by turns of 1, 8 and 512
    V = 9001
    i = torch.arange(V)
    x = torch.stack([torch.zeros(V), (i % 2).float(), (i // 8 % 2).float(), (i // 512 % 2).float(), torch.where(i > 4000, 2., 1.)]).repeat((rows + 4) // 5, 1)[:rows].to(TYPES[type])
    tokens = torch.arange(rows) * 977 % V
    for _ in range(3):
        check(qa.logprobs(x.cuda(), tokens.int().cuda(), top), x, tokens, top)


@pytest.mark.parametrize("below", [1.0, -1.0, 0.0, -2.0 ** -149, 2.0 ** -149, 12345.678])
@pytest.mark.parametrize("top", [1, 5, 20, 64])
def test_plateaus_one_step_below_the_first(below, top):
    # a wave's loads are 256 logits, 1024 apart; its first bound is what `top` of the lanes' largest of two loads reach.  Much of every row is one step of fp32 below those
    below = torch.tensor(below)
    up = torch.nextafter(below, torch.tensor(math.inf))
    V = 6144
    i = torch.arange(V)
    gen = torch.Generator().manual_seed(top)
    x = below.repeat(10, V)
    x[0, 1029] = up                                               # the only one, in the second load
    x[1, 1024:1024 + 4 * (top + 3):4] = up                        # a lane each, all of them in the second load
    x[2, :4 * (top // 2):4] = up                                  # fewer than top in the first load, the others in the second
    x[2, 1024:1024 + 4 * (top - top // 2 + 1):4] = up
    x[3] = torch.where(i < 40, below, torch.nextafter(below, torch.tensor(-math.inf)))   # 40 one step below, the others two
    x[3, 1024] = up
    x[4] = torch.where(torch.rand(V, generator=gen) < 0.002, up, below)
    x[5] = torch.where(torch.rand(V, generator=gen) < 0.5, up, below)
    x[6, 5000:] = up                                              # past both loads
    x[7] = torch.where(i % 2 == 0, below, -below)
    x[7, 1300] = torch.nextafter(below.abs(), torch.tensor(math.inf))
    x[8] = torch.where(i < 1024, below, torch.nextafter(up, torch.tensor(math.inf)))
    x[8, 2048:] = -math.inf
    x[9] = torch.where(i < 2048, below, up)
    tokens = torch.tensor([1029, 0, 1024, 1024, 7, 8, 6143, 1300, 1024, 2048])
    wide = torch.cat([below.repeat(10, 128256 - V - 2100), x, below.repeat(10, 2100)], -1)   # shares of several units, what matters in the last ones
    whole = below.repeat(10, 40000)
    whole[:, :V] = x
    for y, t in ((x[:, :4096], tokens.clamp(max=4095)), (x, tokens), (whole, tokens), (wide, tokens + 128256 - V - 2100)):
        for some in (slice(0, 1), slice(2, 3), slice(0, 10)):   # (rows alone, too: other shares)
            check(qa.logprobs(y[some].cuda(), t[some].int().cuda(), top), y[some], t[some], top)
    r = qa.logprobs(x.repeat(103, 1).cuda(), tokens.repeat(103).int().cuda(), top)   # (as many rows as take no shares)
    check(qa.LogProbs(*(z[1020:] for z in r)), x, tokens, top)


def test_refused_where_another_device_is_current():
    """tensors without memory of their own (functorch's) while another device is current: refused, and that device stays current"""
    from qpack_amd import kvcache

    class Guard:   # as torch.cuda.device of the tensors' device, entered from another one
        inside = entered = 0

        def __init__(self, device):
            assert device == 0

        def __enter__(self):
            Guard.inside += 1
            Guard.entered += 1

        def __exit__(self, *error):
            Guard.inside -= 1

    x, t = torch.randn(3, 2, 700, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    kvcache._binding().setup(qa.QphError, torch._C._cuda_getCurrentRawStream, lambda: 1, Guard)
    try:
        there = qa.logprobs(x[0], t[0], 3)
        assert Guard.entered == 1 and Guard.inside == 0
        for call in (lambda: torch.func.vmap(lambda y: qa.logprobs(y))(x), lambda: torch.func.vmap(lambda u: qa.logprobs(x[0], u))(t)):
            with pytest.raises(qa.QphError, match="plain tensors"):
                call()
            assert Guard.inside == 0
    finally:
        kvcache._bind = None
        kvcache._binding()
    check(there, x[0], t[0], 3)
