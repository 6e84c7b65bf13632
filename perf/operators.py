"""The key / value cache's operators: what is timed of them, and their plain forms.

  write   rows quantised into a 4-bit cache as they are written, and read back as the values it then holds
  attend  causal attention of n new tokens a sequence over such a cache or over an fp16 one, all of it or a sliding
          window with a few first positions that stay visible

A 4-bit cache is one record of 9 head_dim bytes per (sequence, kv head, 8 positions):
  K codes   position i at bytes i head_dim / 2; a row's 32-bit word w holds dims 8 w .. 8 w + 7, dim 8 w + 2 e + o at bits 16 o + 4 e
  V codes   at bytes 4 head_dim: dim d in the word (d % 16) (head_dim / 16) + d / 16, position 2 e + o at bits 16 o + 4 e
  K scales  at bytes 8 head_dim: fp16 [8 positions][head_dim / 32]
  V scales  at bytes 8.5 head_dim: fp16 [head_dim / 32][8 positions]
and stands for (code - 8) * scale."""
import torch

own = False

F16, Q4 = "f16", "q4"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, kind, type, nseq, n, past, heads, kv_heads, head_dim, ctx, ragged=False, window=0, sinks=0):
    return dict(name=name, op=op, kind=kind, type=type, nseq=nseq, n=n, past=past, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                ctx=ctx, ragged=ragged, window=window, sinks=sinks)


def listed():
    return [
        # the cache's side of one decode step of the 8B shape, and of a prompt; two-head ragged batch at odd positions
        _case("write_step", "write", Q4, "f32", 1, 1, 9001, 32, 8, 128, 16384),
        _case("write_prompt", "write", Q4, "f16", 1, 2048, 0, 32, 8, 128, 4096),
        _case("write_ragged", "write", Q4, "bf16", 6, 777, 1203, 14, 2, 64, 2100, ragged=True),
        # decode: the 0.5B shape in a short chat, the 7B one at 16K positions, a server's batch of the 8B one
        _case("q4_step_short", "attend", Q4, "f32", 1, 1, 332, 14, 2, 64, 1024),
        _case("q4_step_long", "attend", Q4, "f16", 1, 1, 16383, 28, 4, 128, 16400),
        _case("q4_batch", "attend", Q4, "bf16", 32, 1, 8191, 32, 8, 128, 8192, ragged=True),
        # four drafted tokens verified at once; a prompt; a short turn behind a long conversation
        _case("q4_verify", "attend", Q4, "bf16", 2, 4, 12001, 32, 8, 128, 16384),
        _case("q4_prompt", "attend", Q4, "f16", 1, 2048, 0, 32, 8, 128, 4096),
        _case("q4_turn", "attend", Q4, "bf16", 1, 77, 16000, 28, 4, 128, 16384),
        # the window: a batch far into its texts, a prompt longer than it, one step over a 4-bit cache of 100K positions
        _case("window_batch", "attend", F16, "f16", 4, 1, 30000, 32, 8, 128, 32768, ragged=True, window=4096, sinks=4),
        _case("window_prompt", "attend", F16, "f16", 1, 4096, 0, 32, 8, 128, 4096, window=1024, sinks=4),
        _case("q4_window_step", "attend", Q4, "bf16", 1, 1, 100003, 28, 4, 128, 102400, window=2048, sinks=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    while True:
        op = rng.choice(["write", "attend", "attend"])
        head_dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        rep = rng.choice([1, 2, 3, 4, 5, 7, 8])
        nseq = _log(rng, 1, 32)
        n = 1 if rng.random() < 0.4 else _log(rng, 2, 2048)
        past = 0 if rng.random() < 0.15 else _log(rng, 1, 30000)
        kind = Q4 if op == "write" or rng.random() < 0.6 else F16
        window, sinks = (_log(rng, 1, 5000), rng.choice([0, 1, 4, 16, 33])) if op == "attend" and (kind == F16 or rng.random() < 0.3) else (0, 0)
        c = _case("", op, kind, rng.choice(["f32", "f16", "bf16"]), nseq, n, past, kv_heads * rep, kv_heads, head_dim,
                  past + n + rng.randrange(0, 70), ragged=rng.random() < 0.5, window=window, sinks=sinks)
        del c["name"]
        if nseq * n * (past + n) * c["heads"] <= 2 ** 28 and nseq * c["ctx"] * kv_heads * head_dim <= 2 ** 28 and work(c)["flops"] < 3e10:
            return c


def _places(case):
    """each sequence's first position and its number of new tokens"""
    S, n, past = case["nseq"], case["n"], case["past"]
    if not case["ragged"]:
        return [past] * S, [n] * S
    return [past - past * b * 5 // (8 * S) for b in range(S)], [max(1, n - n * b // (2 * S)) for b in range(S)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    S, n, G, D, ctx, t = case["nseq"], case["n"], case["kv_heads"], case["head_dim"], case["ctx"], TYPES[case["type"]]
    randn = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    # keys have a few channels that are larger throughout, as rotated keys do
    loud = 1 + 3 * (torch.rand(G, D, generator=g, device="cuda") < 0.06).float()
    pos, lens = _places(case)
    s = {"case": case, "pos": torch.tensor(pos, dtype=torch.int32, device="cuda"), "lens": torch.tensor(lens, dtype=torch.int32, device="cuda") if case["ragged"] else None,
         "upto": max(p + m for p, m in zip(pos, lens))}
    if case["op"] == "write":
        s["k"], s["v"] = (randn(S, n, G, D) * loud).to(t), randn(S, n, G, D).to(t)
        s["data"] = torch.zeros(S, G, (ctx + 7) // 8, 9 * D, dtype=torch.uint8, device="cuda")
        s["out"] = (torch.zeros(S, n, G, D, dtype=t, device="cuda"), torch.zeros(S, n, G, D, dtype=t, device="cuda"))
        return s
    s["q"] = randn(S, n, case["heads"], D).to(t)
    s["out"] = torch.zeros(S, n, case["heads"], D, dtype=t, device="cuda")
    if case["kind"] == F16:
        s["data"] = (randn(S, ctx, G, D, dtype=torch.float16) * loud.half(), randn(S, ctx, G, D, dtype=torch.float16))
        return s
    # the cache's contents: normal values' codes, and scales near those of their groups
    nb = (ctx + 7) // 8
    code = torch.randn(S, G, nb, 16 * D, generator=g, device="cuda", dtype=torch.float16).mul_(3).round_().clamp_(-7, 7).add_(8).to(torch.uint8)
    scale = (0.25 + 0.2 * torch.rand(S, G, nb, D // 2, generator=g, device="cuda")).bfloat16().half()
    s["data"] = torch.cat([code[..., 0::2] | code[..., 1::2] << 4, scale.view(torch.uint8)], -1)
    return s


def _shifts(device):
    e = torch.arange(8, device=device)
    return (16 * (e % 2) + 4 * (e // 2)).int()


def _values(data, ctx):
    """the records' values: K and V as fp32 [sequence][kv head][position][dim]"""
    S, G, nb, D = data.shape[0], data.shape[1], (ctx + 7) // 8, data.shape[3] // 9
    r, sh = data[:, :, :nb], _shifts(data.device)
    kw = r[..., :4 * D].view(torch.int32).reshape(S, G, nb, 8, D // 8, 1)
    k = (((kw >> sh) & 15) - 8).view(S, G, nb, 8, D // 32, 32) * r[..., 8 * D:8 * D + D // 2].view(torch.float16).float().view(S, G, nb, 8, D // 32, 1)
    vw = r[..., 4 * D:8 * D].view(torch.int32).reshape(S, G, nb, 16, D // 16).transpose(3, 4).reshape(S, G, nb, 1, D)
    v = (((vw >> sh.view(8, 1)) & 15) - 8).view(S, G, nb, 8, D // 32, 32)
    v = v * r[..., 8 * D + D // 2:].view(torch.float16).float().view(S, G, nb, D // 32, 8).transpose(3, 4).unsqueeze(-1)
    return k.reshape(S, G, 8 * nb, D)[:, :, :ctx], v.reshape(S, G, 8 * nb, D)[:, :, :ctx]


def _rounded(x):
    """what a 4-bit cache holds of these rows; the codes in 64 bits, where a value may lie next to a border"""
    y = x.float().unflatten(-1, (-1, 32))
    a = y.abs().amax(-1, keepdim=True)
    s = (a.clamp(max=65504) / 7).bfloat16().half().double()
    s = torch.where(torch.isfinite(a), s, torch.nan)
    c = torch.where(s == 0, 0, (y.double() / s).round().clamp(-7, 7))
    return (c * s).flatten(-2)


def _live(s):
    """[sequence][token]: whether the sequence has this token"""
    t = torch.arange(s["case"]["n"], device="cuda")
    return (t < s["lens"].unsqueeze(1)) if s["lens"] is not None else torch.ones(s["case"]["nseq"], s["case"]["n"], dtype=torch.bool, device="cuda")


def _plain_write(s):
    keep = _live(s)[:, :, None, None]
    return torch.where(keep, _rounded(s["k"]), 0).to(s["k"].dtype), torch.where(keep, _rounded(s["v"]), 0).to(s["v"].dtype)


def _plain_attend(s):
    c = s["case"]
    S, n, H, G, D, T = c["nseq"], c["n"], c["heads"], c["kv_heads"], c["head_dim"], s["upto"]
    if c["kind"] == F16:
        k, v = (x[:, :T].float().transpose(1, 2) for x in s["data"])
    else:
        k, v = _values(s["data"], T)
    q = s["q"].float().view(S, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(S, G, H // G * n, D)
    x = (torch.matmul(q, k.transpose(2, 3).contiguous()) / D ** 0.5).view(S, G, H // G, n, T)
    P = s["pos"].view(S, 1, 1, 1, 1) + torch.arange(n, device="cuda").view(n, 1)
    p = torch.arange(T, device="cuda")
    seen = p <= P
    if c["window"]:
        seen = seen & ((p > P - c["window"]) | (p < c["sinks"]))
    x = x.masked_fill_(~seen, float("-inf"))
    e = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(e.view(S, G, H // G * n, T), v.contiguous()).view(S, G, H // G, n, D) / e.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, n, H, D)
    return torch.where(_live(s)[:, :, None, None], o, 0).to(s["q"].dtype)


def run(state):
    c = state["case"]
    if own:
        import qpack_amd
        if "cache" not in state:   # the handle that a program keeps beside the cache's memory
            state["cache"] = qpack_amd.KvCache(c["kind"], c["nseq"], c["kv_heads"], c["head_dim"], c["ctx"], data=state["data"])
        cache = state["cache"]
        if c["op"] == "write":
            cache.write(state["k"], state["v"], state["pos"], lens=state["lens"])
            return cache.read(state["pos"], c["n"], lens=state["lens"], out=state["out"])
        return cache.attention(state["q"], state["pos"], lens=state["lens"], window=c["window"], sinks=c["sinks"], out=state["out"])
    return _plain_write(state) if c["op"] == "write" else _plain_attend(state)


def _seen(case, pos, n):
    """visible positions summed over the tokens pos .. pos + n - 1, and the positions that any of them sees"""
    W, K = case["window"], case["sinks"]
    if not W:
        return sum(range(pos + 1, pos + n + 1)), pos + n
    pairs = 0
    for P in range(pos, pos + n):
        a = max(0, P + 1 - W)
        pairs += P + 1 - a + min(K, a)
    a = max(0, pos + 1 - W)
    return pairs, pos + n - a + min(K, a)


def work(case):
    pos, lens = _places(case)
    size, G, D, H = TYPES[case["type"]].itemsize, case["kv_heads"], case["head_dim"], case["heads"]
    held = 2 * G * D * (2 if case["kind"] == F16 else 9 / 16)   # bytes of a position in the cache
    tokens = sum(lens)
    if case["op"] == "write":   # rows in, records out; records in, rows out
        return {"bytes": tokens * (2 * 2 * G * D * size + 2 * held), "flops": tokens * 2 * G * D * 4}
    seen = [_seen(case, p, m) for p, m in zip(pos, lens)]
    return {"bytes": 2 * tokens * H * D * size + sum(x[1] for x in seen) * held, "flops": 4 * D * H * sum(x[0] for x in seen)}


def exact(case, seed):
    s = prepare(case, seed)
    pos, lens = _places(case)
    if case["op"] == "write":
        def stands_for(x, m):
            x = x[:m].double()
            m, G, D = x.shape
            x = x.reshape(m, G, D // 32, 32)
            top = x.abs().max(-1, keepdim=True).values.minimum(torch.tensor(65504., dtype=torch.float64, device="cuda"))
            step = (top / 7).to(torch.float32).to(torch.bfloat16).to(torch.float16).double()
            code = torch.div(x, step).round().clip(-7, 7)
            return torch.where(step > 0, code * step, torch.zeros_like(x)).reshape(m, G, D)
        outs = tuple(torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (s["k"], s["v"]))
        for b, m in enumerate(lens):
            for o, x in zip(outs, (s["k"], s["v"])):
                o[b, :m] = stands_for(x[b], m)
        return outs
    H, G, D, W = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    out = torch.zeros(case["nseq"], case["n"], H, D, dtype=torch.float64, device="cuda")
    bits = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device="cuda")
    for b, (p0, m) in enumerate(zip(pos, lens)):
        T = p0 + m
        for h in range(G):
            if case["kind"] == F16:
                k, v = s["data"][0][b, :T, h].double(), s["data"][1][b, :T, h].double()
            else:
                r = s["data"][b, h]
                nb = r.shape[0]
                word = r[:, :8 * D].contiguous().view(torch.int32).view(nb, 2 * D, 1)
                nib = ((word >> bits) & 15).double() - 8
                sc = r[:, 8 * D:].contiguous().view(torch.float16).double()
                k = (nib[:, :D].reshape(nb, 8, D // 32, 32) * sc[:, :D // 4].reshape(nb, 8, D // 32, 1)).reshape(8 * nb, D)[:T]
                vd = nib[:, D:].view(nb, 16, D // 16, 8).permute(0, 3, 2, 1).reshape(nb, 8, D)
                v = (vd.view(nb, 8, D // 32, 32) * sc[:, D // 4:].view(nb, D // 32, 8).transpose(1, 2).unsqueeze(-1)).reshape(8 * nb, D)[:T]
            for t0 in range(0, m, 512):
                t1 = min(m, t0 + 512)
                q = s["q"][b, t0:t1, h * (H // G):(h + 1) * (H // G)].double()
                at = p0 + torch.arange(t0, t1, device="cuda").view(-1, 1, 1)
                p = torch.arange(T, device="cuda")
                hidden = p > at
                if W:
                    hidden = hidden | ((p <= at - W) & (p >= case["sinks"]))
                x = (q.reshape(-1, D) @ k.T.contiguous() / D ** 0.5).view(t1 - t0, H // G, T)
                w = torch.softmax(x.masked_fill(hidden, -torch.inf), -1)
                out[b, t0:t1, h * (H // G):(h + 1) * (H // G)] = (w.reshape(-1, T) @ v).view(t1 - t0, H // G, D)
    return out
