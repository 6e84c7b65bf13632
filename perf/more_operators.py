"""The operators of a served batch's step beside the caches' write and attention: what is timed of them, and their plain forms.

  append    norms of queries and keys for each head, the position rotation, and keys and values into the cache
  prefix    causal attention of n new tokens a sequence over a prefix that all sequences share and their own positions
  copy      positions of a cache copied to places of another or the same one, by index
  logprobs  log probabilities of given tokens, entropy, the tokens' ranks, and the most probable alternatives

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


def _append(name, type, nseq, n, past, heads, kv_heads, head_dim, rot, norm=True, ragged=False, behind=0):
    """behind: positions of a common prefix that the rotation counts and the cache does not hold"""
    return dict(name=name, op="append", type=type, nseq=nseq, n=n, past=past, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rot=rot, norm=norm,
                ragged=ragged, behind=behind)


def _prefix(name, kind, type, nseq, n, shared, past, heads, kv_heads, head_dim, ragged=False):
    return dict(name=name, op="prefix", kind=kind, type=type, nseq=nseq, n=n, shared=shared, past=past, heads=heads, kv_heads=kv_heads, head_dim=head_dim, ragged=ragged)


def _copy(name, kind, nseq, n, source, kv_heads, head_dim, fork):
    """fork: all sequences from one of the same cache, positions in order; else of each sequence of another cache those that are kept"""
    return dict(name=name, op="copy", kind=kind, nseq=nseq, n=n, source=source, kv_heads=kv_heads, head_dim=head_dim, fork=fork)


def _logprobs(name, type, rows, vocab, top, padded=0):
    """padded: entries at the vocabulary's end that no token has (-inf)"""
    return dict(name=name, op="logprobs", type=type, rows=rows, vocab=vocab, top=top, padded=padded)


def listed():
    return [
        # one token of a 0.5B chat; a server's batch of the 8B shape behind a common prefix; a prompt of the 7B shape, half of each head rotated
        _append("append_step", "f32", 1, 1, 332, 14, 2, 64, 64, norm=False),
        _append("append_batch", "bf16", 64, 1, 900, 32, 8, 128, 128, ragged=True, behind=4096),
        _append("append_prompt", "f16", 1, 4001, 96, 28, 4, 128, 64),
        # few samples of a short prompt; a batch behind a system prompt; many behind a 4-bit document; questions of some length to one document
        _prefix("prefix_samples", F16, "f32", 4, 1, 700, 90, 14, 2, 64),
        _prefix("prefix_batch", F16, "bf16", 32, 1, 8190, 511, 32, 8, 128, ragged=True),
        _prefix("prefix_q4", Q4, "f16", 96, 1, 16411, 1000, 28, 4, 128, ragged=True),
        _prefix("prefix_questions", F16, "bf16", 8, 128, 12001, 0, 32, 8, 128, ragged=True),
        # a prompt forked into eight sequences; a quarter of each long text's positions kept
        _copy("copy_fork", Q4, 9, 6001, 6001, 8, 128, True),
        _copy("copy_keep", F16, 4, 4096, 16384, 8, 128, False),
        # a sampled token of the 8B vocabulary with 20 alternatives; a batch's of the 0.5B one, its end unused; a text scored
        _logprobs("logprobs_step", "f32", 1, 128256, 20),
        _logprobs("logprobs_batch", "bf16", 64, 151936, 5, padded=271),
        _logprobs("logprobs_text", "f32", 1023, 128256, 1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    while True:
        op = rng.choice(["append", "prefix", "prefix", "copy", "logprobs"])
        type, head_dim, kv_heads = rng.choice(["f32", "f16", "bf16"]), rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
        nseq = _log(rng, 1, 128)
        n = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
        ragged = rng.random() < 0.5
        if op == "append":
            c = _append("", type, nseq, n, rng.randrange(0, 1200), heads, kv_heads, head_dim, head_dim * rng.choice([1, 2, 3, 4, 4, 4]) // 4, rng.random() < 0.6, ragged,
                        rng.choice([0, _log(rng, 1, 8192)]))
            fits = nseq * (c["past"] + n) * kv_heads * head_dim <= 2 ** 24 and nseq * n * heads * head_dim <= 2 ** 24
        elif op == "prefix":
            c = _prefix("", rng.choice([F16, Q4]), type, nseq, n, _log(rng, 16, 32768), 0 if rng.random() < 0.3 else _log(rng, 1, 2000), heads, kv_heads, head_dim, ragged)
            upto = c["past"] + n
            fits = nseq * n * (c["shared"] + upto) * heads <= 2 ** 28 and nseq * upto * kv_heads * head_dim <= 2 ** 27 and work(c)["flops"] < 5e10
        elif op == "copy":
            source = _log(rng, 1, 16384)
            c = _copy("", rng.choice([F16, Q4]), nseq + 1, max(1, min(source, _log(rng, 1, 16384))), source, kv_heads, head_dim, rng.random() < 0.5)
            fits = nseq * source * kv_heads * head_dim <= 2 ** 25
        else:
            vocab = _log(rng, 1000, 160000)
            c = _logprobs("", type, _log(rng, 1, 1000), vocab, rng.choice([0, 1, 5, 8, 20, 64]), rng.choice([0, 0, 1, 300]))
            fits = c["rows"] * vocab <= 2 ** 26
        del c["name"]
        if fits:
            return c


def _places(case):
    """each sequence's first position and its number of new tokens"""
    S, n, past = case["nseq"], case["n"], case["past"]
    if not case["ragged"]:
        return [past] * S, [n] * S
    return [past - past * b * 5 // (8 * S) for b in range(S)], [max(1, n - n * b // (2 * S)) for b in range(S)]


def _cache(g, kind, S, ctx, G, D):
    """a cache's contents: keys have a few channels that are larger throughout, as rotated keys do; 4-bit: normal values' codes, and scales near those of their groups"""
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float16)  # noqa: E731
    if kind == F16:
        loud = 1 + 3 * (torch.rand(G, D, generator=g, device="cuda") < 0.06).half()
        return randn(S, ctx, G, D) * loud, randn(S, ctx, G, D)
    nb = (ctx + 7) // 8
    code = randn(S, G, nb, 16 * D).mul_(3).round_().clamp_(-7, 7).add_(8).to(torch.uint8)
    scale = (0.25 + 0.2 * torch.rand(S, G, nb, D // 2, generator=g, device="cuda")).bfloat16().half()
    return torch.cat([code[..., 0::2] | code[..., 1::2] << 4, scale.view(torch.uint8)], -1)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _kept(case, seed):
    """positions in rising order, of each sequence its own: a few first ones, some of the middle, the last ones"""
    g = torch.Generator().manual_seed(seed)
    return torch.stack([torch.randperm(case["source"], generator=g)[:case["n"]].sort().values for _ in range(case["nseq"])])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["op"] == "logprobs":
        t, R, V = TYPES[case["type"]], case["rows"], case["vocab"]
        x = rand(R, V) * 2.2
        x[:, torch.randint(0, V, (40,), generator=g, device="cuda")] += 6 * torch.rand(R, 40, generator=g, device="cuda")   # (a model's favourites)
        if case["padded"]:
            x[:, V - case["padded"]:] = float("-inf")
        s["logits"] = x.to(t)
        s["tokens"] = torch.stack([(row - torch.empty_like(row).exponential_(generator=g).log_()).argmax() for row in x]).int()
        return s
    G, D = case["kv_heads"], case["head_dim"]
    S = case["nseq"]
    if case["op"] == "copy":
        n, src = case["n"], case["source"]
        s["data"] = _cache(g, case["kind"], S, src if case["fork"] else n, G, D)
        s["source"] = None if case["fork"] else _cache(g, case["kind"], S, src, G, D)
        s["index"] = (torch.arange(n).repeat(S, 1) if case["fork"] else _kept(case, seed)).int().cuda()
        s["pos"] = _ints([-1] + [0] * (S - 1) if case["fork"] else [0] * S)   # (the first sequence of a fork is where the others come from)
        s["seqs"] = _ints([0] * S) if case["fork"] else None
        s["out"] = tuple(torch.zeros(S, n, G, D, dtype=torch.float16, device="cuda") for _ in range(2))
        return s
    t, n, H = TYPES[case["type"]], case["n"], case["heads"]
    pos, lens = _places(case)
    s["pos"], s["lens"], s["upto"] = _ints(pos), _ints(lens) if case["ragged"] else None, max(p + m for p, m in zip(pos, lens))
    if case["op"] == "append":
        # the rows as one projection leaves them, and tables as a program keeps them
        qkv = (rand(S, n, H + 2 * G, D) * (1 + 3 * (torch.rand(H + 2 * G, D, generator=g, device="cuda") < 0.06).float())).to(t)
        s["q"], s["k"], s["v"] = qkv[:, :, :H], qkv[:, :, H:H + G], qkv[:, :, H + G:]
        R = case["rot"]
        angle = torch.arange(case["behind"] + s["upto"], dtype=torch.float64, device="cuda").unsqueeze(1) * 10000.0 ** (torch.arange(R // 2, dtype=torch.float64, device="cuda") * -2 / R)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["at"] = _ints([p + case["behind"] for p in pos]) if case["behind"] else None
        s["weights"] = (1 + 0.2 * rand(D), 1 + 0.2 * rand(D)) if case["norm"] else (None, None)
        s["data"] = tuple(torch.zeros(S, s["upto"], G, D, dtype=torch.float16, device="cuda") for _ in range(2))
        s["out"] = torch.zeros(S, n, H, D, dtype=t, device="cuda")
        return s
    s["q"] = rand(S, n, H, D).to(t)
    s["out"] = torch.zeros(S, n, H, D, dtype=t, device="cuda")
    s["data"], s["prefix"] = _cache(g, case["kind"], S, s["upto"], G, D), _cache(g, case["kind"], 1, case["shared"] + 5, G, D)
    s["shared"] = _ints([case["shared"]])
    return s


def _shifts(device):
    e = torch.arange(8, device=device)
    return (16 * (e % 2) + 4 * (e // 2)).int()


def _values(data, ctx, kind):
    """a cache's values: K and V as fp32 [sequence][kv head][position][dim]"""
    if kind == F16:
        return tuple(x[:, :ctx].float().transpose(1, 2) for x in data)
    S, G, nb, D = data.shape[0], data.shape[1], (ctx + 7) // 8, data.shape[3] // 9
    r, sh = data[:, :, :nb], _shifts(data.device)
    kw = r[..., :4 * D].view(torch.int32).reshape(S, G, nb, 8, D // 8, 1)
    k = (((kw >> sh) & 15) - 8).view(S, G, nb, 8, D // 32, 32) * r[..., 8 * D:8 * D + D // 2].view(torch.float16).float().view(S, G, nb, 8, D // 32, 1)
    vw = r[..., 4 * D:8 * D].view(torch.int32).reshape(S, G, nb, 16, D // 16).transpose(3, 4).reshape(S, G, nb, 1, D)
    v = (((vw >> sh.view(8, 1)) & 15) - 8).view(S, G, nb, 8, D // 32, 32)
    v = v * r[..., 8 * D + D // 2:].view(torch.float16).float().view(S, G, nb, D // 32, 8).transpose(3, 4).unsqueeze(-1)
    return k.reshape(S, G, 8 * nb, D)[:, :, :ctx], v.reshape(S, G, 8 * nb, D)[:, :, :ctx]


def _live(s):
    """[sequence][token]: whether the sequence has this token"""
    t = torch.arange(s["case"]["n"], device="cuda")
    return (t < s["lens"].unsqueeze(1)) if s["lens"] is not None else torch.ones(s["case"]["nseq"], s["case"]["n"], dtype=torch.bool, device="cuda")


def _plain_append(s):
    c = s["case"]
    t = torch.arange(c["n"], device="cuda")
    p = s["pos"].unsqueeze(1) + t
    P = ((s["at"] if s["at"] is not None else s["pos"]).unsqueeze(1) + t).clamp(max=s["cos"].shape[0] - 1)
    cos, sin, h = s["cos"][P].unsqueeze(2), s["sin"][P].unsqueeze(2), c["rot"] // 2

    def rotated(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        a, b = x[..., :h], x[..., h:2 * h]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)

    live = _live(s)
    q = torch.where(live[:, :, None, None], rotated(s["q"], s["weights"][0]), 0).to(s["q"].dtype)
    b, i = live.nonzero(as_tuple=True)
    k, v = s["data"]
    k[b, p[b, i]] = rotated(s["k"], s["weights"][1])[b, i].half()
    v[b, p[b, i]] = s["v"][b, i].half()
    return q, k, v


def _plain_prefix(s):
    c = s["case"]
    S, n, H, G, D, T, L = c["nseq"], c["n"], c["heads"], c["kv_heads"], c["head_dim"], s["upto"], c["shared"]
    k0, v0 = (x[0] for x in _values(s["prefix"], L, c["kind"]))
    k, v = _values(s["data"], T, c["kind"])
    q = s["q"].float().view(S, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(S, G, H // G * n, D) / D ** 0.5
    x0 = torch.matmul(q.transpose(0, 1).reshape(G, -1, D), k0.transpose(1, 2).contiguous()).view(G, S, -1, L).transpose(0, 1)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(S, G, H // G, n, T)
    P = s["pos"].view(S, 1, 1, 1, 1) + torch.arange(n, device="cuda").view(n, 1)
    x = x.masked_fill_(torch.arange(T, device="cuda") > P, float("-inf")).view(S, G, -1, T)
    m = torch.maximum(x0.amax(-1, keepdim=True), x.amax(-1, keepdim=True))
    e0, e = (x0 - m).exp_(), (x - m).exp_()
    o = torch.matmul(e0.transpose(0, 1).reshape(G, -1, L), v0.contiguous()).view(G, S, -1, D).transpose(0, 1) + torch.matmul(e, v.contiguous())
    o = (o / (e0.sum(-1, keepdim=True) + e.sum(-1, keepdim=True))).view(S, G, H // G, n, D).permute(0, 3, 1, 2, 4).reshape(S, n, H, D)
    return torch.where(_live(s)[:, :, None, None], o, 0).to(s["q"].dtype)


def _plain_copy(s):
    c = s["case"]
    S, n = c["nseq"], c["n"]
    index = s["index"].long()
    rows = torch.arange(S, device="cuda").unsqueeze(1) if s["seqs"] is None else s["seqs"].long().unsqueeze(1)
    source = s["data"] if s["source"] is None else s["source"]
    first = 1 if c["fork"] else 0   # sequences before it take no part
    if c["kind"] == F16:
        new = [x[rows[first:], index[first:]] for x in source]
        for x, y in zip(s["data"], new):
            x[first:, :n] = y
        return s["data"]
    out = [x.transpose(1, 2)[rows, index].half() for x in _values(source, c["source"], Q4)]
    for x in out:
        x[:first] = 0
    return tuple(out)


def _plain_logprobs(s):
    c = s["case"]
    V, K = c["vocab"], c["top"]
    x, token = s["logits"].float(), s["tokens"].long().unsqueeze(1)
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp_()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    entropy = (log_total - torch.where(e > 0, e * (x - m), 0).sum(-1, keepdim=True) / total).squeeze(1)
    chosen, index = x.gather(1, token), torch.arange(V, device="cuda")
    rank = ((x > chosen) | ((x == chosen) & (index < token))).sum(-1).int()
    out = {"logp": (chosen - m - log_total).squeeze(1), "entropy": entropy, "rank": rank}
    if K:
        # the order of the values, then of the indices, as whole numbers
        bits = (x + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * 2 ** 32 + (2 ** 31 - index)
        at = key.topk(K, -1).indices
        out["top_index"], out["top_logp"] = at.int(), x.gather(1, at) - m - log_total
    return out


def run(state):
    c = state["case"]
    if not own:
        return {"append": _plain_append, "prefix": _plain_prefix, "copy": _plain_copy, "logprobs": _plain_logprobs}[c["op"]](state)
    import qpack_amd
    if c["op"] == "logprobs":
        r = qpack_amd.logprobs(state["logits"], state["tokens"], top=c["top"])
        out = {"logp": r.logp, "entropy": r.entropy, "rank": r.rank}
        return {**out, "top_index": r.top_index, "top_logp": r.top_logp} if c["top"] else out
    if "cache" not in state:   # the handles that a program keeps beside the caches' memory
        kind, G, D = c.get("kind", F16), c["kv_heads"], c["head_dim"]
        handle = lambda data: qpack_amd.KvCache(kind, (data[0] if kind == F16 else data).shape[0], G, D, ctx(data), data=data)  # noqa: E731
        ctx = lambda data: data[0].shape[1] if kind == F16 else 8 * data.shape[2]  # noqa: E731
        state["cache"], other = handle(state["data"]), state.get("source") if c["op"] == "copy" else state.get("prefix")
        state["other"] = handle(other) if other is not None else None
    cache = state["cache"]
    if c["op"] == "append":
        q = cache.append(state["q"], state["k"], state["v"], state["pos"], state["cos"], state["sin"], q_weight=state["weights"][0], k_weight=state["weights"][1], eps=1e-6,
                         at=state["at"], lens=state["lens"], out=state["out"])
        return q, *state["data"]
    if c["op"] == "prefix":
        return cache.attention(state["q"], state["pos"], lens=state["lens"], prefix=state["other"], prefix_len=state["shared"], out=state["out"])
    cache.copy(state["index"], state["pos"], seqs=state["seqs"], source=state["other"], apart=True)
    return state["data"] if c["kind"] == F16 else cache.read(state["pos"], c["n"], out=state["out"])


def work(case):
    if case["op"] == "logprobs":
        R, V, K = case["rows"], case["vocab"], case["top"]
        return {"bytes": R * (V * TYPES[case["type"]].itemsize + 16 + 8 * K), "flops": 8 * R * V}
    G, D = case["kv_heads"], case["head_dim"]
    held = 2 * G * D * (2 if case.get("kind", F16) == F16 else 9 / 16)   # bytes of a position in the cache
    if case["op"] == "copy":
        tokens = (case["nseq"] - 1 if case["fork"] else case["nseq"]) * case["n"]
        back = 0 if case["kind"] == F16 else held + 2 * G * D * 2        # (and read back)
        read = held * (case["n"] if case["fork"] else tokens)
        return {"bytes": tokens * (held + 4 + back) + read, "flops": tokens * 2 * G * D}
    pos, lens = _places(case)
    size, H, tokens = TYPES[case["type"]].itemsize, case["heads"], sum(lens)
    if case["op"] == "append":
        return {"bytes": tokens * (2 * (H + G) * D * size + held) + 4 * case["rot"] * (max(lens) if not case["ragged"] else tokens), "flops": tokens * (H + G) * D * 8}
    seen = sum(m * p + m * (m + 1) // 2 for p, m in zip(pos, lens))
    return {"bytes": 2 * tokens * H * D * size + (case["shared"] + sum(p + m for p, m in zip(pos, lens))) * held, "flops": 4 * D * H * (tokens * case["shared"] + seen)}


def _exact_records(r, T):
    """the values of one kv head's records r [record][byte], positions below T: K and V in 64 bits"""
    nb, D = r.shape[0], r.shape[1] // 9
    bits = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device="cuda")
    nib = ((r[:, :8 * D].contiguous().view(torch.int32).view(nb, 2 * D, 1) >> bits) & 15).double() - 8
    sc = r[:, 8 * D:].contiguous().view(torch.float16).double()
    k = (nib[:, :D].reshape(nb, 8, D // 32, 32) * sc[:, :D // 4].reshape(nb, 8, D // 32, 1)).reshape(8 * nb, D)[:T]
    vd = nib[:, D:].view(nb, 16, D // 16, 8).permute(0, 3, 2, 1).reshape(nb, 8, D)
    return k, (vd.view(nb, 8, D // 32, 32) * sc[:, D // 4:].view(nb, D // 32, 8).transpose(1, 2).unsqueeze(-1)).reshape(8 * nb, D)[:T]


def _exact_head(data, kind, b, h, T):
    return (data[0][b, :T, h].double(), data[1][b, :T, h].double()) if kind == F16 else _exact_records(data[b, h], T)


def exact(case, seed):
    s = prepare(case, seed)
    f64 = lambda *n: torch.zeros(*n, dtype=torch.float64, device="cuda")  # noqa: E731
    if case["op"] == "logprobs":
        R, K = case["rows"], case["top"]
        logp, entropy, best = f64(R), f64(R), f64(R, K)
        for r in range(R):
            y = torch.log_softmax(s["logits"][r].double(), 0)
            logp[r] = y[s["tokens"][r]]
            entropy[r] = -torch.special.xlogy(y.exp(), y.exp()).sum()
            best[r] = y.sort(descending=True).values[:K]
        out = {"logp": logp, "entropy": entropy, "rank": None}
        return {**out, "top_index": None, "top_logp": best} if K else out
    G, D, S, n = case["kv_heads"], case["head_dim"], case["nseq"], case["n"]
    if case["op"] == "copy":
        source = s["data"] if s["source"] is None else s["source"]
        if case["kind"] == F16:
            out = tuple(x.double() for x in s["data"])
        else:
            out = f64(S, n, G, D), f64(S, n, G, D)
        for b in range(1 if case["fork"] else 0, S):
            at = s["index"][b].long()
            for h in range(G):
                k, v = _exact_head(source, case["kind"], 0 if case["fork"] else b, h, case["source"])
                out[0][b, :n, h], out[1][b, :n, h] = k[at], v[at]
        return out
    pos, lens = _places(case)
    H = case["heads"]
    if case["op"] == "append":
        q, k, v = f64(S, n, H, D), f64(S, s["upto"], G, D), f64(S, s["upto"], G, D)
        R = case["rot"]
        for b, (p, m) in enumerate(zip(pos, lens)):
            a = p + case["behind"]
            # a pair of dims as a complex number, turned by its angle
            turn = torch.complex(s["cos"][a:a + m].double(), s["sin"][a:a + m].double()).unsqueeze(1)
            for x, w, out in ((s["q"], s["weights"][0], q[b, :m]), (s["k"], s["weights"][1], k[b, p:p + m])):
                y = x[b, :m].double()
                if w is not None:
                    y = y / ((y * y).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
                z = torch.complex(y[..., :R // 2].contiguous(), y[..., R // 2:R].contiguous()) * turn
                out.copy_(torch.cat([z.real, z.imag, y[..., R:]], -1))
            v[b, p:p + m] = s["v"][b, :m].double()
        return q, k, v
    out, L = f64(S, n, H, D), case["shared"]
    for h in range(G):
        k0, v0 = _exact_head(s["prefix"], case["kind"], 0, h, L)
        for b, (p, m) in enumerate(zip(pos, lens)):
            k, v = _exact_head(s["data"], case["kind"], b, h, p + m)
            k, v = torch.cat([k0, k]), torch.cat([v0, v])
            for t0 in range(0, m, 512):
                t1 = min(m, t0 + 512)
                q = s["q"][b, t0:t1, h * (H // G):(h + 1) * (H // G)].double()
                x = (q.reshape(-1, D) @ k.T.contiguous() / D ** 0.5).view(t1 - t0, H // G, L + p + m)
                hidden = torch.arange(-L, p + m, device="cuda") > p + torch.arange(t0, t1, device="cuda").view(-1, 1, 1)
                w = torch.softmax(x.masked_fill(hidden, -torch.inf), -1)
                out[b, t0:t1, h * (H // G):(h + 1) * (H // G)] = (w.reshape(-1, L + p + m) @ v).view(t1 - t0, H // G, D)
    return out
