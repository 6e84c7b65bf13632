"""A served batch, as a program runs it: a prompt appended to a cache of its own, samples behind it as a common prefix, steps of the batch (projections, append, attention behind the
prefix, projections, log probabilities, the next tokens), one sample forked over another; and the same with the prompt copied into every sequence's own cache.  One layer, in
64 bits beside it on the CPU."""
import pytest

import qpack_amd as qa

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv import i32  # noqa: E402


class Model:
    """one attention layer between an embedding and a head"""

    def __init__(self, V, H, G, D, gen):
        self.H, self.G, self.D = H, G, D
        r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)   # noqa: E731
        self.embed, self.qkv, self.head = r(V, 64), r(64, (H + 2 * G) * D) / 8, r(H * D, V) * 0.15
        self.wq, self.wk = (1 + 0.1 * r(D), 1 + 0.1 * r(D))
        a = torch.arange(400, dtype=torch.float64).unsqueeze(1) * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)
        self.cos, self.sin = a.cos(), a.sin()

    def logits(self, tokens):
        """of the whole text [n], causal, in 64 bits"""
        n, H, G, D = len(tokens), self.H, self.G, self.D
        q, k, v = (self.embed[tokens] @ self.qkv).view(n, H + 2 * G, D).split((H, G, G), 1)

        def turned(x, w):
            x = x / ((x * x).mean(-1, keepdim=True) + 1e-6).sqrt() * w
            a, b = x.chunk(2, -1)
            c, s = self.cos[:n].unsqueeze(1), self.sin[:n].unsqueeze(1)
            return torch.cat([a * c - b * s, b * c + a * s], -1)
        q, k = turned(q, self.wq), turned(k, self.wk)
        k, v = (x.repeat_interleave(H // G, 1).transpose(0, 1) for x in (k, v))
        x = torch.matmul(q.transpose(0, 1), k.transpose(1, 2).contiguous()) / D ** 0.5
        x = x.masked_fill(torch.ones(n, n).triu(1).bool(), -torch.inf)
        return torch.matmul(torch.softmax(x, -1), v.contiguous()).transpose(0, 1).reshape(n, H * D) @ self.head


# what 16-bit rows and caches move: q, k, v and the output rounded to 2^-11 of themselves (bf16 2^-8 is not used here), scores by 2^-9 or so of their size, under 12; logits of size 2 by some 2^-7.  A 4-bit cache
# rounds keys and values by a fourteenth of their groups' largest: its runs are held to one another and not to 64 bits
@pytest.mark.parametrize("kind", ["f16", "q4"])
@pytest.mark.parametrize("hd,H,G", [(64, 6, 2), (128, 4, 1)])
def test_batch(kind, hd, H, G):
    gen = torch.Generator().manual_seed(hd)
    V, S, P, steps = 301, 5, 131, 12
    m = Model(V, H, G, hd, gen)
    g = {k: v.half().cuda() for k, v in (("embed", m.embed), ("qkv", m.qkv), ("head", m.head))}
    cos, sin, wq, wk = (x.float().cuda() for x in (m.cos, m.sin, m.wq, m.wk))
    prompt = torch.randint(0, V, (P,), generator=gen)
    prefix, own, whole = qa.KvCache(kind, 1, G, hd, P + 3), qa.KvCache(kind, S, G, hd, steps + 2), qa.KvCache(kind, S, G, hd, P + steps)

    def rows(tokens):   # [sequences][n] -> q, k, v as one projection leaves them
        x = torch.matmul(g["embed"][tokens], g["qkv"]).view(*tokens.shape, H + 2 * G, hd)
        return x[:, :, :H], x[:, :, H:H + G], x[:, :, H + G:]

    def scored(out, next_tokens):
        return qa.logprobs(torch.matmul(out.reshape(-1, H * hd), g["head"]), next_tokens, top=4)
    q, k, v = rows(prompt[None].cuda())
    q = prefix.append(q, k, v, i32([0]), cos, sin, wq, wk)
    out = prefix.attention(q, i32([0]))
    got = scored(out, torch.cat([prompt[1:], torch.tensor([-1])]).int().cuda())
    want = torch.log_softmax(m.logits(prompt), -1)
    if kind == "f16":
        assert float((got.logp[:-1].cpu() - want[torch.arange(P - 1), prompt[1:]]).abs().max()) < 0.05
    # the samples' first tokens: the prompt's alternatives
    length = i32([P])
    whole.copy(torch.arange(P, dtype=torch.int32, device="cuda").unsqueeze(0).expand(S, P), i32([0] * S), seqs=i32([0] * S), source=prefix)
    token = torch.tensor([0, 1, 2, 3, 0])
    token = got.top_index[-1].cpu()[token].long()
    texts = [prompt.tolist() + [int(t)] for t in token]
    lens = [0] * S   # of the own caches
    for step in range(steps):
        q, k, v = rows(token[:, None].cuda())
        qo = own.append(q, k, v, i32(lens), cos, sin, wq, wk, at=i32([P + n for n in lens]))
        a = own.attention(qo, i32(lens), prefix=prefix, prefix_len=length)
        qw = whole.append(q, k, v, i32([P + n for n in lens]), cos, sin, wq, wk)
        b = whole.attention(qw, i32([P + n for n in lens]))
        assert torch.equal(qo, qw)
        assert float((a.float() - b.float()).abs().max()) < 2.0 ** -9 * float(b.float().abs().max())
        picks = torch.tensor([(step + i) % 3 for i in range(S)])   # one of the first three alternatives
        r = scored(a, None)
        token = r.top_index.cpu()[torch.arange(S), picks].long()
        again = scored(a, token.int().cuda())
        assert again.rank.tolist() == picks.tolist()
        assert torch.equal(again.logp, r.top_logp[torch.arange(S), picks.cuda()])
        if kind == "f16":
            for i in range(S):
                want = torch.log_softmax(m.logits(torch.tensor(texts[i]))[-1], -1)
                assert abs(float(again.logp[i]) - float(want[token[i]])) < 0.05
        lens = [n + 1 for n in lens]
        if step == 5:   # sample 4 goes on from sample 1's text, and sample 0 forgets its last two tokens but one
            seqs = [0, 1, 2, 3, 1]
            index = torch.arange(steps + 2, dtype=torch.int32).repeat(S, 1)
            own.copy(index[:, :6].contiguous().cuda(), i32([0] * S), seqs=i32(seqs))
            whole.copy(torch.arange(P + 6, dtype=torch.int32, device="cuda").unsqueeze(0).expand(S, -1), i32([-1, -1, -1, -1, 0]), seqs=i32(seqs), apart=True)
            texts[4], token[4] = list(texts[1]), token[1]
        for i in range(S):
            texts[i].append(int(token[i]))
