"""The operators on packed tokens together, as a server calls them: a small model with rotary positions, root-mean-square norms and grouped
heads, whose requests come and go, bring their prompts in pieces and decode among each other, gives every request the logits that the
whole context at once gives in 64 bits; the same captured in a graph whose sequences change from replay to replay."""

import math

import pytest
import torch

from lighthouse_amd import ops

pytestmark = pytest.mark.gpu

bf16, f32, e4m3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
C, H, HKV, D, LAYERS, HIDDEN, VOCAB, SIZE, TURNED = 128, 4, 2, 32, 2, 256, 96, 8, 24


class Model:
    def __init__(self, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)
        w = lambda *shape: (0.15 * torch.randn(shape, generator=g)).to(dtype).cuda()  # noqa: E731
        norm = lambda: (1 + 0.2 * torch.randn(C, generator=g)).cuda()  # noqa: E731
        self.dtype, self.emb = dtype, torch.randn(VOCAB, C, generator=g).cuda()
        self.layers = [{"n1": norm(), "qkv": w(C, (H + 2 * HKV) * D), "o": w(H * D, C), "n2": norm(), "up": w(C, HIDDEN), "down": w(HIDDEN, C)} for _ in range(LAYERS)]
        self.last, self.head = norm(), w(C, VOCAB)
        self.freqs = ops.rotary_frequencies(TURNED, base=1000.0)

    def whole(self, tokens):
        """Logits of one request, every position, in 64 bits."""
        x = self.emb[tokens].double()
        n = len(tokens)
        norm = lambda x, g: x / ((x * x).mean(-1, keepdim=True) + 1e-5).sqrt() * g.double()  # noqa: E731
        angle = torch.arange(n, device="cuda").double()[:, None, None] * self.freqs

        def turn(x):
            a, b = x[..., : TURNED // 2], x[..., TURNED // 2:TURNED]
            return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., TURNED:]], -1)

        for p in self.layers:
            q, k, v = (norm(x, p["n1"]) @ p["qkv"].double()).view(n, -1, D).split([H, HKV, HKV], 1)
            q, k = turn(q), turn(k)
            k, v = (t.repeat_interleave(H // HKV, 1) for t in (k, v))
            s = torch.stack([q[:, h] @ k[:, h].t().contiguous() for h in range(H)]) / math.sqrt(D)
            s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf).softmax(-1)
            o = torch.stack([s[h] @ v[:, h] for h in range(H)], 1)
            x = x + o.reshape(n, -1) @ p["o"].double()
            x = x + torch.nn.functional.gelu(norm(x, p["n2"]) @ p["up"].double(), approximate="tanh") @ p["down"].double()
        return norm(x, self.last) @ self.head.double()


class Server:
    def __init__(self, m, B, pages, P, cache_dtype=None):
        self.m, self.scale = m, 0.05 if cache_dtype == e4m3 else 1.0
        self.table = torch.full((B, P), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        self.n_free = torch.full((1,), pages, dtype=torch.int32, device="cuda")
        make = lambda: torch.full((pages, HKV, SIZE, D), math.nan).to(cache_dtype or m.dtype).cuda()  # noqa: E731
        self.caches = [(make(), make()) for _ in range(LAYERS)]

    def step(self, tokens, counts):
        """Logits of the packed tokens' rows."""
        m, N = self.m, len(tokens)
        _, starts, positions, slots = ops.kv_pages(self.table, self.lengths, counts, self.free, self.n_free, SIZE, N, out=self.lengths)
        scales = {"k_scale": self.scale, "v_scale": self.scale}
        x = m.emb[tokens]  # the residual, in f32
        y = torch.zeros(N, C, dtype=m.dtype, device="cuda")
        for p, cache in zip(m.layers, self.caches):
            h = ops.rms_norm(y, p["n1"], residual=x, out_dtype=m.dtype)
            qkv = ops.gemm(h, p["qkv"]).view(N, H + 2 * HKV, D)
            q, _, _ = ops.kv_store(qkv[:, H:H + HKV], qkv[:, H + HKV:], *cache, slots, q=qkv[:, :H], q_out=qkv[:, :H], positions=positions, freqs=m.freqs, **scales)
            o = ops.paged_attention_chunk(q, *cache, self.table, self.lengths, starts, out=torch.zeros(N, H, D, dtype=m.dtype, device="cuda"), **scales)
            h = ops.rms_norm(ops.gemm(o.view(N, H * D), p["o"]), p["n2"], residual=x, out_dtype=m.dtype)
            y = ops.gemm(ops.gemm(h, p["up"], gelu=True), p["down"])
        return ops.gemm(ops.rms_norm(y, m.last, residual=x, out_dtype=m.dtype), m.head, out_dtype=f32)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# Which piece of its request a place gets in each step: (request, from, to), None: nothing, "end": it leaves.
STEPS = [
    [(0, 0, 21), (1, 0, 5), None, None],
    [(0, 21, 40), (1, 5, 6), (2, 0, 33), None],
    [(0, 40, 41), (1, 6, 7), None, (3, 0, 1)],
    ["end", (1, 7, 8), (2, 33, 34), (3, 1, 2)],
    [(4, 0, 18), (1, 8, 9), (2, 34, 35), "end"],
    [(4, 18, 19), "end", (2, 35, 70), (5, 0, 70)],
    [(4, 19, 20), (6, 0, 2), (2, 70, 71), (5, 70, 71)],
]
LENGTHS = [41, 9, 71, 2, 20, 71, 2]


def pack(prompts, step, room):
    counts = [0 if p is None else -1 if p == "end" else p[2] - p[1] for p in step]
    tokens = [prompts[p[0]][p[1]:p[2]] for p in step if isinstance(p, tuple)]
    tokens = torch.cat([*tokens, torch.zeros(room - sum(max(c, 0) for c in counts), dtype=torch.int64)])
    return tokens.cuda(), i32(*counts)


# What a row of logits may be off, of the largest: the weights' and activations' roundings on the way through two layers
# (f32: sums of at most 256 products over a dozen products, 2^-24 each; bf16: 2^-8 for each of a dozen roundings, which add up like their root;
# a cache of 8 bits: 2^-4 of keys and values, twice).
OFF = {(f32, None): 1e-4, (bf16, None): 12 * 2.0**-8, (bf16, e4m3): 0.25}


@pytest.mark.parametrize("dtype,cache", [(f32, None), (bf16, None), (bf16, e4m3)])
def test_requests_that_come_and_go(dtype, cache):
    m = Model(dtype)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in LENGTHS]
    want = [m.whole(p.cuda()) for p in prompts]
    server = Server(m, 4, 34, 10, cache)
    for step in STEPS:
        tokens, counts = pack(prompts, step, 110)
        logits = server.step(tokens, counts)
        at = 0
        for p in step:
            if isinstance(p, tuple):
                exact = want[p[0]][p[1]:p[2]]
                off = (logits[at:at + p[2] - p[1]].double() - exact).abs().max() / exact.abs().max()
                assert off <= OFF[dtype, cache], (p, float(off))
                at += p[2] - p[1]
        held = (server.table >= 0).sum().item()
        assert held + server.n_free.item() == 34 and held == sum(-(-n // SIZE) for n in server.lengths.tolist())


def test_single_tokens_through_either_attention():
    """A step of one token each: paged_attention and paged_attention_chunk read the same cache."""
    m = Model(f32, seed=3)
    server = Server(m, 3, 40, 8)
    g = torch.Generator().manual_seed(4)
    counts = [30, 7, 12]
    server.step(torch.randint(0, VOCAB, (49,), generator=g).cuda(), i32(*counts))
    q = torch.randn(3, H, D, generator=g).cuda()
    one = ops.paged_attention(q, *server.caches[0], server.table, server.lengths)
    other = ops.paged_attention_chunk(q, *server.caches[0], server.table, server.lengths, i32(0, 1, 2, 3))
    assert (one - other).abs().max() <= 1e-5 * one.abs().max()


def test_a_server_out_of_pages_goes_on():
    """A request that gets no pages has rows that mean nothing; the others' are what they would be, and it gets its pages once another has ended."""
    m = Model(f32, seed=5)
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (24, 30, 10)]
    want = [m.whole(p.cuda()) for p in prompts]
    server = Server(m, 3, 5, 8)  # 40 slots
    tokens, counts = pack(prompts, [(0, 0, 24), (1, 0, 30), None], 60)
    logits = server.step(tokens, counts)
    assert server.lengths.tolist() == [24, 0, 0] and server.n_free.item() == 2
    assert (logits[:24].double() - want[0]).abs().max() <= 1e-4 * want[0].abs().max()
    tokens, counts = pack(prompts, ["end", (1, 0, 30), (2, 0, 8)], 60)
    logits = server.step(tokens, counts)
    assert server.lengths.tolist() == [0, 30, 8] and server.n_free.item() == 0
    for b, rows in ((1, slice(0, 30)), (2, slice(30, 38))):
        exact = want[b][: rows.stop - rows.start]
        assert (logits[rows].double() - exact).abs().max() <= 1e-4 * exact.abs().max()


def test_captured_steps():
    """Two graphs of a step, of servers of their own, replayed in turn with eager work between, each time with other requests."""
    m = Model(bf16, seed=7)
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in LENGTHS]
    servers, eager, graphs = [], [], []
    for _ in range(2):
        s, e = Server(m, 4, 34, 10), Server(m, 4, 34, 10)
        s.tokens, s.counts = torch.zeros(110, dtype=torch.int64, device="cuda"), i32(0, 0, 0, 0)
        s.step(s.tokens, s.counts)  # (warm: no tokens)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.logits = s.step(s.tokens, s.counts)
        servers.append(s), eager.append(e), graphs.append(graph)
    for step in STEPS:
        tokens, counts = pack(prompts, step, 110)
        for s, e, graph in zip(servers, eager, graphs):
            s.tokens.copy_(tokens), s.counts.copy_(counts)
            graph.replay()
            want = e.step(tokens, counts)
            torch.cuda.synchronize()
            n = int(counts.clamp(min=0).sum())
            assert torch.equal(s.logits[:n], want[:n]) and torch.equal(s.table, e.table) and torch.equal(s.lengths, e.lengths) and torch.equal(s.n_free, e.n_free)
