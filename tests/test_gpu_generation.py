"""The operators of a paged cache together, as a program that generates tokens calls them: a small GPT whose steps read the cache give
the logits that the forward over the whole context gives; a step captured in a graph; two streams; eviction between steps."""

import math

import pytest
import torch

from lighthouse_amd import ops
from tests import paged_reference as ref
from tests.conftest import assert_close

pytestmark = pytest.mark.gpu

bf16, f32 = torch.bfloat16, torch.float32
C, HEADS, LAYERS, VOCAB, D = 128, 2, 2, 300, 64


def model(dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def w(*shape):
        return (torch.randn(shape, device="cuda", generator=g) * 0.08).to(dtype)

    def norm():
        return 1.0 + 0.1 * torch.randn(C, device="cuda", generator=g), 0.05 * torch.randn(C, device="cuda", generator=g)

    layers = []
    for _ in range(LAYERS):
        p = {"w_qkv": w(C, 3 * C), "b_qkv": w(3 * C), "w_o": w(C, C), "b_o": w(C), "w_fc": w(C, 4 * C), "b_fc": w(4 * C), "w_proj": w(4 * C, C), "b_proj": w(C)}
        (p["ln1_g"], p["ln1_b"]), (p["ln2_g"], p["ln2_b"]) = norm(), norm()
        layers.append(p)
    return {"layers": layers, "lnf": norm(), "lm_w": w(C, VOCAB), "lm_b": w(VOCAB), "emb": torch.randn(VOCAB, C, device="cuda", generator=g),
            "pos": torch.randn(64, C, device="cuda", generator=g) * 0.3, "dtype": dtype}


class Generator:
    """Pages for B sequences of up to `room` tokens; a cache per layer."""

    def __init__(self, m, B, room=64, size=16, layout="heads"):
        self.m, self.B = m, B
        P = -(-room // size)
        pages = B * P + 2
        shape = (pages, HEADS, size, D) if layout == "heads" else (pages, size, HEADS, D)
        make = lambda: torch.full(shape, math.nan, dtype=m["dtype"], device="cuda") if layout == "heads" else torch.full(shape, math.nan, dtype=m["dtype"], device="cuda").transpose(1, 2)  # noqa: E731
        self.caches = [(make(), make()) for _ in range(LAYERS)]
        self.table = torch.randperm(pages, generator=torch.Generator().manual_seed(3))[: B * P].to(torch.int32).view(B, P).cuda()
        self.weights = torch.zeros(LAYERS, B, HEADS, P * size, device="cuda")

    def residual(self, x, y, w, b):
        return ops.gemm(y, w, b.float(), residual=x, out_dtype=f32) if w.dtype != f32 else ops.gemm(y, w, b, residual=x)

    def layer(self, i, x, attend):
        p, dt = self.m["layers"][i], self.m["dtype"]
        h = ops.layer_norm(x, p["ln1_g"], p["ln1_b"], out_dtype=dt)
        qkv = ops.gemm(h, p["w_qkv"], p["b_qkv"])
        x = self.residual(x, attend(i, qkv), p["w_o"], p["b_o"])
        h = ops.layer_norm(x, p["ln2_g"], p["ln2_b"], out_dtype=dt)
        return self.residual(x, ops.gemm(h, p["w_fc"], p["b_fc"], gelu=True), p["w_proj"], p["b_proj"])

    def logits(self, x):
        h = ops.layer_norm(x, *self.m["lnf"], out_dtype=self.m["dtype"])
        return ops.gemm(h, self.m["lm_w"], self.m["lm_b"].float(), out_dtype=f32) if self.m["dtype"] != f32 else ops.gemm(h, self.m["lm_w"], self.m["lm_b"])

    def step(self, tokens, positions, lengths, slots=None):
        """One token of every sequence; `slots`: where it goes in the cache, if not at its position."""
        slots = positions if slots is None else slots

        def attend(i, qkv):
            q, k, v = (qkv[:, j * C:(j + 1) * C].view(self.B, HEADS, D) for j in range(3))
            ops.kv_append(k.unsqueeze(2), v.unsqueeze(2), *self.caches[i], self.table, slots)
            return ops.paged_attention(q, *self.caches[i], self.table, lengths, weights=self.weights[i]).view(self.B, C)

        x = self.m["emb"][tokens] + self.m["pos"][positions.long()]
        for i in range(LAYERS):
            x = self.layer(i, x, attend)
        return self.logits(x)

    def prompt(self, tokens, counts):
        """Prompts padded to one length: keys and values into the cache, logits of every position."""
        T = tokens.shape[1]
        zero = torch.zeros(self.B, dtype=torch.int32, device="cuda")

        def attend(i, qkv):
            q, k, v = (qkv.view(self.B, T, 3, HEADS, D)[:, :, j].transpose(1, 2) for j in range(3))
            ops.kv_append(k, v, *self.caches[i], self.table, zero, counts=counts)
            return ops.attention(q, k, v, causal=True).transpose(1, 2).reshape(self.B * T, C)

        x = (self.m["emb"][tokens] + self.m["pos"][:T]).reshape(self.B * T, C)
        for i in range(LAYERS):
            x = self.layer(i, x, attend)
        return self.logits(x).view(self.B, T, VOCAB)


def whole(m, tokens):
    x = (m["emb"][tokens] + m["pos"][: tokens.shape[1]]).contiguous()
    return ops.nanogpt_forward(x, m["layers"], *m["lnf"], m["lm_w"], m["lm_b"], HEADS)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,layout", [(f32, "heads"), (f32, "slots"), (bf16, "heads")])
def test_steps_over_the_cache_are_the_forward(dtype, layout):
    """Prompts of 5, 1 and 17 tokens, then steps of given tokens: logits as from the forward over the whole context."""
    m = model(dtype)
    lengths, steps = [5, 1, 17], 14
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, VOCAB, (3, max(lengths) + steps), device="cuda", generator=g)
    want = [whole(m, tokens[b:b + 1, : n + steps])[0].cpu().numpy() for b, n in enumerate(lengths)]
    gen = Generator(m, 3, layout=layout)
    rtol = 1e-4 if dtype == f32 else 2e-2
    got = gen.prompt(tokens[:, : max(lengths)], i32(*lengths))
    for b, n in enumerate(lengths):
        assert_close(got[b, :n].cpu().numpy(), want[b][:n], rtol, f"prompt {b}")
    for s in range(steps):
        at = i32(*[n + s for n in lengths])
        now = torch.stack([tokens[b, n + s] for b, n in enumerate(lengths)])
        got = gen.step(now, at, at + 1)
        for b, n in enumerate(lengths):
            assert_close(got[b].cpu().numpy(), want[b][n + s], rtol, f"sequence {b} step {s}")
    # what the steps attended to adds up to the number of steps
    for b, n in enumerate(lengths):
        total = gen.weights[:, b, :, : n + steps].sum(-1)
        assert (total - steps).abs().max() < 1e-3 and (gen.weights[:, b, :, n + steps:] == 0).all()


def test_generating_greedily_is_the_forward_s_choice():
    m = model(f32, seed=2)
    gen = Generator(m, 2)
    prompt = torch.randint(0, VOCAB, (2, 9), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    logits = gen.prompt(prompt, None)[:, -1]
    out = prompt
    for s in range(10):
        token = ops.sample(logits.contiguous(), torch.zeros(2, device="cuda"), temperature=0.0)
        assert torch.equal(token, logits.argmax(-1))
        out = torch.cat([out, token[:, None]], 1)
        at = i32(9 + s, 9 + s)
        logits = gen.step(token, at, at + 1)
    full = torch.cat([whole(m, out[b:b + 1]) for b in range(2)])
    top2 = full[:, 8:-1].topk(2, -1).values
    clear = top2[..., 0] - top2[..., 1] > 1e-3  # (the choice does not hang on a rounding)
    assert clear.float().mean() > 0.5 and (out[:, 9:] == full[:, 8:-1].argmax(-1))[clear].all()


def test_steps_go_on_over_an_evicted_cache():
    """30 tokens, cut to 12 a head; the next step attends to what stayed, in the order it stood, and to itself."""
    m = model(f32, seed=5)
    gen = Generator(m, 2)
    g = torch.Generator(device="cuda").manual_seed(6)
    tokens = torch.randint(0, VOCAB, (2, 31), device="cuda", generator=g)
    for t in range(30):
        at = i32(t, t)
        gen.step(tokens[:, t], at, at + 1)
    lengths = i32(30, 30)
    rows = lambda cache, b, h, n: cache[gen.table[b].long(), h].reshape(-1, D)[:n].cpu()  # noqa: E731
    for i in range(LAYERS):
        kept = [[ref.evict(gen.weights[i, b, h].cpu(), 30, 12, 4) for h in range(HEADS)] for b in range(2)]
        before = [[[rows(c, b, h, 30)[kept[b][h]] for h in range(HEADS)] for b in range(2)] for c in gen.caches[i]]
        new = ops.kv_evict(*gen.caches[i], gen.weights[i], gen.table, lengths, 12, recent=4)
        assert new.tolist() == [12, 12]
        for c, was in zip(gen.caches[i], before):
            for b in range(2):
                for h in range(HEADS):
                    assert torch.equal(rows(c, b, h, 12), was[b][h])
    q = torch.randn(2, HEADS, D, device="cuda", generator=g)
    out = ops.paged_attention(q, *gen.caches[0], gen.table, new).cpu().double()
    for b in range(2):
        k, v = (torch.stack([rows(c, b, h, 12) for h in range(HEADS)]) for c in gen.caches[0])
        want, _, allowed, _ = ref.attention(q[b].cpu(), k, v, D**-0.5)
        assert ((out[b] - want).abs() <= allowed).all()
    gen.step(tokens[:, 30], i32(30, 30), new + 1, slots=new)
    assert (gen.weights[:, :, :, 13:] == 0).all() and (gen.weights[:, :, :, 12] > 0).all()


def test_a_captured_step_replays_as_it_runs():
    """Two graphs of a step (append, attention with weights, sampling), replayed in turn with eager work between, each time on new inputs."""
    m = model(bf16, seed=7)

    def build(seed):
        gen = Generator(m, 2)
        s = {"gen": gen, "tokens": torch.zeros(2, dtype=torch.int64, device="cuda"), "at": i32(0, 0), "u": torch.zeros(2, device="cuda")}
        s["run"] = lambda: ops.sample(gen.step(s["tokens"], s["at"], s["at"] + 1), s["u"], temperature=0.9, top_k=40, top_p=0.95)
        return s

    graphs, eager = [build(1), build(2)], [build(1), build(2)]
    for s in graphs:
        s["run"]()  # (warm)
        for k, v in s["gen"].caches:
            k.fill_(math.nan), v.fill_(math.nan)
        s["gen"].weights.zero_()
        torch.cuda.synchronize()
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            s["out"] = s["run"]()
    g = torch.Generator(device="cuda").manual_seed(8)
    for t in range(20):
        for s, e in zip(graphs, eager):
            tokens, u = torch.randint(0, VOCAB, (2,), device="cuda", generator=g), torch.rand(2, device="cuda", generator=g)
            for x in (s, e):
                x["tokens"].copy_(tokens), x["u"].copy_(u), x["at"].fill_(t)
            s["graph"].replay()
            want = e["run"]()
            torch.cuda.synchronize()
            assert torch.equal(s["out"], want)
            assert torch.equal(s["gen"].weights, e["gen"].weights)


def test_captured_eviction_and_large_rows():
    """An eviction and sampling with a workspace, captured; the pages and logits change between replays."""
    c = ref.Cache([300, 120], 2, 16, 64, bf16, seed=9)
    other = ref.Cache([300, 120], 2, 16, 64, bf16, seed=9)
    g = torch.Generator(device="cuda").manual_seed(9)
    w, w2 = (torch.zeros(2, 2, c.capacity, device="cuda") for _ in range(2))
    x, u = torch.zeros(2, 20000, device="cuda"), torch.zeros(2, device="cuda")
    run = lambda cache, weights: (ops.kv_evict(cache.k_cache, cache.v_cache, weights, cache.table, cache.device_lengths, 100, recent=9), ops.sample(x, u, top_p=0.8))  # noqa: E731
    run(c, w.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(c, w)
    for _ in range(4):
        for cache, o in ((c.k_cache, other.k_cache), (c.v_cache, other.v_cache)):
            ref.as_bits(cache).copy_(ref.as_bits(o))
        w.copy_(torch.rand(w.shape, device="cuda", generator=g))
        w2.copy_(w)
        x.copy_(2 * torch.randn(x.shape, device="cuda", generator=g))
        u.copy_(torch.rand(2, device="cuda", generator=g))
        graph.replay()
        want = run(other, w2)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]) and torch.equal(w, w2)
        assert torch.equal(ref.as_bits(c.k_cache), ref.as_bits(other.k_cache)) and torch.equal(ref.as_bits(c.v_cache), ref.as_bits(other.v_cache))


def test_two_streams_at_once():
    caches = [ref.Cache([2500, 700], 2, 16, 64, bf16, seed=10 + i) for i in range(2)]
    g = torch.Generator(device="cuda").manual_seed(10)
    q = torch.randn(2, 8, 64, device="cuda", generator=g).to(bf16)
    x, u = torch.randn(4, 30000, device="cuda", generator=g), torch.rand(4, device="cuda", generator=g)

    def run(c):
        w = torch.zeros(2, 2, c.capacity, device="cuda")
        out = ops.paged_attention(q, c.k_cache, c.v_cache, c.table, c.device_lengths, weights=w)
        return out, w, ops.sample(x, u, top_p=0.7)

    want = [run(c) for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(run(caches[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for result in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[i]))
