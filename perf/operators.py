"""Generating tokens over a paged key / value cache: what these operators compute, and calls of real sizes.

Four operators of `lighthouse_amd.ops`: `kv_append` writes the keys and values of new tokens into pages, `paged_attention`
reads them for one new token of every sequence (and adds up how much attention each position got), `kv_evict` drops the
positions that got least, `sample` draws the next token from logits and given random numbers.

A cache is [pages, kv heads, page size, d]; position t of sequence b lies in page `table[b, t // size]`, slot `t % size`.
`listed()` names calls that stand for the rest, `draw()` gives others of the same ranges, `prepare` makes what a program holds
before a call, `run` is one call (`own`: the library's kernels, otherwise elementary torch operations in 32 or 64 bits),
`exact` the same from the definitions in 64 bits, `work` the bytes and operations that a call cannot do without.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
E4M3_MAX = 448.0
LARGEST_CACHE = 2 * 16 * 32768 * 8 * 128 * 2  # bytes of keys and values behind the largest attention
LARGEST_EVICT = 2 * 4 * 16384 * 8 * 128 * 2
LARGEST_APPEND = 8 * 1024 * 12 * 64           # values of k
LARGEST_LOGITS = 128 * 131072


def _append(name, dtype, cache, B, Hkv, T, d, page, ragged):
    return {"name": name, "kind": "append", "dtype": dtype, "cache": cache, "B": B, "Hkv": Hkv, "T": T, "d": d, "page": page,
            "ragged": ragged}


def _attention(name, dtype, cache, B, Hkv, G, d, length, page, ragged, weights=False):
    return {"name": name, "kind": "attention", "dtype": dtype, "cache": cache, "B": B, "Hkv": Hkv, "G": G, "d": d,
            "length": length, "page": page, "ragged": ragged, "weights": weights}


def _evict(name, cache, B, Hkv, d, length, page, ragged, budget, recent):
    return {"name": name, "kind": "evict", "cache": cache, "B": B, "Hkv": Hkv, "d": d, "length": length, "page": page,
            "ragged": ragged, "budget": budget, "recent": recent}


def _sample(name, dtype, B, V, top_k, top_p, min_p, temperature, per_row):
    return {"name": name, "kind": "sample", "dtype": dtype, "B": B, "V": V, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "temperature": temperature, "per_row": per_row}


def listed():
    return [
        # One decoding step of a batch: the keys and values of one token of each of 64 sequences.
        _append("append_bf16_step", "bf16", "bf16", 64, 12, 1, 64, 16, False),
        # Eight prompts of different lengths, padded to one, into a cache of 8 bits.
        _append("append_e4m3_prompts", "bf16", "e4m3", 8, 12, 1024, 64, 16, True),
        # A single user: one sequence of a short conversation, where latency is all.
        _attention("attention_bf16_single", "bf16", "bf16", 1, 12, 1, 64, 1000, 16, False),
        # A batch of the GPT that this repository's benchmark runs (12 heads of 64, context 1024).
        _attention("attention_bf16_batch", "bf16", "bf16", 64, 12, 1, 64, 1024, 16, True),
        # Long documents with grouped heads: the largest cache.
        _attention("attention_bf16_long", "bf16", "bf16", 16, 8, 4, 128, 32768, 64, True),
        # The same kind of batch from a cache of 8 bits, wide groups.
        _attention("attention_e4m3_grouped", "bf16", "e4m3", 32, 4, 8, 128, 8192, 32, True),
        # Sizes nobody tuned for, in 32 bits: head dimension 80, pages of 24, odd lengths.
        _attention("attention_f32_odd", "f32", "f32", 3, 5, 1, 80, 2999, 24, True),
        # A step whose attention weights are kept for eviction.
        _attention("attention_f16_weights", "f16", "f16", 8, 4, 4, 96, 4096, 16, True, weights=True),
        # A batch at the end of its context, cut back to half.
        _evict("evict_bf16_batch", "bf16", 16, 12, 64, 1024, 16, False, 512, 128),
        # Long documents kept to a quarter.
        _evict("evict_f16_long", "f16", 4, 8, 128, 16384, 64, True, 4096, 512),
        # The next token of one sequence over this repository's vocabulary, with the usual filters.
        _sample("sample_f32_single", "f32", 1, 50257, 50, 0.95, 0.0, 0.8, False),
        # The next tokens of a batch over a large vocabulary, each row with settings of its own.
        _sample("sample_bf16_batch", "bf16", 128, 131072, 0, 0.9, 0.02, 1.0, True),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "evict", "sample", "sample"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    d = rng.choice([32, 64, 64, 80, 96, 128, 128, 256, rng.randint(1, 256)])
    cache = rng.choice(["bf16", "bf16", "f16", "f32", "e4m3"])
    dtype = rng.choice(["bf16", "f16"]) if cache == "e4m3" else cache
    ragged = rng.random() < 0.7
    if kind == "append":
        while True:
            B, Hkv, T = _log_uniform(rng, 1, 128), rng.randint(1, 16), rng.choice([1, 1, _log_uniform(rng, 2, 2048)])
            if B * Hkv * T * d <= LARGEST_APPEND:
                break
        case = _append("", dtype, cache, B, Hkv, T, d, page, ragged)
    elif kind == "attention":
        while True:
            B, Hkv, length = _log_uniform(rng, 1, 128), rng.randint(1, 16), _log_uniform(rng, 1, 32768)
            if 2 * B * Hkv * length * d * BYTES[cache] <= LARGEST_CACHE:
                break
        case = _attention("", dtype, cache, B, Hkv, rng.choice([1, 1, 2, 3, 4, 5, 8, 16]), d, length, page, ragged, rng.random() < 0.3)
    elif kind == "evict":
        while True:
            B, Hkv, length = _log_uniform(rng, 1, 32), rng.randint(1, 16), _log_uniform(rng, 16, 16384)
            if 2 * B * Hkv * length * d * BYTES[cache] <= LARGEST_EVICT:
                break
        budget = rng.randint(1, length)
        case = _evict("", cache, B, Hkv, d, length, page, ragged, budget, rng.randint(0, budget))
    else:
        while True:
            B, V = _log_uniform(rng, 1, 512), _log_uniform(rng, 2, 131072)
            if B * V <= LARGEST_LOGITS:
                break
        case = _sample("", rng.choice(["f32", "bf16", "f16"]), B, V, rng.choice([0, 0, 1, 50, _log_uniform(rng, 2, 4096)]),
                       rng.choice([1.0, 0.5, 0.9, 0.95]), rng.choice([0.0, 0.0, 0.02, 0.1]), rng.choice([0.0, 0.5, 0.8, 1.0, 1.3]),
                       rng.random() < 0.5)
    case.pop("name")  # (a drawn case has none)
    return case


# ------------------------------------------------------------------------------------------------ inputs


def _lengths(case, most):
    """Of every sequence: all alike, or spread evenly from a quarter of the longest up."""
    B = case["B"]
    return [most - (3 * most // 4) * b // max(B - 1, 1) if case["ragged"] else most for b in range(B)]


def _scattered(counts, most, page, g):
    """(pages of the pool, block table): each sequence has the pages that its positions need, scattered over a pool
    that is a little larger; the table's other entries are -1."""
    need = [-(-n // page) for n in counts]
    width, pool = -(-most // page), sum(need) + 8
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    column = torch.arange(width, device="cuda")
    held = torch.tensor(need, device="cuda")
    rank = held.cumsum(0) - held
    table = order[(rank[:, None] + column[None, :]).clamp(max=pool - 1)]
    return pool, torch.where(column[None, :] < held[:, None], table, -1).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = dict(case)
    B = case["B"]
    if case["kind"] == "sample":
        V = case["V"]
        # Logits of a language model: most words far below a few; whole rows shifted by a constant of their own.
        s["logits"] = (2.5 * randn(B, V) + 4.0 * randn(B, 1)).to(DTYPES[case["dtype"]])
        s["uniform"] = torch.rand(B, device="cuda", generator=g)
        if case["per_row"]:  # every second row goes without the filters
            odd = torch.arange(B, device="cuda") % 2 == 1
            s["top_k"] = torch.where(odd, 0, case["top_k"]).to(torch.int32)
            s["top_p"] = torch.where(odd, 1.0, case["top_p"]).to(torch.float32)
            s["min_p"] = torch.where(odd, 0.0, case["min_p"]).to(torch.float32)
            s["temperature"] = case["temperature"] * (0.75 + 0.5 * torch.rand(B, device="cuda", generator=g))
        return s
    Hkv, d, page = case["Hkv"], case["d"], case["page"]
    cache = DTYPES[case["cache"]]
    most = case["T"] + 37 if case["kind"] == "append" else case["length"]
    order = torch.randperm(B, generator=g, device="cuda")
    if case["kind"] == "append":
        counts = _lengths(case, case["T"])
        pool, table = _scattered([most] * B, most, page, g)
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")[order] if case["ragged"] else None
        s["positions"] = torch.randint(0, 38, (B,), generator=g, device="cuda", dtype=torch.int32)
        # a projection's output [B, T, kv heads * d], seen as [B, kv heads, T, d]
        s["k"], s["v"] = (randn(B, case["T"], Hkv, d).to(DTYPES[case["dtype"]]).transpose(1, 2) for _ in range(2))
        s["k_cache"], s["v_cache"] = (torch.zeros(pool, Hkv, page, d, device="cuda").to(cache) for _ in range(2))
        s["table"] = table
    else:
        lengths = torch.tensor(_lengths(case, most), dtype=torch.int32, device="cuda")[order]
        pool, table = _scattered(_lengths(case, most), most, page, g)
        s["lengths"], s["table"] = lengths, table[order].contiguous()
        s["k_cache"], s["v_cache"] = (randn(pool, Hkv, page, d).to(cache) for _ in range(2))
        capacity = table.shape[1] * page
        # weights as many steps of attention leave them: a few positions hold most of it
        live = torch.arange(capacity, device="cuda") < lengths[:, None, None]
        if case["kind"] == "evict":
            s["weights"] = torch.exp(2.0 * randn(B, Hkv, capacity)) * live
        elif case["weights"]:
            s["weights"] = torch.rand((B, Hkv, capacity), device="cuda", generator=g) * live
        else:
            s["weights"] = None
        if case["kind"] == "attention":
            s["q"] = (2.0 * randn(B, Hkv * case["G"], d)).to(DTYPES[case["dtype"]])
    s["k_scale"], s["v_scale"] = (0.75, 1.25) if case["cache"] == "e4m3" else (1.0, 1.0)
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _append_plain(s):
    B, Hkv, T, d = s["k"].shape
    size = s["k_cache"].shape[2]
    t = torch.arange(T, device=s["k"].device)
    at = s["positions"].long()[:, None] + t[None, :]
    there = torch.ones_like(at, dtype=torch.bool) if s["counts"] is None else t[None, :] < s["counts"][:, None]
    page = torch.gather(s["table"].long(), 1, at // size)

    def put(cache, x, scale):
        x = x.transpose(1, 2)[there]  # [tokens, kv heads, d]
        if cache.dtype == torch.float8_e4m3fn:
            x = (x.float() / scale).clamp(-E4M3_MAX, E4M3_MAX)
        codes = x.to(cache.dtype).contiguous()
        as_bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[cache.element_size()]
        cache.view(as_bits)[page[there], :, (at % size)[there]] = codes.view(as_bits)

    put(s["k_cache"], s["k"], s["k_scale"])
    put(s["v_cache"], s["v"], s["v_scale"])
    return s["k_cache"], s["v_cache"]


def _rows(cache, table, dtype):
    """[B, kv heads, positions, d] of a cache; whatever lies behind an unused entry of the table comes from page 0."""
    B, P = table.shape
    _, Hkv, size, d = cache.shape
    got = cache[table.long().clamp(min=0)].to(dtype)  # [B, P, kv heads, size, d]
    return got.transpose(1, 2).reshape(B, Hkv, P * size, d)


def _attention_plain(s):
    B, H, d = s["q"].shape
    Hkv = s["k_cache"].shape[1]
    q = s["q"].float().reshape(B, Hkv, H // Hkv, d)
    k, v = _rows(s["k_cache"], s["table"], torch.float32), _rows(s["v_cache"], s["table"], torch.float32)
    live = torch.arange(k.shape[2], device=q.device) < s["lengths"][:, None, None, None]
    scores = (k @ q.transpose(2, 3).contiguous()).transpose(2, 3) * (s["k_scale"] / math.sqrt(d))
    scores = scores.masked_fill(~live, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (e / e.sum(-1, keepdim=True)).contiguous()
    out = ((p @ v) * s["v_scale"]).reshape(B, H, d).to(s["q"].dtype)
    if s["weights"] is None:
        return out
    s["weights"] += p.sum(2)
    return out, s["weights"]


def _evict_plain(s):
    w, lengths = s["weights"], s["lengths"].long()[:, None, None]
    B, Hkv, capacity = w.shape
    budget = min(s["budget"], capacity)
    size = s["k_cache"].shape[2]
    t = torch.arange(capacity, device=w.device)
    rank = torch.where(t >= lengths - s["recent"], math.inf, w)
    rank = torch.where(t < lengths, rank, -math.inf)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget].sort(-1).values
    j = t[:budget].expand(B, Hkv, budget)
    kept = torch.where(lengths > s["budget"], kept, j)
    new = torch.minimum(lengths, torch.full_like(lengths, s["budget"]))
    table = s["table"].long().clamp(min=0)
    head = torch.arange(Hkv, device=w.device)[None, :, None].expand(B, Hkv, budget)
    from_page = torch.gather(table, 1, (kept // size).reshape(B, -1)).reshape(kept.shape)
    to_page = torch.gather(table, 1, (j // size).reshape(B, -1)).reshape(kept.shape)
    there = j < new
    to = (to_page[there], head[there], (j % size)[there])
    for cache in (s["k_cache"], s["v_cache"]):
        bits = cache.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[cache.element_size()])
        bits[to] = bits[from_page[there], head[there], (kept % size)[there]]
    moved = torch.where(there, torch.gather(w, 2, kept), w[..., :budget])
    w[..., :budget] = moved
    w.masked_fill_((t >= new) & (t < lengths), 0.0)
    return new.reshape(B).to(torch.int32), s["k_cache"], s["v_cache"], w


def _column(v, like):
    return v[:, None].double() if isinstance(v, torch.Tensor) else torch.full((like.shape[0], 1), v, device=like.device, dtype=torch.float32).double()


def _sample_plain(s):
    x = s["logits"].double()
    B, V = x.shape
    temperature, top_p, min_p = (_column(s[n], x) for n in ("temperature", "top_p", "min_p"))
    top_k = s["top_k"][:, None] if isinstance(s["top_k"], torch.Tensor) else torch.full((B, 1), s["top_k"], device=x.device)
    ordered, index = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((ordered - ordered[:, :1]) / torch.where(temperature > 0, temperature, 1.0))
    place = torch.arange(V, device=x.device)
    w = torch.where((top_k <= 0) | (place < top_k), w, 0.0)
    before = w.cumsum(-1) - w
    keep = (top_p >= 1) | (before < top_p * w.sum(-1, keepdim=True))
    keep &= (min_p <= 0) | (w >= min_p)
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0.0))
    running = w.cumsum(-1)
    token = (running > s["uniform"][:, None].double() * running[:, -1:]).int().argmax(-1)
    return torch.where(temperature[:, 0] > 0, token, index[:, 0])


# ------------------------------------------------------------------------------------------------ a pass


def run(s):
    kind = s["kind"]
    if own:
        from lighthouse_amd import ops

        if kind == "append":
            return ops.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["positions"], counts=s["counts"],
                                 k_scale=s["k_scale"], v_scale=s["v_scale"])
        if kind == "attention":
            out = ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], weights=s["weights"],
                                      k_scale=s["k_scale"], v_scale=s["v_scale"])
            return out if s["weights"] is None else (out, s["weights"])
        if kind == "evict":
            new = ops.kv_evict(s["k_cache"], s["v_cache"], s["weights"], s["table"], s["lengths"], s["budget"], recent=s["recent"])
            return new, s["k_cache"], s["v_cache"], s["weights"]
        return ops.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    if kind == "append":
        return _append_plain(s)
    if kind == "attention":
        return _attention_plain(s)
    return _evict_plain(s) if kind == "evict" else _sample_plain(s)


# ------------------------------------------------------------------------------------------------ 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _sample_exact(s)
    size = case["page"]
    table = s["table"].tolist()
    if case["kind"] == "append":
        for b, first in enumerate(s["positions"].tolist()):
            n = case["T"] if s["counts"] is None else int(s["counts"][b])
            slots = torch.arange(first, first + n, device="cuda")
            pages = s["table"][b].long()[slots // size]
            for cache, x, scale in ((s["k_cache"], s["k"], s["k_scale"]), (s["v_cache"], s["v"], s["v_scale"])):
                x = x[b, :, :n].transpose(0, 1)
                if case["cache"] == "e4m3":
                    x = torch.clamp(x.float() / scale, -E4M3_MAX, E4M3_MAX)
                bits = cache.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[cache.element_size()])
                bits[pages, :, slots % size] = x.to(cache.dtype).contiguous().view(bits.dtype)
        return s["k_cache"].double(), s["v_cache"].double()
    lengths = s["lengths"].tolist()
    if case["kind"] == "attention":
        G, d = case["G"], case["d"]
        out = torch.zeros(case["B"], case["Hkv"], G, d, dtype=torch.float64, device="cuda")
        weights = None if s["weights"] is None else s["weights"].double()
        for b, n in enumerate(lengths):
            pages = table[b][:-(-n // size)]
            for h in range(case["Hkv"]):
                k = s["k_cache"][pages, h].reshape(-1, d)[:n].double() * s["k_scale"]
                v = s["v_cache"][pages, h].reshape(-1, d)[:n].double() * s["v_scale"]
                q = s["q"][b, h * G:(h + 1) * G].double()
                p = torch.softmax((k @ q.t().contiguous()).t().contiguous() / math.sqrt(d), -1)
                out[b, h] = p @ v
                if weights is not None:
                    weights[b, h, :n] += p.sum(0)
        out = out.reshape(case["B"], -1, d)
        return out if weights is None else (out, weights)
    new = []
    for b, n in enumerate(lengths):
        m = min(n, case["budget"])
        new.append(m)
        if m == n:
            continue
        pages = torch.tensor(table[b], device="cuda")
        for h in range(case["Hkv"]):
            w = s["weights"][b, h]
            old = n - case["recent"]
            best = torch.argsort(w[:old], descending=True, stable=True)[:m - case["recent"]]
            kept = torch.cat([best.sort().values, torch.arange(old, n, device="cuda")])
            to = torch.arange(m, device="cuda")
            for cache in (s["k_cache"], s["v_cache"]):
                bits = cache.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[cache.element_size()])
                bits[pages[to // size], h, to % size] = bits[pages[kept // size], h, kept % size].clone()
            w[:m] = w[kept].clone()
            w[m:n] = 0.0
    return torch.tensor(new, dtype=torch.int32, device="cuda"), s["k_cache"].double(), s["v_cache"].double(), s["weights"].double()


def _sample_exact(s):
    import numpy as np

    rows = s["logits"].double().cpu().numpy()
    u = s["uniform"].double().cpu().numpy()

    def of_rows(v, dtype):
        return v.cpu().numpy() if isinstance(v, torch.Tensor) else np.full(len(rows), v, dtype)

    temperature, top_p, min_p = (of_rows(s[n], np.float32) for n in ("temperature", "top_p", "min_p"))
    top_k = of_rows(s["top_k"], np.int32)
    tokens = np.zeros(len(rows), np.int64)
    for r, x in enumerate(rows):
        order = np.argsort(-x, kind="stable")
        if temperature[r] <= 0:
            tokens[r] = order[0]
            continue
        n = min(int(top_k[r]), x.size) if top_k[r] > 0 else x.size
        w = np.exp((x[order[:n]] - x[order[0]]) / np.float64(temperature[r]))
        if top_p[r] < 1:
            n = max(1, int(np.searchsorted(np.concatenate([[0.0], np.cumsum(w)[:-1]]), np.float64(top_p[r]) * w.sum(), "left")))
        if min_p[r] > 0:
            n = max(1, min(n, int(np.count_nonzero(w >= np.float64(min_p[r])))))
        kept = np.sort(order[:n])
        running = np.cumsum(np.exp((x[kept] - x[order[0]]) / np.float64(temperature[r])))
        tokens[r] = kept[min(n - 1, int(np.searchsorted(running, u[r] * running[-1], "right")))]
    return torch.from_numpy(tokens)


# ------------------------------------------------------------------------------------------------ work


def work(case):
    B = case["B"]
    if case["kind"] == "sample":
        return {"bytes": B * case["V"] * BYTES[case["dtype"]] + 12 * B, "flops": 4 * B * case["V"]}
    Hkv, d, ec = case["Hkv"], case["d"], BYTES[case["cache"]]
    if case["kind"] == "append":
        values = 2 * sum(_lengths(case, case["T"])) * Hkv * d
        return {"bytes": values * (BYTES[case["dtype"]] + ec), "flops": 2 * values}
    lengths = _lengths(case, case["length"])
    if case["kind"] == "attention":
        rows = sum(lengths) * Hkv
        return {"bytes": 2 * rows * d * ec + 2 * B * Hkv * case["G"] * d * BYTES[case["dtype"]] + (8 * rows if case["weights"] else 0),
                "flops": 4 * rows * case["G"] * d}
    cut = [n for n in lengths if n > case["budget"]]
    kept = len(cut) * case["budget"] * Hkv
    return {"bytes": 4 * sum(cut) * Hkv + 2 * kept * 2 * d * ec + 4 * sum(cut) * Hkv, "flops": 2 * sum(cut) * Hkv}
