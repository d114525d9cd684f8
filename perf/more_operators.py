"""Prompts in chunks over a paged key / value cache: what these operators compute, and calls of real sizes.

A step of a server packs the new tokens of all sequences into N rows, those of sequence b at `starts[b] .. starts[b + 1] - 1`; some
sequences bring a piece of a prompt, some a single token, and rows behind the last may be left over.  Five operators of `lighthouse_amd.ops`:
`kv_pages` gives every sequence the pages that its new length needs (and takes those of sequences that ended), and says at which position and
in which slot each row lies; `rms_norm` adds a residual and scales rows to a root mean square of 1, in 8 bits where the next product
takes those; `rotary` turns queries or keys by angles that grow with the position; `kv_store` puts keys and values into their slots,
turning queries and keys on the way; `paged_attention_chunk` attends from every row to its sequence's positions up to its own.

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
LARGEST_PAGES = 1024 * 64                      # tokens of a step
LARGEST_ROTARY = 8192 * 40 * 128               # values
LARGEST_STORE = 8192 * 24 * 64
LARGEST_SCORES = 2048 * 32 * 16384             # of one call's attention, as its plain form makes them
LARGEST_CACHE = 2 * 4 * 16384 * 8 * 128 * 2    # bytes of keys and values
LARGEST_NORM = 8192 * 8192


def _pages(name, B, T, mode, length, page, free, ended):
    return {"name": name, "kind": "pages", "B": B, "T": T, "mode": mode, "length": length, "page": page, "free": free, "ended": ended}


def _rotary(name, dtype, N, H, d, turned, interleaved, far):
    return {"name": name, "kind": "rotary", "dtype": dtype, "N": N, "H": H, "d": d, "turned": turned, "interleaved": interleaved, "far": far}


def _store(name, dtype, cache, N, Hkv, G, d, turned, interleaved, page):
    return {"name": name, "kind": "store", "dtype": dtype, "cache": cache, "N": N, "Hkv": Hkv, "G": G, "d": d, "turned": turned,
            "interleaved": interleaved, "page": page}


def _chunk(name, dtype, cache, B, T, mode, Hkv, G, d, length, page):
    return {"name": name, "kind": "chunk", "dtype": dtype, "cache": cache, "B": B, "T": T, "mode": mode, "Hkv": Hkv, "G": G, "d": d,
            "length": length, "page": page}


def _norm(name, dtype, out, M, C, residual, scale):
    return {"name": name, "kind": "norm", "dtype": dtype, "out": out, "M": M, "C": C, "residual": residual, "scale": scale}


def listed():
    return [
        # One step of 64 sequences that each get a token; some begin a page, a few have ended.
        _pages("pages_step", 64, 1, "one", 1024, 16, 1.5, 0.05),
        # A full server: pieces of prompts among many single tokens, a tight pool.
        _pages("pages_prompts", 1024, 512, "mixed", 8192, 16, 1.0, 0.02),
        # Queries and keys of one step of the GPT that this repository's benchmark runs (12 heads of 64).
        _rotary("rotary_bf16_step", "bf16", 64, 24, 64, 64, False, 1024),
        # A long prompt's queries and keys, three quarters of the head turned, positions far out.
        _rotary("rotary_f16_prompt", "f16", 8192, 40, 128, 96, True, 1000000),
        # One step: queries turned, keys turned into the cache, values after them.
        _store("store_bf16_step", "bf16", "bf16", 64, 12, 1, 64, 64, False, 16),
        # Prompts into a cache of 8 bits, grouped heads.
        _store("store_e4m3_prompts", "bf16", "e4m3", 8192, 4, 4, 64, 64, False, 16),
        # A few drafted tokens of each sequence to be looked over at once: latency and the cache's bytes.
        _chunk("chunk_bf16_drafts", "bf16", "bf16", 8, 4, "even", 8, 4, 128, 4096, 16),
        # Prompts of a context of 1024 from their beginning (12 heads of 64).
        _chunk("chunk_bf16_prompts", "bf16", "bf16", 8, 1024, "even", 12, 1, 64, 1024, 16),
        # A piece of a long document with what came before: the largest.
        _chunk("chunk_f16_long", "f16", "f16", 1, 2048, "even", 8, 4, 128, 16384, 64),
        # Pieces of prompts among single tokens, from a cache of 8 bits.
        _chunk("chunk_e4m3_mixed", "bf16", "e4m3", 16, 512, "mixed", 4, 4, 128, 4096, 32),
        # One step between two layers, a residual in 32 bits.
        _norm("norm_bf16_step", "bf16", "bf16", 64, 768, "f32", 0.0),
        # A long prompt on its way into a product of 8 bits, a scale for every row.
        _norm("norm_bf16_e4m3_prompt", "bf16", "e4m3", 8192, 8192, "bf16", 0.0),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["pages", "rotary", "store", "chunk", "chunk", "chunk", "chunk", "norm", "norm"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    d = rng.choice([32, 64, 64, 80, 96, 128, 128, 256, rng.randint(2, 256)])
    turned = rng.choice([d // 2 * 2, d // 2 * 2, 2 * rng.randint(1, d // 2)])
    cache = rng.choice(["bf16", "bf16", "f16", "f32", "e4m3"])
    dtype = rng.choice(["bf16", "f16"]) if cache == "e4m3" else cache
    mode = rng.choice(["one", "even", "ragged", "ragged", "mixed"])
    if kind == "pages":
        while True:
            case = _pages("", _log_uniform(rng, 1, 1024), _log_uniform(rng, 1, 4096), mode, _log_uniform(rng, 1, 32768), page,
                          rng.choice([0.5, 1.0, 1.5]), rng.choice([0.0, 0.05, 0.3]))
            if sum(_counts(case)) <= LARGEST_PAGES:
                break
    elif kind == "rotary":
        while True:
            N, H = _log_uniform(rng, 1, 16384), rng.randint(1, 64)
            if N * H * d <= LARGEST_ROTARY:
                break
        case = _rotary("", rng.choice(["bf16", "f16", "f32"]), N, H, d, turned, rng.random() < 0.5, _log_uniform(rng, 64, 4000000))
    elif kind == "store":
        while True:
            N, Hkv, G = _log_uniform(rng, 1, 16384), rng.randint(1, 16), rng.choice([1, 2, 4, 5, 8])
            if N * Hkv * (G + 2) * d <= LARGEST_STORE:
                break
        case = _store("", dtype, cache, N, Hkv, G, d, turned, rng.random() < 0.5, page)
    elif kind == "chunk":
        while True:
            B, T, length = _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 2048), _log_uniform(rng, 1, 32768)
            Hkv, G = rng.randint(1, 16), rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
            case = _chunk("", dtype, cache, B, T, mode, Hkv, G, d, max(length, T), page)
            if B * max(_counts(case)) * Hkv * G * case["length"] <= LARGEST_SCORES and 2 * B * Hkv * case["length"] * d * BYTES[cache] <= LARGEST_CACHE:
                break
    else:
        while True:
            M, C = _log_uniform(rng, 1, 16384), _log_uniform(rng, 2, 16384)
            if M * C <= LARGEST_NORM:
                break
        dtype = rng.choice(["bf16", "f16", "f32"])
        out = rng.choice([dtype, dtype, "e4m3"])
        case = _norm("", dtype, out, M, C, rng.choice(["", dtype, "f32"]), rng.choice([0.0, 0.02]) if out == "e4m3" else 0.0)
    case.pop("name")  # (a drawn case has none)
    return case


# ------------------------------------------------------------------------------------------------ inputs


def _counts(case):
    """New tokens of every sequence: one each, as many each, from a quarter up, or every eighth a piece of a prompt and the others one."""
    B, T, mode = case["B"], case["T"], case["mode"]
    if mode == "one":
        return [1] * B
    if mode == "even":
        return [T] * B
    if mode == "ragged":
        return [T - (3 * T // 4) * b // max(B - 1, 1) for b in range(B)]
    return [T if b % 8 == 0 else 1 for b in range(B)]


def _lengths(case):
    """Of every sequence, the new tokens among them: from a quarter of the longest up."""
    B, most = case["B"], case["length"]
    return [max(c, most - (3 * most // 4) * ((b * 7) % B) // max(B - 1, 1)) for b, c in enumerate(_counts(case))]


def _frequencies(turned):
    return 10000.0 ** (-torch.arange(0, turned, 2, dtype=torch.float64, device="cuda") / turned)


def _scattered(counts, width, page, g, spare=8):
    """(pages of the pool, block table, pages that no sequence has): each sequence has the pages that its positions need, scattered; the
    table's other entries are -1."""
    held = torch.tensor([-(-n // page) for n in counts], device="cuda")
    pool = int(held.sum()) + spare
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    column = torch.arange(width, device="cuda")
    table = order[((held.cumsum(0) - held)[:, None] + column[None, :]).clamp(max=pool - 1)]
    return pool, torch.where(column[None, :] < held[:, None], table, -1).contiguous(), order[pool - spare:]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = dict(case)
    kind = case["kind"]
    if kind == "norm":
        M, C = case["M"], case["C"]
        # activations of a model: a few columns far larger than the others
        spread = torch.exp(0.5 * randn(C))
        s["x"] = (randn(M, C) * spread).to(DTYPES[case["dtype"]])
        s["residual"] = (3.0 * randn(M, C) * spread).to(DTYPES[case["residual"]]) if case["residual"] else None
        s["gamma"] = 1.0 + 0.2 * randn(C)
        s["after"] = torch.empty_like(s["residual"]) if case["residual"] else None
        return s
    if kind == "rotary":
        s["x"] = randn(case["N"], case["H"], case["d"]).to(DTYPES[case["dtype"]])
        s["positions"] = torch.randint(0, case["far"], (case["N"],), generator=g, device="cuda", dtype=torch.int32)
        s["freqs"] = _frequencies(case["turned"])
        return s
    page = case["page"]
    if kind == "store":
        N, Hkv, H, d = case["N"], case["Hkv"], case["Hkv"] * case["G"], case["d"]
        # a projection's output [N, (heads + 2 kv heads) d], seen as its three parts
        qkv = randn(N, H + 2 * Hkv, d).to(DTYPES[case["dtype"]])
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        pool = -(-N // page) + 3
        s["k_cache"], s["v_cache"] = (torch.zeros(pool, Hkv, page, d, device="cuda").to(DTYPES[case["cache"]]) for _ in range(2))
        # slots as kv_pages leaves them: runs of positions on scattered pages, a few rows that have none
        runs = torch.randperm(pool, generator=g, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
        slots = runs.reshape(-1)[:N].clone()
        slots[N - N // 16:] = -1
        s["slots"] = slots
        s["positions"] = (torch.arange(N, device="cuda") % 4096).to(torch.int32)
        s["freqs"] = _frequencies(case["turned"])
        s["k_scale"], s["v_scale"] = (0.02, 0.03) if case["cache"] == "e4m3" else (1.0, 1.0)
        return s
    B = case["B"]
    order = torch.randperm(B, generator=g, device="cuda")
    if kind == "pages":
        counts = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
        lengths = torch.tensor([n - c for n, c in zip(_lengths(case), _counts(case))], dtype=torch.int32, device="cuda")
        width = -(-max(_lengths(case)) // page)
        wanted = sum(-(-n // page) - -(-(n - c) // page) for n, c in zip(_lengths(case), _counts(case)))
        spare = max(1, int(wanted * case["free"]))
        pool, table, left = _scattered(lengths.tolist(), width, page, g, spare)
        s["counts"], s["lengths"], s["table"] = counts[order].contiguous(), lengths[order].contiguous(), table[order].contiguous()
        s["counts"][torch.rand(B, device="cuda", generator=g) < case["ended"]] = -1
        s["free_pages"] = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
        s["free_pages"][:spare] = left
        s["n_free"] = torch.tensor([spare], dtype=torch.int32, device="cuda")
        s["N"] = sum(_counts(case))
        return s
    counts, lengths = torch.tensor(_counts(case), device="cuda")[order], torch.tensor(_lengths(case), device="cuda")[order]
    pool, table, _ = _scattered(lengths.tolist(), -(-max(_lengths(case)) // page), page, g)
    s["starts"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    s["lengths"], s["table"] = lengths.to(torch.int32), table
    Hkv, d, N = case["Hkv"], case["d"], sum(_counts(case))
    s["longest"] = max(_counts(case))
    s["k_cache"], s["v_cache"] = (randn(pool, Hkv, page, d).to(DTYPES[case["cache"]]) for _ in range(2))
    s["q"] = (2.0 * randn(N, Hkv * case["G"], d)).to(DTYPES[case["dtype"]])
    s["k_scale"], s["v_scale"] = (0.75, 1.25) if case["cache"] == "e4m3" else (1.0, 1.0)
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _pages_plain(s):
    table, free, page, N = s["table"], s["free_pages"], s["page"], s["N"]
    B, P = table.shape
    counts, old = s["counts"].long(), s["lengths"].long().clamp(0, P * page)
    j = torch.arange(P, device=table.device)
    held = ((table >= 0) & (table < free.shape[0])).long().cumprod(1).sum(1)
    total = counts.clamp(min=0).cumsum(0)
    starts = torch.cat([total.new_zeros(1), total]).clamp(max=N).to(torch.int32)
    new = torch.where(counts < 0, 0, old + counts)
    fits = (new <= P * page) & (total <= N)
    need = (new + page - 1) // page
    # pages behind what is needed go back, in the order of the sequences and positions
    back = (j >= need[:, None]) & (j < held[:, None]) & fits[:, None]
    n = s["n_free"].long()
    place = n + back.reshape(-1).long().cumsum(0) - 1
    free[place[back.reshape(-1)]] = table[back]
    table[back] = -1
    n = n + back.sum()
    # what is missing is taken from the end of the list, sequence by sequence while there is enough
    more = torch.where(fits, (need - held).clamp(min=0), 0)
    fits &= (more == 0) | (more.cumsum(0) <= n)
    take = (j >= held[:, None]) & (j < need[:, None]) & fits[:, None]
    place = n - take.reshape(-1).long().cumsum(0)
    table[take] = free[place[take.reshape(-1)]]
    s["n_free"].copy_(n - take.sum())
    i = torch.arange(N, device=table.device)
    b = torch.searchsorted(total, i, right=True).clamp(max=B - 1)
    there = (i < total[-1]) & fits[b]
    at = torch.where(there, old[b] + i - (total - counts.clamp(min=0))[b], 0)
    slots = torch.where(there, table[b, at // page].long() * page + at % page, -1)
    lengths = torch.where(fits, new, old).to(torch.int32)
    return lengths, starts, torch.where(there, at, -1).to(torch.int32), slots, table, free, s["n_free"]


def _turn(x, positions, freqs, interleaved):
    """In 32 bits, with angles in 64: pairs of columns (i, i + half) or (2 i, 2 i + 1)."""
    angle = positions.double()[:, None, None] * freqs
    c, n, half, x = angle.cos().float(), angle.sin().float(), freqs.shape[0], x.float()
    a, b = (x[..., :2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    a, b = a * c - b * n, b * c + a * n
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _store_plain(s):
    slots, size = s["slots"], s["page"]
    there = slots >= 0
    q = _turn(s["q"], s["positions"], s["freqs"], s["interleaved"]).to(s["q"].dtype)

    def put(cache, x, scale):
        x = x[there]
        if cache.dtype == torch.float8_e4m3fn:
            x = (x / scale).clamp(-E4M3_MAX, E4M3_MAX)
        codes = x.to(cache.dtype).contiguous()
        as_bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[cache.element_size()]
        cache.view(as_bits)[slots[there] // size, :, slots[there] % size] = codes.view(as_bits)

    put(s["k_cache"], _turn(s["k"], s["positions"], s["freqs"], s["interleaved"]), s["k_scale"])
    put(s["v_cache"], s["v"].float(), s["v_scale"])
    return q, s["k_cache"], s["v_cache"]


def _rows(cache, table):
    """[B, kv heads, positions, d] of a cache; whatever lies behind an unused entry of the table comes from page 0."""
    B, P = table.shape
    _, Hkv, size, d = cache.shape
    return cache[table.long().clamp(min=0)].float().transpose(1, 2).reshape(B, Hkv, P * size, d)


def _chunk_plain(s):
    q, starts = s["q"], s["starts"].long()
    N, H, d = q.shape
    Hkv = s["k_cache"].shape[1]
    B, T = starts.shape[0] - 1, s["longest"]
    k, v = _rows(s["k_cache"], s["table"]), _rows(s["v_cache"], s["table"])
    i = torch.arange(T, device=q.device)
    row = (starts[:-1, None] + i).clamp(max=N - 1)  # (rows behind a sequence's last are computed and dropped)
    padded = q[row].float().reshape(B, T, Hkv, H // Hkv, d).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, d)
    at = s["lengths"].long()[:, None] - (starts[1:] - starts[:-1])[:, None] + i
    seen = torch.arange(k.shape[2], device=q.device) <= at[:, :, None]
    scores = (padded @ k.transpose(2, 3).contiguous()).mul_(s["k_scale"] / math.sqrt(d)).view(B, Hkv, T, H // Hkv, -1)
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    e = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    o = (e / e.sum(-1, keepdim=True)).view(B, Hkv, T * (H // Hkv), -1) @ v * s["v_scale"]
    o = o.view(B, Hkv, T, H // Hkv, d).transpose(1, 2).reshape(B, T, H, d).to(q.dtype)
    b = torch.searchsorted(starts[1:], torch.arange(N, device=q.device), right=True)
    return o[b, torch.arange(N, device=q.device) - starts[b]]


def _norm_plain(s):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
        s["after"].copy_(x)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * s["gamma"]
    scales = None
    if s["out"] == "e4m3":
        if s["scale"]:
            y = (y / s["scale"]).clamp(-E4M3_MAX, E4M3_MAX)
        else:
            scales = y.abs().amax(-1) / E4M3_MAX
            y = (y / scales[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return [t for t in (y.to(DTYPES[s["out"]]), s["after"], scales) if t is not None]


# ------------------------------------------------------------------------------------------------ a pass


def run(s):
    kind = s["kind"]
    if own:
        from lighthouse_amd import ops

        if kind == "pages":
            plan = ops.kv_pages(s["table"], s["lengths"], s["counts"], s["free_pages"], s["n_free"], s["page"], s["N"])
            return *plan, s["table"], s["free_pages"], s["n_free"]
        if kind == "rotary":
            return ops.rotary(s["x"], s["positions"], s["freqs"], interleaved=s["interleaved"])
        if kind == "store":
            return ops.kv_store(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], q=s["q"], positions=s["positions"], freqs=s["freqs"],
                                interleaved=s["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        if kind == "chunk":
            return ops.paged_attention_chunk(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["starts"],
                                             k_scale=s["k_scale"], v_scale=s["v_scale"])
        if s["out"] == "e4m3" and not s["scale"]:
            out, scales = ops.rms_norm(s["x"], s["gamma"], residual=s["residual"], residual_out=s["after"], out_dtype=DTYPES["e4m3"])
        else:
            scales = None
            out = ops.rms_norm(s["x"], s["gamma"], residual=s["residual"], residual_out=s["after"], out_dtype=DTYPES[s["out"]],
                               scale=s["scale"] or None)
        return [t for t in (out, s["after"], scales) if t is not None]
    if kind == "pages":
        return _pages_plain(s)
    if kind == "rotary":
        return _turn(s["x"], s["positions"], s["freqs"], s["interleaved"]).to(s["x"].dtype)
    if kind == "store":
        return _store_plain(s)
    return _chunk_plain(s) if kind == "chunk" else _norm_plain(s)


# ------------------------------------------------------------------------------------------------ 64 bits


def _turned_exactly(x, positions, turned, interleaved):
    """As a product of complex numbers."""
    f = 10000.0 ** (-torch.arange(0, turned, 2, dtype=torch.float64, device="cuda") / turned)
    turn = torch.polar(torch.ones_like(f)[None].expand(x.shape[0], -1), positions.double()[:, None] * f)[:, None]
    out, half = x.double().clone(), turned // 2
    if interleaved:
        out[..., :turned] = torch.view_as_real(torch.view_as_complex(out[..., :turned].reshape(*x.shape[:2], half, 2).contiguous()) * turn).flatten(-2)
    else:
        z = torch.complex(out[..., :half].contiguous(), out[..., half:turned].contiguous()) * turn
        out[..., :half], out[..., half:turned] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _turned_exactly(s["x"], s["positions"], case["turned"], case["interleaved"])
    if kind == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x = x + s["residual"].double()
        after = x
        y = x / ((x ** 2).sum(-1, keepdim=True) / case["C"] + 1e-5).sqrt() * s["gamma"].double()
        scales = None
        if case["out"] == "e4m3":
            scales = y.abs().max(-1).values / 448 if not case["scale"] else None
            y = (y / (case["scale"] if scales is None else scales[:, None])).clamp(-448, 448)
        return [t for t in (y, after if s["residual"] is not None else None, scales) if t is not None]
    size = case["page"]
    if kind == "store":
        k = _turned_exactly(s["k"], s["positions"], case["turned"], case["interleaved"]) / s["k_scale"]
        out = [_turned_exactly(s["q"], s["positions"], case["turned"], case["interleaved"])]
        there = (s["slots"] >= 0).nonzero()[:, 0]
        for x in (k, s["v"].double() / s["v_scale"]):
            if case["cache"] == "e4m3":
                x = x.clamp(-448, 448)
            rows = torch.zeros(s["k_cache"].shape[0] * size, case["Hkv"], case["d"], dtype=torch.float64, device="cuda")
            rows[s["slots"][there]] = x[there]
            out.append(rows.view(-1, size, case["Hkv"], case["d"]).transpose(1, 2).contiguous())
        return out
    if kind == "pages":
        return _pages_exactly(s)
    q, G, d = s["q"], case["G"], case["d"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for b, n in enumerate(lengths):
        count = starts[b + 1] - starts[b]
        pages = s["table"][b, :-(-n // size)].long()
        hidden = torch.arange(n, device="cuda")[None] > (n - count + torch.arange(count, device="cuda"))[:, None]
        for h in range(case["Hkv"]):
            k, v = (c[pages, h].reshape(-1, d)[:n].double() for c in (s["k_cache"], s["v_cache"]))
            for g in range(h * G, (h + 1) * G):
                x = q[starts[b]:starts[b + 1], g].double() @ k.t().contiguous() * (s["k_scale"] / math.sqrt(d))
                out[starts[b]:starts[b + 1], g] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v * s["v_scale"]
    return out


def _pages_exactly(s):
    """One sequence after the other, as lists."""
    table, lengths, counts = s["table"].tolist(), s["lengths"].tolist(), s["counts"].tolist()
    free, n_free = s["free_pages"].tolist(), int(s["n_free"])
    B, size, room, N = len(table), s["page"], len(table[0]) * s["page"], s["N"]
    starts, new = [0], []
    for b in range(B):
        starts.append(starts[-1] + max(counts[b], 0))
        new.append(0 if counts[b] < 0 else lengths[b] + counts[b])
    fits = [new[b] <= room and starts[b + 1] <= N for b in range(B)]
    held = [next((j for j, p in enumerate(row) if not 0 <= p < len(free)), len(row)) for row in table]
    need = [-(-n // size) for n in new]
    for b in range(B):
        if fits[b]:
            for j in range(need[b], held[b]):
                free[n_free], table[b][j] = table[b][j], -1
                n_free += 1
    wanted, there = 0, n_free
    positions, slots = [-1] * N, [-1] * N
    for b in range(B):
        more = max(need[b] - held[b], 0) if fits[b] else 0
        wanted += more
        fits[b] = fits[b] and (more == 0 or wanted <= there)
        if fits[b]:
            for j in range(held[b], need[b]):
                n_free -= 1
                table[b][j] = free[n_free]
            for i in range(max(counts[b], 0)):
                at = lengths[b] + i
                positions[starts[b] + i], slots[starts[b] + i] = at, table[b][at // size] * size + at % size
    lengths = [n if f else o for n, o, f in zip(new, lengths, fits)]
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, [min(x, N) for x in starts], positions)]
    return *ints, torch.tensor(slots, device="cuda"), *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (table, free, [n_free]))


# ------------------------------------------------------------------------------------------------ work


def work(case):
    kind = case["kind"]
    if kind == "pages":
        N, B = sum(_counts(case)), case["B"]
        moved = sum(-(-n // case["page"]) - -(-(n - c) // case["page"]) for n, c in zip(_lengths(case), _counts(case)))
        return {"bytes": 12 * N + 16 * B + 8 * moved, "flops": 4 * N + 8 * B}
    if kind == "rotary":
        values = case["N"] * case["H"] * case["d"]
        return {"bytes": 2 * values * BYTES[case["dtype"]] + 4 * case["N"] + 4 * case["turned"], "flops": 3 * case["N"] * case["H"] * case["turned"]}
    if kind == "store":
        N, Hkv, G, d, e = case["N"], case["Hkv"], case["G"], case["d"], BYTES[case["dtype"]]
        there = N - N // 16
        return {"bytes": 2 * N * Hkv * G * d * e + 2 * there * Hkv * d * (e + BYTES[case["cache"]]) + 12 * N,
                "flops": 3 * (N * G + there) * Hkv * case["turned"]}
    if kind == "norm":
        values, r = case["M"] * case["C"], case["residual"]
        return {"bytes": values * (BYTES[case["dtype"]] + BYTES[case["out"]] + (2 * BYTES[r] if r else 0)) + 4 * case["C"], "flops": 4 * values}
    counts, lengths = _counts(case), _lengths(case)
    H, d = case["Hkv"] * case["G"], case["d"]
    pairs = sum(c * (n - c) + c * (c + 1) // 2 for c, n in zip(counts, lengths))
    return {"bytes": 2 * sum(lengths) * case["Hkv"] * d * BYTES[case["cache"]] + 2 * sum(counts) * H * d * BYTES[case["dtype"]],
            "flops": 4 * pairs * H * d}
