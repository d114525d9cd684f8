"""Plain 64-bit statements of the operators over a paged key / value cache and of sampling, and caches to try them on."""

import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn


class Cache:
    """A cache whose every slot that no sequence uses holds NaN, its pages scattered, unused table entries outside the pool."""

    def __init__(self, lengths, heads, size, d, dtype, *, room=0, layout="heads", pad=0, seed=0, device="cuda", scales=(1.0, 1.0)):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.heads, self.size, self.d, self.dtype = list(lengths), heads, size, d, dtype
        B = len(lengths)
        self.P = max(1, max(-(-(n + room) // size) for n in lengths))
        held = [-(-(n + room) // size) for n in lengths]
        self.pages = sum(held) + 3
        order = torch.randperm(self.pages, generator=g).tolist()
        table = torch.full((B, self.P), -1, dtype=torch.int32)
        for b in range(B):
            for i in range(held[b]):
                table[b, i] = order.pop()
            if held[b] < self.P:
                table[b, -1] = (self.pages, 2**31 - 1, -(2**31))[b % 3]  # no page either
        self.k_scale, self.v_scale = scales
        self.k, self.v = (torch.randn(B, heads, max(lengths) if max(lengths) else 1, d, generator=g).to(dtype) for _ in range(2))
        self.table_cpu = table

        def store():
            shape = (self.pages, heads, size, d + pad) if layout == "heads" else (self.pages, size, heads, d + pad)
            full = torch.full(shape, math.nan).to(dtype).to(device)
            view = full[..., :d] if layout == "heads" else full[..., :d].transpose(1, 2)
            return view

        self.k_cache, self.v_cache = store(), store()
        for cache, x in ((self.k_cache, self.k), (self.v_cache, self.v)):
            host = as_bits(cache).cpu()
            for b in range(B):
                for t in range(lengths[b]):
                    host[table[b, t // size], :, t % size] = as_bits(x[b, :, t])
            as_bits(cache).copy_(host)
        self.table = table.to(device)
        self.device_lengths = torch.tensor(lengths, dtype=torch.int32, device=device)

    @property
    def capacity(self):
        return self.P * self.size

    def rows(self, cache, b, n):
        """The first n rows of sequence b: [heads, n, d], on the CPU."""
        host = as_bits(cache).cpu()
        if n == 0:
            return host.new_zeros(self.heads, 0, self.d).view(self.dtype)
        at = torch.arange(n)
        return host[self.table_cpu[b].long()[at // self.size], :, at % self.size].transpose(0, 1).contiguous().view(self.dtype)


def as_bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def attention(q, k, v, scale, v_scale=1.0):
    """(out, weights summed over the heads of a group, error allowed of out, of the weights) of one sequence, in 64 bits.
    q [H, d]; k, v [heads, n, d] as numbers (k times its scale).

    What may be off: the result's own rounding, half a step; a score, a sum of d products in f32, by (d + 8) steps of 2^-24 of the
    sum of their magnitudes, which is a relative error of its p; the sums over n positions by n + 64 such steps; P as two 16-bit
    values by the product of their half steps (and, in f16, by 2^-25, half its smallest step, of the largest p)."""
    H, d = q.shape
    heads, n = k.shape[:2]
    G = H // heads
    dtype = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(H, d, dtype=torch.float64)
    weights = torch.zeros(heads, n, dtype=torch.float64)
    allowed, w_allowed = torch.zeros(H, d, dtype=torch.float64), torch.zeros(heads, n, dtype=torch.float64)
    step = 2.0**-24
    half = torch.finfo(dtype).eps / 2
    for h in range(H):
        if n == 0:
            continue
        kk, vv = k[h // G], v[h // G]
        s = kk @ q[h] * scale
        p = torch.softmax(s, 0)
        out[h] = p @ vv * v_scale
        weights[h // G] += p
        off = 2 * (d + 8) * step * ((kk.abs() @ q[h].abs()) * abs(scale)).max() + (n + 64) * step
        split = 0.0 if dtype == torch.float32 else half * half
        size = p @ vv.abs() * v_scale
        tiny = n * 2.0**-25 * vv.abs().max() * v_scale * p.max() if dtype == torch.float16 else 0.0
        allowed[h] = half * out[h].abs() + (off + split) * size * (1 + half) + tiny + 1e-30
        w_allowed[h // G] += p * off
    return out, weights, allowed, w_allowed + step * weights * G


def evict(weights, n, budget, recent):
    """Which positions stay of one head's weights [n], in order."""
    if n <= budget:
        return list(range(n))
    w = weights[:n].double().cpu().numpy()
    rank = [(-math.inf if math.isnan(x) else x) for x in w]
    below = [math.isnan(x) for x in w]
    order = sorted(range(n - recent), key=lambda t: (below[t], -rank[t], t))
    return sorted(order[:budget - recent]) + list(range(n - recent, n))


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row: the words in falling order, the beginning that every filter leaves, the draw by index; sums in the
    widest floating point there is."""
    x = np.asarray(x, np.float64)
    words = np.flatnonzero(x > -np.inf)  # (NaN is not)
    if np.isposinf(x[words]).any():
        words = words[np.isposinf(x[words])]
    if not len(words):
        return -1
    order = words[np.lexsort((words, -x[words]))]
    top = x[order[0]]
    if not temperature > 0:
        return int(order[0])
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / np.float64(np.float32(temperature)))).astype(np.longdouble)
    n = len(order)
    if top_k > 0:
        n = min(n, top_k)
    if np.float32(top_p) < 1:
        before = np.concatenate([[0], np.cumsum(w[:n])[:-1]])
        n = max(1, int(np.count_nonzero(before < np.longdouble(np.float32(top_p)) * w[:n].sum())))
    if min_p > 0:
        n = max(1, int(np.count_nonzero(w[:n] >= np.float64(np.float32(min_p)))))
    by_index = np.argsort(order[:n])
    kept, w = order[:n][by_index], w[:n][by_index]
    if not u < 1:
        return int(kept[w > 0][-1])
    run = np.cumsum(w)
    above = np.flatnonzero(run > max(np.longdouble(np.float32(u)), 0) * run[-1])
    return int(kept[above[0]]) if len(above) else int(kept[w > 0][-1])
