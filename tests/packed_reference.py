"""Plain statements of the operators on packed tokens, in 64 bits (or as lists of whole numbers), with what a kernel's result may be off."""

import math

import torch

U = 2.0**-24  # half a step of an f32 of 1


def half_step(dtype, x):
    """Half a step of the type at |x|, that of its smallest normal number included."""
    smallest = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24, torch.float8_e4m3fn: 2.0**-9}[dtype]
    eps = {torch.float8_e4m3fn: 2.0**-3}.get(dtype) or torch.finfo(dtype).eps
    return eps / 2 * x.abs() + smallest / 2


def pages(table, lengths, counts, free, n_free, size, N):
    """One sequence after the other.  All lists; (lengths, starts, positions, slots, table, free, n_free) after the step."""
    table, free = [list(row) for row in table], list(free)
    B, P = len(table), len(table[0]) if table else 1
    old = [min(max(n, 0), P * size) for n in lengths]
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + max(c, 0))
    new = [0 if c < 0 else n + c for n, c in zip(old, counts)]
    fits = [new[b] <= P * size and starts[b + 1] <= N for b in range(B)]
    held = [next((j for j, p in enumerate(row) if not 0 <= p < len(free)), P) for row in table]
    need = [-(-n // size) for n in new]
    n_free = min(max(n_free, 0), len(free))
    for b in range(B):
        if fits[b]:
            for j in range(need[b], held[b]):
                if n_free < len(free):
                    free[n_free] = table[b][j]
                    n_free += 1
                table[b][j] = -1
    there, wanted = n_free, 0
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
                at = old[b] + i
                page = table[b][at // size]
                positions[starts[b] + i] = at
                slots[starts[b] + i] = page * size + at % size if 0 <= page < len(free) else -1
    return [n if f else o for n, o, f in zip(new, old, fits)], [min(s, N) for s in starts], positions, slots, table, free, n_free


def rotary(x, positions, freqs, interleaved=False, amplitude=1.0):
    """(result, error allowed before its rounding).  x [N, heads, d] on the CPU.

    Sine and cosine: the reduced angle, at most pi / 4, is rounded to f32, multiplied by 2 pi rounded to f32 and rounded: 3 U of it; the
    series' last two steps and what it leaves out 1.6 U: 4 U.  The amplitude is rounded to f32 and its product rounded, the products of the
    pair and their difference take a rounding each: 8 U (|a| + |b|) in all.  The angle in 64 bits: two roundings here and there."""
    x, half = x.double(), len(freqs)
    angle = positions.double()[:, None, None] * freqs.double()
    c, s = amplitude * angle.cos(), amplitude * angle.sin()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    out, allowed = x.clone(), torch.zeros_like(x)
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    off = abs(amplitude) * (8 * U + angle.abs() * 2.0**-51) * (a.abs() + b.abs())
    allowed[..., first] = allowed[..., second] = off
    return out, allowed


def rms_norm(x, gamma, eps, residual=None):
    """(s, y, error allowed of s, of y, before their roundings).  On the CPU.

    s: a rounding.  The sum of squares: at most C / 1024 + 64 additions one after the other, and a square's own error of 3 U;
    half of that for the root, and 7 roundings of the mean, eps, root, reciprocal and two products; the error of s in y."""
    C = x.shape[1]
    s = x.double() if residual is None else x.double() + residual.double()
    s_off = 0 * s if residual is None else U * s.abs()
    y = s / ((s * s).mean(-1, keepdim=True) + eps).sqrt() * gamma.double()
    return s, y, s_off, ((C / 1024 + 64 + 3) / 2 + 8) * U * y.abs()
