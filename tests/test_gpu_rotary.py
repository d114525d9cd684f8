"""Rotary positions and stores into slots against their definitions in 64 bits."""

import math

import pytest
import torch

from lighthouse_amd import ops
from tests import packed_reference as ref
from tests.paged_reference import as_bits

pytestmark = pytest.mark.gpu

bf16, f16, f32, e4m3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def case(N, heads, d, dtype, seed=0, pad=0, far=5000):
    g = torch.Generator().manual_seed(seed)
    x = torch.full((N, heads, d + pad), math.nan).to(dtype)
    x[..., :d] = (2 * torch.randn(N, heads, d, generator=g)).to(dtype)
    return x.cuda()[..., :d], torch.randint(0, far, (N,), generator=g, dtype=torch.int32).cuda()


def close(got, want, allowed, dtype):
    got = got.cpu().double()
    assert (torch.isfinite(got)).all()
    bad = ~((got - want).abs() <= allowed + ref.half_step(dtype, want) + allowed * 2.0**-3)
    assert not bad.any(), float(((got - want).abs() / (allowed + ref.half_step(dtype, want))).max())


@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,turned,pad", [(64, 64, 0), (128, 96, 0), (80, 80, 0), (2, 2, 0), (33, 6, 1), (93, 92, 0), (256, 2, 3), (7, 4, 0), (300, 300, 0), (40, 24, 1)])
def test_columns(dtype, interleaved, d, turned, pad):
    x, positions = case(9, 5, d, dtype, seed=d, pad=pad)
    freqs = ops.rotary_frequencies(turned)
    want, allowed = ref.rotary(x.cpu(), positions.cpu(), freqs.cpu(), interleaved)
    out = ops.rotary(x, positions, freqs, interleaved=interleaved)
    close(out, want, allowed, dtype)
    assert torch.equal(out[..., turned:], x[..., turned:])
    y = x.clone()  # (contiguous)
    assert ops.rotary(y, positions, freqs, interleaved=interleaved, out=y) is y and torch.equal(y, out)
    z = x[:, :3]
    ops.rotary(z, positions, freqs, interleaved=interleaved, out=z)  # some heads, where they lie
    assert torch.equal(x[:, :3], out[:, :3])


@pytest.mark.parametrize("N,heads", [(1, 1), (1, 130), (3000, 3), (513, 17), (70000, 1), (20000, 12)])
def test_few_and_many_tokens(N, heads):
    x, positions = case(N, heads, 64, bf16, seed=N)
    freqs = ops.rotary_frequencies(64)
    want, allowed = ref.rotary(x.cpu(), positions.cpu(), freqs.cpu())
    close(ops.rotary(x, positions, freqs), want, allowed, bf16)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,d,turned", [(5, 100, 72), (1, 64, 64), (3, 40, 6)])
def test_many_tokens_are_what_few_are(interleaved, heads, d, turned):
    """A call with as many values as have two heads a thread, and the same tokens 100 at a time."""
    x, positions = case(60000 // heads, heads, d, f16, seed=d)
    freqs = ops.rotary_frequencies(turned)
    whole = ops.rotary(x, positions, freqs, interleaved=interleaved)
    for at in range(0, x.shape[0], 1900):
        part = slice(at, at + 100)
        assert torch.equal(whole[part], ops.rotary(x[part], positions[part], freqs, interleaved=interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions_and_quarters_of_the_circle(interleaved):
    """Positions up to the largest number and below 0; angles right at, before and behind the borders of the eighths."""
    x = torch.randn(4096, 1, 32, generator=torch.Generator().manual_seed(1)).cuda()
    positions = torch.randint(-(2**31), 2**31 - 1, (4096,), generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda()
    positions[:4] = torch.tensor([2**31 - 1, -(2**31), 0, -1])
    freqs = ops.rotary_frequencies(32, base=1e6)
    want, allowed = ref.rotary(x.cpu(), positions.cpu(), freqs.cpu(), interleaved, 1.25)
    close(ops.rotary(x, positions, freqs, interleaved=interleaved, amplitude=1.25), want, allowed, f32)
    eighths = torch.tensor([math.pi / 4 * (1 + s) for s in (0, 1e-15, -1e-15, 1e-8, -1e-8, 1e-4, -1e-4, 0.5)] * 2, dtype=torch.float64)
    at = torch.arange(4096, dtype=torch.int32)
    want, allowed = ref.rotary(x.cpu(), at, eighths, interleaved)
    close(ops.rotary(x, at.cuda(), eighths.cuda(), interleaved=interleaved), want, allowed, f32)


def test_more_than_2_to_the_31_values():
    N, heads, d = 2**31 // (128 * 64) + 100, 128, 64
    x = torch.zeros(N, heads, d, dtype=bf16, device="cuda")
    x[-50:] = torch.randn(50, heads, d, generator=torch.Generator().manual_seed(1)).to(bf16).cuda()
    positions = torch.arange(N, dtype=torch.int32, device="cuda")
    freqs = ops.rotary_frequencies(d)
    want = ops.rotary(x[-50:], positions[-50:], freqs)
    assert ops.rotary(x, positions, freqs, out=x) is x and torch.equal(x[-50:], want) and (x[:-50:997] == 0).all()


def test_small_angles_of_either_sign():
    """Sines of small angles, alone in their columns, are right to the type's last places: a column of 0 beside one of 1."""
    x = torch.zeros(4, 1, 8, device="cuda")
    x[..., :4] = 1
    positions = torch.tensor([1, -1, 3, -70], dtype=torch.int32, device="cuda")
    freqs = torch.tensor([1e-3, 1e-9, 1e-14, 1e-20], dtype=torch.float64, device="cuda")
    for turn in (freqs, -freqs):
        got = ops.rotary(x, positions, turn)[:, 0, 4:].cpu().double()
        want = torch.sin(positions.cpu().double()[:, None] * turn.cpu())
        # the reduced angle and its product with 2 pi are rounded, the series' last sum, and the product with the amplitude and 1
        assert ((got - want).abs() <= 6 * 2.0**-24 * want.abs()).all()


def test_turning_back_and_the_gradient():
    x, positions = case(50, 4, 96, f32, seed=5)
    freqs = ops.rotary_frequencies(64)
    y = ops.rotary(x, positions, freqs)
    back = ops.rotary(y, positions, -freqs)
    size = x.abs() + y.abs() + 4.0
    assert ((back - x).abs() <= 20 * 2.0**-24 * size).all()
    # d / dx of sum(g * rotary(x)) is rotary(g, -freqs): against the formula, and against differences of the operator (linear: any step does)
    g = torch.randn(x.shape, generator=torch.Generator().manual_seed(6)).cuda()
    grad = ops.rotary(g, positions, -freqs)
    xx = x.cpu().double().requires_grad_()
    out, _ = ref.rotary(xx.detach(), positions.cpu(), freqs.cpu())
    angle = positions.cpu().double()[:, None, None] * freqs.cpu()
    a, b = xx[..., :32], xx[..., 32:64]
    formula = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), xx[..., 64:]], -1)
    assert torch.allclose(formula.detach(), out, atol=1e-12)
    (formula * g.cpu().double()).sum().backward()
    _, allowed = ref.rotary(g.cpu(), positions.cpu(), -freqs.cpu())
    close(grad, xx.grad, allowed, f32)
    step = torch.randn(x.shape, generator=torch.Generator().manual_seed(7)).cuda()
    by_difference = ((ops.rotary(x + step, positions, freqs).double() - ops.rotary(x - step, positions, freqs).double()) * g.double()).sum().item() / 2
    by_gradient = (grad.double() * step.double()).sum().item()
    # each result off by 10 U of its pair, of at most 2 (|x| + |step|)
    bound = 20 * 2.0**-24 * float(((x.abs() + step.abs()).double() * 2 * g.abs().double()).sum())
    assert abs(by_difference - by_gradient) <= bound


def test_scaled_frequencies():
    f = ops.rotary_frequencies(64, base=500.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1.0 and abs(f[-1].item() - 500.0 ** (-62 / 64)) < 1e-15
    assert torch.equal(ops.rotary_frequencies(64, base=500.0, factor=4.0, device="cpu"), f / 4)
    mixed = ops.rotary_frequencies(64, base=500.0, factor=4.0, context=100, low=1.0, high=8.0, device="cpu")
    turns = f * 100 / (2 * math.pi)
    assert torch.equal(mixed[turns >= 8], f[turns >= 8]) and torch.equal(mixed[turns <= 1], f[turns <= 1] / 4)
    between = (turns > 1) & (turns < 8)
    assert between.any() and ((mixed < f) & (mixed > f / 4))[between].all()


# ------------------------------------------------------------------------------------------------ stores


def caches(pages, heads, size, d, dtype, layout="heads", pad=0):
    shape = (pages, heads, size, d + pad) if layout == "heads" else (pages, size, heads, d + pad)
    make = lambda: torch.full(shape, math.nan).to(dtype).cuda()[..., :d]  # noqa: E731
    return [make() if layout == "heads" else make().transpose(1, 2) for _ in range(2)]


@pytest.mark.parametrize("dtype,cache_dtype", [(bf16, bf16), (f16, f16), (f32, f32), (bf16, e4m3), (f16, e4m3), (f32, e4m3)])
@pytest.mark.parametrize("d,turned,size,layout,pad", [(64, 64, 16, "heads", 0), (64, 0, 16, "slots", 0), (7, 4, 5, "slots", 0), (100, 96, 16, "slots", 3),
                                                      (1, 0, 1, "heads", 0), (256, 64, 32, "heads", 8), (93, 92, 24, "heads", 0)])
@pytest.mark.parametrize("H,interleaved", [(0, False), (6, True), (4, False)])
def test_store(dtype, cache_dtype, d, turned, size, layout, pad, H, interleaved):
    if H and not turned:
        pytest.skip("queries are passed to be turned")
    N, heads, pages = 37, 2, 11
    g = torch.Generator().manual_seed(d)
    qkv = (100 * torch.randn(N, (H + 2 * heads) * d, generator=g)).to(dtype).cuda().view(N, H + 2 * heads, d)
    q, k, v = qkv[:, :H], qkv[:, H:H + heads], qkv[:, H + heads:]
    k_cache, v_cache = caches(pages, heads, size, d, cache_dtype, layout, pad)
    before = [as_bits(c).cpu().clone() for c in (k_cache, v_cache)]
    slots = torch.randperm(pages * size, generator=g)[:N] if pages * size >= N else torch.arange(N)
    slots[5], slots[6], slots[7], slots[8] = -1, pages * size, 2**40, -(2**62)
    live = [(n, int(s)) for n, s in enumerate(slots) if 0 <= s < pages * size]
    positions = torch.randint(0, 9000, (N,), generator=g, dtype=torch.int32)
    scales = (0.37, 1.7) if cache_dtype == e4m3 else (1.0, 1.0)
    freqs = ops.rotary_frequencies(turned) if turned else None
    host = qkv.cpu().clone()
    turn = {"positions": positions.cuda(), "freqs": freqs, "interleaved": interleaved} if turned else {}
    got = ops.kv_store(k, v, k_cache, v_cache, slots.cuda(), k_scale=scales[0], v_scale=scales[1], **turn, **({"q": q} if H else {}))
    assert got[-2] is k_cache and got[-1] is v_cache and torch.equal(qkv.cpu(), host)
    if H:
        want, allowed = ref.rotary(q.cpu(), positions, freqs.cpu(), interleaved)
        close(got[0], want, allowed, dtype)
        q_at = qkv.clone()
        ops.kv_store(q_at[:, H:H + heads], q_at[:, H + heads:], k_cache, v_cache, slots.cuda(), k_scale=scales[0], v_scale=scales[1], q=q_at[:, :H], q_out=q_at[:, :H], **turn)
        assert torch.equal(q_at[:, :H], got[0]) and torch.equal(q_at[:, H:], qkv[:, H:])
    if turned:
        k_want, k_allowed = ref.rotary(k.cpu(), positions, freqs.cpu(), interleaved)
    else:
        k_want, k_allowed = k.cpu().double(), torch.zeros(k.shape, dtype=torch.float64)
    for cache, was, want, allowed, scale in ((k_cache, before[0], k_want, k_allowed, scales[0]), (v_cache, before[1], v.cpu().double(), 0 * k_allowed, scales[1])):
        bits, values = as_bits(cache).cpu(), cache.cpu().float().double()
        for n, s in live:
            row, ok = want[n], allowed[n]
            if cache_dtype == e4m3:  # (the quotient: the scale is an f32, a rounding)
                scale32 = float(torch.tensor(scale, dtype=f32))
                row, ok = (row / scale32), ok / scale32 + 2.0**-24 * (row / scale32).abs()
                ok = ok + (row.abs() > 448) * 0.0
                row = row.clamp(-448, 448)
            off = (values[s // size, :, s % size] - row).abs()
            assert (off <= ok * 1.125 + ref.half_step(cache_dtype, row)).all()
            if not turned and cache_dtype != e4m3:
                assert torch.equal(bits[s // size, :, s % size], as_bits((k if cache is k_cache else v)[n].cpu().contiguous()))
            was[s // size, :, s % size] = bits[s // size, :, s % size]
        assert torch.equal(bits, was)  # nothing else was written


def test_codes_are_those_of_the_formula():
    """Values that do not turn: e4m3(clamp(x / scale)), bit for bit, with infinities and NaN."""
    x = torch.randn(64, 2, 40, generator=torch.Generator().manual_seed(3)) * torch.logspace(-6, 6, 64)[:, None, None]
    x[0, 0, :6] = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0, 1e38])
    x = x.cuda()
    k_cache, v_cache = caches(4, 2, 16, 40, e4m3)
    slots = torch.arange(64, device="cuda")
    for scale in (1.0, 0.37, 1.9999999, 3e-30, 1e-42, 1e30):
        ops.kv_store(x, x, k_cache, v_cache, slots, k_scale=scale, v_scale=scale)
        want = (x / torch.tensor(scale, device="cuda")).clamp(-448.0, 448.0).to(e4m3)
        for cache in (k_cache, v_cache):
            got = cache.transpose(1, 2).reshape(64, 2, 40)
            nan = torch.isnan(want.float())
            assert torch.equal(torch.isnan(got.float()), nan) and torch.equal(as_bits(got)[~nan], as_bits(want)[~nan])


def test_infinities_and_nan_stay_where_they_are():
    x, positions = case(20, 3, 64, bf16, seed=8)
    x[3, 1, 5], x[4, 2, 40], x[5, 0, 63] = math.inf, math.nan, -math.inf
    freqs = ops.rotary_frequencies(32)
    clean = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)
    out, want = ops.rotary(x, positions, freqs), ops.rotary(clean, positions, freqs)
    hit = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
    hit[3, 1, 5] = hit[3, 1, 21] = hit[4, 2, 40] = hit[5, 0, 63] = True
    assert torch.equal(out[~hit], want[~hit]) and not torch.isfinite(out[hit]).any()
    assert out[5, 0, 63] == -math.inf


def test_many_tokens_are_stored():
    N, heads, d, size = 9000, 4, 128, 64
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v = (torch.randn(N, heads, d, device="cuda", generator=g).to(bf16) for _ in range(2))
    k_cache, v_cache = caches(N // size + 2, heads, size, d, bf16)
    slots = torch.randperm(k_cache.shape[0] * size, device="cuda", generator=g)[:N]
    positions = torch.arange(N, dtype=torch.int32, device="cuda")
    freqs = ops.rotary_frequencies(d)
    ops.kv_store(k, v, k_cache, v_cache, slots, positions=positions, freqs=freqs)
    turned = ops.rotary(k, positions, freqs)
    assert torch.equal(k_cache.transpose(1, 2).reshape(-1, heads, d)[slots], turned)
    assert torch.equal(v_cache.transpose(1, 2).reshape(-1, heads, d)[slots], v)
    assert torch.isnan(v_cache.float()).sum() == (v_cache.shape[0] * size - N) * heads * d


def test_captured_and_replayed():
    N, heads, d = 40, 2, 64
    g = torch.Generator(device="cuda").manual_seed(10)
    qkv = torch.randn(N, 8, d, device="cuda", generator=g).to(bf16)
    k_cache, v_cache = caches(5, heads, 16, d, bf16)
    other = caches(5, heads, 16, d, bf16)
    slots, positions = torch.arange(N, device="cuda"), torch.zeros(N, dtype=torch.int32, device="cuda")
    freqs = ops.rotary_frequencies(d)
    run = lambda c: (ops.kv_store(qkv[:, 4:6], qkv[:, 6:], *c, slots, q=qkv[:, :4], positions=positions, freqs=freqs)[0], ops.rotary(qkv, positions, freqs, interleaved=True))  # noqa: E731
    run((k_cache, v_cache))  # (warm; both caches hold the same from here on)
    run(other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run((k_cache, v_cache))
    for i in range(5):
        qkv.copy_(torch.randn(N, 8, d, device="cuda", generator=g))
        positions.copy_(torch.randint(0, 10000, (N,), device="cuda", generator=g))
        slots.copy_(torch.randperm(80, device="cuda", generator=g)[:N])
        graph.replay()
        want = run(other)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert torch.equal(as_bits(k_cache), as_bits(other[0])) and torch.equal(as_bits(v_cache), as_bits(other[1]))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("amplitude", [0.25, 1.3])
def test_the_gradient_at_an_amplitude(interleaved, amplitude):
    """Turning by -freqs at the same amplitude: against the formula's gradient, whose matrix is the transposed one."""
    g, positions = case(50, 4, 96, f32, seed=9)
    freqs = ops.rotary_frequencies(64)
    grad = ops.rotary(g, positions, -freqs, interleaved=interleaved, amplitude=amplitude)
    xx = torch.randn(g.shape, generator=torch.Generator().manual_seed(10), dtype=torch.float64).requires_grad_()
    angle = positions.cpu().double()[:, None, None] * freqs.cpu()
    a, b = (xx[..., 0:64:2], xx[..., 1:64:2]) if interleaved else (xx[..., :32], xx[..., 32:64])
    turned = [amplitude * (a * angle.cos() - b * angle.sin()), amplitude * (b * angle.cos() + a * angle.sin())]
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    (torch.cat([turned, xx[..., 64:]], -1) * g.cpu().double()).sum().backward()
    _, allowed = ref.rotary(g.cpu(), positions.cpu(), -freqs.cpu(), interleaved, amplitude)
    close(grad, xx.grad, allowed, f32)
