"""Sampling against the 64-bit statement of it: the token has to be the same one."""

import math

import numpy as np
import pytest
import torch

from lighthouse_amd import ops
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32


def check(logits, uniform, **options):
    x = logits.cuda()
    u = torch.as_tensor(uniform, dtype=f32)
    row = lambda v, b: v[b].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    got = ops.sample(x, u.cuda(), **{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in options.items()}).tolist()
    rows = logits.double().numpy()
    want = [ref.sample(rows[b], u[b].item(), **{k: row(v, b) for k, v in options.items()}) for b in range(len(rows))]
    assert got == want


FILTERS = [{}, {"top_k": 1}, {"top_k": 50}, {"top_p": 0.9}, {"min_p": 0.05}, {"top_k": 40, "top_p": 0.8}, {"top_k": 300, "top_p": 0.95, "min_p": 0.01},
           {"temperature": 0.0}, {"temperature": -1.0}, {"temperature": 0.05, "top_p": 0.9}, {"temperature": 5.0, "top_p": 0.99},
           {"top_p": 0.0}, {"top_p": 1e-6}, {"min_p": 2.0}, {"top_k": 10**6, "top_p": 0.5}, {"temperature": math.inf, "top_k": 9}]


@pytest.mark.parametrize("options", FILTERS, ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()) or "plain")
@pytest.mark.parametrize("dtype,V", [(f32, 5000), (bf16, 5000), (f16, 1237)])
def test_filters(options, dtype, V):
    g = torch.Generator().manual_seed(V)
    logits = (2.5 * torch.randn(24, V, generator=g) + 30).to(dtype)
    check(logits, torch.rand(24, generator=g), **options)


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 255, 256, 257, 1023, 1025, 4096, 8191, 16385, 50257])
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_sizes(V, dtype):
    g = torch.Generator().manual_seed(V)
    logits = (3 * torch.randn(6, V, generator=g)).to(dtype)
    u = torch.rand(6, generator=g)
    for options in ({}, {"top_k": 5}, {"top_p": 0.7}):
        check(logits, u, **options)


def test_a_large_vocabulary_with_settings_for_every_row():
    g = torch.Generator().manual_seed(1)
    logits = (2.5 * torch.randn(8, 131072, generator=g)).to(bf16)
    check(logits, torch.rand(8, generator=g), temperature=torch.tensor([0.7, 1.0, 1.3, 0.0, 0.9, 1.0, 2.0, 1.0]),
          top_k=torch.tensor([0, 50, 3000, 7, 0, 0, 20000, 0], dtype=torch.int32),
          top_p=torch.tensor([0.9, 0.95, 1.0, 0.5, 0.99, 1.0, 0.9, 0.3]), min_p=torch.tensor([0.0, 0.0, 0.1, 0.0, 0.02, 0.0, 0.0, 0.5]))


@pytest.mark.parametrize("dtype", [f32, bf16, f16])
def test_ties(dtype):
    """Few values, thousands of words each: the cut falls among words of one value, the lowest indices stay."""
    g = torch.Generator().manual_seed(2)
    logits = torch.randint(0, 3, (12, 6000), generator=g).to(dtype)
    u = torch.tensor([0.0, 0.1, 0.25, 0.5, 0.75, 0.9, 0.99, 0.999, 0.9999, 0.33, 0.66, 0.5])
    for options in ({}, {"top_k": 777}, {"top_k": 2500}, {"top_p": 0.3}, {"top_p": 0.8}, {"top_k": 1999, "top_p": 0.5}, {"temperature": 0.0}, {"top_k": 1}):
        check(logits, u, **options)
    same = torch.full((4, 4096), -3.5, dtype=dtype)
    check(same, [0.0, 0.25, 0.5, 0.75])
    check(same, [0.0, 0.25, 0.5, 0.75], top_p=0.5)
    check(same, [0.0, 0.25, 0.5, 0.75], top_k=1024)


@pytest.mark.parametrize("u", [0.0, -1.0, 1.0, 2.0, math.inf, math.nan, float(np.nextafter(np.float32(1), np.float32(0)))])
def test_numbers_at_the_ends(u):
    g = torch.Generator().manual_seed(3)
    logits = 4 * torch.randn(3, 900, generator=g)
    for options in ({}, {"top_k": 20}, {"top_p": 0.6}):
        check(logits, [u] * 3, **options)


def test_masked_words():
    """-inf and NaN are no words, the type's lowest value is one; rows of none and of one, infinite ones."""
    g = torch.Generator().manual_seed(4)
    x = 2 * torch.randn(10, 2000, generator=g)
    x[0, ::2] = -math.inf
    x[1, 5:] = -math.inf
    x[2] = -math.inf
    x[3, 1999] = 1.0
    x[3, :1999] = -math.inf
    x[4, ::3] = math.nan
    x[5] = math.nan
    x[6, ::2] = torch.finfo(f32).min
    x[7] = torch.finfo(f32).min
    x[8, [7, 100, 1500]] = math.inf
    x[9, ::2] = -1e9
    u = torch.rand(10, generator=g)
    for options in ({}, {"top_k": 30}, {"top_k": 2}, {"top_k": 1500}, {"top_p": 0.9}, {"top_p": 0.5, "top_k": 1500}, {"min_p": 0.1}, {"temperature": 0.0}, {"temperature": 1e-30}):
        check(x, u, **options)
    check(x.to(bf16), u, top_p=0.9)
    check(torch.full((2, 1), -math.inf), [0.5, 0.5])


def test_values_close_together_and_far_apart():
    """Differences of the last bit, of denormals and of the whole range of f32 all end in the right cut."""
    g = torch.Generator().manual_seed(5)
    near = (torch.full((4, 3000), 1.0).view(torch.int32) + torch.randint(0, 50, (4, 3000), generator=g).int()).view(f32)
    tiny = torch.randint(0, 90, (4, 3000), generator=g).int().view(f32)
    far = torch.randn(4, 3000, generator=g) * 10.0 ** torch.randint(-44, 38, (4, 3000), generator=g).double().float()
    u = torch.rand(4, generator=g)
    for x in (near, tiny, far):
        for options in ({}, {"top_k": 700}, {"top_k": 2999}, {"top_p": 0.4}, {"top_p": 0.95, "temperature": 1e30}, {"top_k": 1000, "temperature": 1e-20}):
            check(x, u, **options)


def test_rows_of_any_stride_and_alignment():
    g = torch.Generator().manual_seed(6)
    for dtype in (f32, bf16):
        store = torch.randn(5, 1003, generator=g).to(dtype).cuda()
        x = store[:, 1:778]
        u = torch.rand(5, generator=g)
        got = ops.sample(x, u.cuda(), top_p=0.8).tolist()
        assert got == [ref.sample(x[b].double().cpu().numpy(), u[b].item(), top_p=0.8) for b in range(5)]


def test_draws_follow_the_probabilities():
    """4096 draws from one row at evenly spaced numbers: each word as often as its share, to the one draw that its ends decide."""
    x = torch.tensor([0.3, -1.0, 2.0, 1.2, -math.inf, 0.0, 1.9])
    n = 4096
    u = (torch.arange(n, dtype=torch.float64) / n).float()
    got = ops.sample(x.repeat(n, 1).cuda(), u.cuda(), temperature=0.7)
    p = torch.softmax(x.double() / 0.7, 0)
    assert ((torch.bincount(got.cpu(), minlength=7) - n * p).abs() <= 1).all()
    assert (got.diff() >= 0).all()


@pytest.mark.parametrize("V", [8192, 8193, 16384, 20011, 131072, 524288, 524289])
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_rows_of_several_chunks(V, dtype):
    """From 8193 words on a row is digested in chunks, up to 524288."""
    g = torch.Generator().manual_seed(V)
    logits = (2.5 * torch.randn(3, V, generator=g)).to(dtype)
    logits[1] += torch.linspace(-30, 30, V).to(dtype)  # chunks whose largest words are far apart
    u = torch.rand(3, generator=g)
    for options in ({}, {"top_k": 40}, {"top_k": 512, "top_p": 0.9}, {"top_k": 513}, {"top_p": 0.9}, {"top_p": 0.2, "min_p": 0.01},
                    {"min_p": 0.001}, {"temperature": 0.0}, {"temperature": 0.1, "top_p": 0.95}):
        check(logits, u, **options)


def test_chunks_that_differ():
    """Empty chunks, one word, all of one value, infinite ones, values far from 0, ties at a chunk's border."""
    V = 40000
    g = torch.Generator().manual_seed(7)
    x = 2 * torch.randn(12, V, generator=g)
    x[0, 8192:24576] = -math.inf
    x[1] = -math.inf
    x[1, 30000] = 2.0
    x[2] = 0.5
    x[3, 5] = math.inf
    x[3, 39999] = math.inf
    x[4] += 1e6
    x[5] -= 1e30
    x[6] = torch.randint(0, 2, (V,), generator=g).float() * 60  # two values, far apart
    x[7] = math.nan
    x[8, 8000:8400] = 9.0
    x[9] *= 1e-30
    x[10] = -math.inf
    x[11, ::2] = torch.finfo(f32).min
    u = torch.tensor([0.1, 0.5, 0.5, 0.7, 0.3, 0.25, 0.5, 0.1, 0.6, 0.9, 0.3, 0.99])
    for options in ({}, {"top_k": 100}, {"top_k": 2}, {"top_p": 0.5}, {"top_p": 0.999}, {"min_p": 0.3}, {"min_p": 5.0}, {"temperature": 0.0},
                    {"top_k": 300, "top_p": 0.3}, {"temperature": 1e-20, "top_p": 0.5}, {"temperature": 1e20, "top_p": 0.5}, {"temperature": math.inf}):
        check(x, u, **options)
    same = torch.full((4, 32768), -3.5)
    check(same, [0.0, 0.25, 0.5, 0.75])
    check(same, [0.0, 0.25, 0.5, 0.75], top_p=0.5)


def test_workspace_of_the_caller():
    g = torch.Generator().manual_seed(8)
    x, u = torch.randn(2, 20000, generator=g).cuda(), torch.rand(2, generator=g).cuda()
    need = ops.sample_workspace_bytes(2, 20000)
    assert need > 0 and ops.sample_workspace_bytes(2, 8192) == 0
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.sample(x, u, top_p=0.9, workspace=ws), ops.sample(x, u, top_p=0.9))
    with pytest.raises(ValueError, match="workspace"):
        ops.sample(x, u, workspace=ws[: need - 256])


@pytest.mark.parametrize("V", [8192, 20011, 131072, 524288, 2**20, 2**24])
@pytest.mark.parametrize("dtype", [f32, bf16])
def test_a_likely_word_and_a_long_tail_of_unlikely_ones(V, dtype):
    """One word of weight 1 at the end, all others 2^-40 to 2^-52 of it: their sum is small, but not lost, and a draw below it falls on
    the one that it says, to what the units lose."""
    # Units of 2^-49 of a chunk's largest weight, half of one lost for each of 8192 words, the largest at least half of 2^power: 2^-36.  Where
    # one workgroup takes a row of several chunks, 2^-51, half of one for each: V 2^-52.  Without chunks and with a sum of 1, 2^-60, all of one.
    allowed = max(2.0**-36, V * (2.0**-52 if V <= 524288 else 2.0**-60))
    for octaves in (40.0, 42.9, 43.1, 44.9, 45.1, 47.0, 49.9, 50.1, 52.0):
        tail = torch.tensor(-octaves * math.log(2.0)).to(dtype)
        x = torch.full((1, V), tail.item()).to(dtype)
        x[0, -1] = 0.0
        w = math.exp(tail.double().item())
        for options, words in (({}, V - 1), ({"min_p": 1e-30}, V - 1), ({"top_k": 3000}, 2999), ({"top_k": 300}, 299)):
            u = torch.tensor([words * w * f for f in (0.0, 0.1, 0.5, 0.9)] + [0.5], dtype=f32)
            got = ops.sample(x.cuda().repeat(len(u), 1), u.cuda(), **options).tolist()
            whole = 1.0 + words * w
            for token, part in zip(got, u.double().tolist()):
                before = (words if token == V - 1 else token) * w
                assert token == V - 1 or 0 <= token < words
                assert before <= (part + allowed) * whole, (octaves, options, part, token)
                assert before + (1.0 if token == V - 1 else w) >= (part - allowed) * whole, (octaves, options, part, token)


def test_sums_of_chunks_far_apart():
    """A chunk holds one likely word, the others only unlikely ones of many sizes: top-p cuts where the sums in 64 bits do."""
    V = 131072
    g = torch.Generator().manual_seed(9)
    x = -25.0 - 15.0 * torch.rand(4, V, generator=g)
    x[0, 70000] = x[1, 0] = x[2, V - 1] = x[3, 8192] = 0.0
    x[:, 8192 * 4:8192 * 8] += torch.linspace(0.0, 20.0, 8192 * 4)
    check(x, [0.1, 0.9, 0.5, 0.999])
    check(x, [0.1, 0.9, 0.5, 0.999], top_p=0.9)
    check(x, [1e-4, 0.9, 0.5, 0.999], top_p=0.999)


@pytest.mark.parametrize("u", [1.0, math.inf, math.nan])
@pytest.mark.parametrize("V", [2, 900, 8192, 20000, 600000])
def test_a_number_of_one_or_none_takes_the_last_word_with_any_weight(u, V):
    """However little: down to what 64 bits hold, which 746 below the largest is no more."""
    x = torch.full((7, V), -math.inf)
    for b, least in enumerate((-20.0, -40.0, -300.0, -700.0, -744.0, -746.0, -1e30)):
        x[b, : V - 1] = -800.0
        x[b, 0], x[b, V - 1] = 0.0, least
    for options in ({}, {"top_k": 2}, {"top_k": 600}, {"top_p": 0.9}, {"min_p": 1e-20}, {"temperature": 2.0}, {"temperature": 0.5, "top_k": 700}, {"top_k": 1}):
        check(x, [u] * 7, **options)


@pytest.mark.parametrize("u", [0.0, -0.0, -1.0, -math.inf])
@pytest.mark.parametrize("V", [2, 900, 8192, 20000, 600000])
def test_a_number_of_zero_or_less_takes_the_first_word_with_any_weight(u, V):
    x = torch.full((7, V), -math.inf)
    for b, least in enumerate((-20.0, -40.0, -300.0, -700.0, -744.0, -746.0, -1e30)):
        x[b, 1:] = -800.0
        x[b, 0], x[b, V - 1] = least, 0.0
    for options in ({}, {"top_k": 2}, {"top_k": 600}, {"top_p": 0.9}, {"min_p": 1e-20}, {"temperature": 2.0}, {"temperature": 0.5, "top_k": 700}, {"top_k": 1}):
        check(x, [u] * 7, **options)
