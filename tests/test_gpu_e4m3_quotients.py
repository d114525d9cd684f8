"""Codes of 8 bits are those of the formula, e4m3(clamp(x / scale, +-448)), for every 16-bit number and scales of any kind, in every operator that makes them."""

import math

import pytest
import torch

from lighthouse_amd import ops

pytestmark = pytest.mark.gpu

bf16, f16, f32, e4m3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn

# 1; a mantissa of ones; of a one at either end; the borders of the short division and beyond them; the smallest numbers
SCALES = [1.0, 2.0 - 2.0**-23, 2.0**-9 - 2.0**-33, 1.0 + 2.0**-23, 1.5, 0.37, 2.0**-60, 2.0**-60 * (1 - 2.0**-24), 2.0**60, 2.0**60 * (1 + 2.0**-23), 2.0**-126, 2.0**-149, 2.0**100]


def every_number(dtype):
    return torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)


def codes_of(x, scale):
    return (x.float() / torch.tensor(scale, dtype=f32)).clamp(-448.0, 448.0).to(e4m3)


def same(got, want):
    got, want = got.cpu().float(), want.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype", [bf16, f16])
@pytest.mark.parametrize("d", [64, 61])
def test_stores_and_appended_tokens(scale, dtype, d):
    x = every_number(dtype)
    x = torch.cat([x, x[: -len(x) % d]]).view(-1, 1, d).cuda()
    N = x.shape[0]
    want = codes_of(x.cpu(), scale)
    k, v = (torch.zeros(N, 1, 1, d, dtype=e4m3, device="cuda") for _ in range(2))
    ops.kv_store(x, x, k, v, torch.arange(N, device="cuda"), k_scale=scale, v_scale=scale)
    same(k.view(N, 1, d), want), same(v.view(N, 1, d), want)
    k, v = (torch.zeros(N, 1, 1, d, dtype=e4m3, device="cuda") for _ in range(2))
    table = torch.arange(N, dtype=torch.int32, device="cuda")[None]
    tokens = x.transpose(0, 1)[None]
    ops.kv_append(tokens, tokens, k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"), k_scale=scale, v_scale=scale)
    same(k.view(N, 1, d), want), same(v.view(N, 1, d), want)


@pytest.mark.parametrize("scale", [s for s in SCALES if math.log2(s) > -130])
def test_norms(scale):
    """A result in f32, and the same in codes."""
    x = every_number(bf16)
    x = x[torch.isfinite(x.float()) & (x.float().abs() < 2.0**60)].cuda()
    x = x[: len(x) // 64 * 64].view(-1, 64)
    gamma = torch.ones(64, device="cuda")
    same(ops.rms_norm(x, gamma, out_dtype=e4m3, scale=scale), codes_of(ops.rms_norm(x, gamma, out_dtype=f32).cpu(), scale))
