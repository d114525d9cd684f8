"""The root-mean-square norm with its residual and its result in 8 bits, against the formula in 64 bits."""

import math

import pytest
import torch

from lighthouse_amd import ops
from tests import packed_reference as ref
from tests.paged_reference import as_bits

pytestmark = pytest.mark.gpu

bf16, f16, f32, e4m3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def rows(M, C, dtype, seed, pad=0, size=1.0):
    x = (size * torch.randn(M, C + pad, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()
    return x[:, :C]


def check(x, gamma, residual, out, after=None, scales=None, scale=None, eps=1e-5, was=None):
    s, y, s_off, off = ref.rms_norm(x.cpu(), gamma.cpu(), eps, None if residual is None else (residual if was is None else was).cpu())
    if residual is not None:
        assert ((after.cpu().double() - s).abs() <= s_off + ref.half_step(after.dtype, s) + s_off * 2.0**-7).all()
    if out.dtype != e4m3:
        bad = ~((out.cpu().double() - y).abs() <= off + ref.half_step(out.dtype, y) + off * 2.0**-7)
        assert not bad.any(), float(((out.cpu().double() - y).abs() / (off + ref.half_step(out.dtype, y))).max())
        return
    if scales is not None:
        top = y.abs().amax(-1)
        assert ((scales.cpu().double() - top / 448).abs() <= (off / (y.abs() + 1e-300)).max() * top / 448 + 2 * ref.U * top / 448).all()
        scale = scales.cpu().double()[:, None]
    codes, want = out.cpu().float().double(), y / scale
    # the quotient: what y is off, and a rounding
    bad = ~((codes - want.clamp(-448, 448)).abs() <= (off / scale + ref.U * want.abs()) * 1.125 + ref.half_step(e4m3, want.clamp(-448, 448)))
    assert not bad.any()


SIZES = [(1, 1), (3, 7), (5, 8), (64, 768), (7, 513), (4, 1000), (9, 1024), (3, 1025), (5, 2048), (2, 2056), (3, 4096), (2, 5000), (3, 8192), (2, 8193),
         (2, 16384), (2, 16391), (1, 50257)]


@pytest.mark.parametrize("M,C", SIZES)
@pytest.mark.parametrize("dtype,residual,out", [(bf16, None, bf16), (bf16, f32, bf16), (f16, f16, f16), (f32, f32, bf16), (f32, None, f32), (bf16, bf16, f32), (f32, f32, f16)])
def test_types_and_sizes(M, C, dtype, residual, out):
    x, gamma = rows(M, C, dtype, C), (1 + 0.3 * torch.randn(C, generator=torch.Generator().manual_seed(1))).cuda()
    r = None if residual is None else rows(M, C, residual, C + 1, size=3.0)
    after = None if r is None else torch.empty_like(r)
    got = ops.rms_norm(x, gamma, residual=r, residual_out=after, out_dtype=out)
    assert got.dtype == out and got.shape == (M, C)
    check(x, gamma, r, got, after)
    if r is not None:  # in place
        was = r.clone()
        again = ops.rms_norm(x, gamma, residual=r, out_dtype=out)
        assert torch.equal(r, after) and torch.equal(again, got) and not torch.equal(was, r)


@pytest.mark.parametrize("M,C", SIZES)
@pytest.mark.parametrize("dtype,residual,scale", [(bf16, None, None), (bf16, f32, 0.01), (f16, f16, None), (f32, None, 0.02), (f32, f32, None), (bf16, bf16, 1e-30)])
def test_8_bits(M, C, dtype, residual, scale):
    x, gamma = rows(M, C, dtype, C, size=5.0), (1 + 0.3 * torch.randn(C, generator=torch.Generator().manual_seed(1))).cuda()
    r = None if residual is None else rows(M, C, residual, C + 1)
    after = None if r is None else torch.empty_like(r)
    got = ops.rms_norm(x, gamma, residual=r, residual_out=after, out_dtype=e4m3, scale=scale)
    if scale is None:
        check(x, gamma, r, got[0], after, scales=got[1])
        assert (got[0].float().abs().amax(-1) == 448).all()
    else:
        check(x, gamma, r, got, after, scale=float(torch.tensor(scale)))


@pytest.mark.parametrize("C", [8192, 4099])
@pytest.mark.parametrize("residual", [bf16, f32])
def test_large_sums(C, residual):
    """A sum that no cache holds, and the same rows a few at a time."""
    M = (36 << 20) // C // (4 if residual == f32 else 2)
    x, r, gamma = rows(M, C, bf16, 3), rows(M, C, residual, 4), torch.ones(C, device="cuda")
    after = torch.empty_like(r)
    out, scales = ops.rms_norm(x, gamma, residual=r, residual_out=after, out_dtype=e4m3)
    for part in (slice(0, 9), slice(M // 2, M // 2 + 9), slice(M - 9, M)):
        few = torch.empty_like(r[part])
        want, each = ops.rms_norm(x[part], gamma, residual=r[part], residual_out=few, out_dtype=e4m3)
        assert torch.equal(out[part].view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales[part], each) and torch.equal(after[part], few)


@pytest.mark.parametrize("C", [1000, 20000])
def test_more_than_2_to_the_31_values(C):
    M, gamma = 2**31 // C + 100, torch.ones(C, device="cuda")
    x = torch.zeros(M, C, dtype=bf16, device="cuda")
    x[-50:] = rows(50, C, bf16, 5)
    want = ops.rms_norm(x[-50:], gamma)
    assert ops.rms_norm(x, gamma, out=x) is x and torch.equal(x[-50:], want) and (x[:-50:997] == 0).all()


@pytest.mark.parametrize("C", [30, 768, 3000, 9000, 20000])
def test_strides(C):
    """Rows further apart than they are long, that begin anywhere; what lies between them stays."""
    x, r = rows(6, C, bf16, 1, pad=3), rows(6, C, f32, 2, pad=1)
    gamma = torch.randn(C + 1, generator=torch.Generator().manual_seed(3)).cuda()[1:]
    store = torch.full((6, C + 5), 7.0, dtype=f16, device="cuda")
    after = torch.full((6, C + 2), 9.0, dtype=f32, device="cuda")
    out = ops.rms_norm(x, gamma, 1e-6, residual=r, residual_out=after[:, :C], out=store[:, 1:C + 1])
    check(x, gamma, r, out, after[:, :C], eps=1e-6)
    assert (store[:, 0] == 7).all() and (store[:, C + 1:] == 7).all() and (after[:, C:] == 9).all()
    codes = torch.full((6, C + 5), 1.0, device="cuda").to(e4m3)
    scales = torch.zeros(8, device="cuda")
    ops.rms_norm(x, gamma, 1e-6, out=codes[:, 3:C + 3], row_scales=scales[:6])
    check(x, gamma, None, codes[:, 3:C + 3], scales=scales[:6], eps=1e-6)
    assert (codes.float()[:, :3] == 1).all() and (codes.float()[:, C + 3:] == 1).all() and (scales[6:] == 0).all()


def test_x_itself_receives_the_result():
    for C in (768, 5000, 20000):
        x, gamma = rows(4, C, bf16, 4), torch.ones(C, device="cuda")
        want = ops.rms_norm(x, gamma)
        assert ops.rms_norm(x, gamma, out=x) is x and torch.equal(x, want)


@pytest.mark.parametrize("C", [8, 900, 4000, 17000])
def test_zeros_infinities_and_nan(C):
    x, gamma = rows(6, C, f32, 5), torch.ones(C, device="cuda")
    x[1] = 0.0
    x[2, 3], x[3, 4], x[4, 5] = math.nan, math.inf, -math.inf
    out = ops.rms_norm(x, gamma)
    assert torch.isfinite(out[[0, 1, 5]]).all() and (out[1] == 0).all() and torch.isnan(out[2]).all()
    for row, col in ((3, 4), (4, 5)):  # an infinite mean: every other column is 0, its own a NaN
        assert torch.isnan(out[row, col]) and (out[row, torch.arange(C, device="cuda") != col] == 0).all()
    codes, scales = ops.rms_norm(x, gamma, out_dtype=e4m3)
    assert scales[1] == 1 and (codes[1].float() == 0).all() and torch.isnan(scales[2:5]).all() and torch.isnan(codes[2:5].float()).all()
    assert torch.isfinite(scales[[0, 5]]).all() and torch.isfinite(codes[[0, 5]].float()).all()
    fixed = ops.rms_norm(x, gamma, out_dtype=e4m3, scale=0.1)
    assert (fixed[1].float() == 0).all() and torch.isnan(fixed[2].float()).all() and torch.isfinite(fixed[[0, 5]].float()).all()
    # one row's do not reach another
    clean = x.clone()
    clean[2:5] = 1.0
    assert torch.equal(ops.rms_norm(clean, gamma)[[0, 1, 5]], out[[0, 1, 5]])


def test_nothing_to_do():
    x = torch.empty(0, 64, device="cuda")
    assert ops.rms_norm(x, torch.ones(64, device="cuda")).shape == (0, 64)


def test_the_result_feeds_a_product_of_8_bits():
    """codes scale_a times codes scale_b, as gemm_fp8 takes them, is the product of the normed rows to the rounding of the codes."""
    M, C, N = 64, 512, 256
    x, gamma = rows(M, C, bf16, 6), torch.ones(C, device="cuda")
    w = torch.randn(C, N, generator=torch.Generator().manual_seed(7)).cuda()
    w_codes = (w / 0.01).to(e4m3)
    codes = ops.rms_norm(x, gamma, out_dtype=e4m3, scale=0.02)
    got = ops.gemm_fp8(codes, w_codes, 0.02, 0.01, out_dtype=f32)
    want = (codes.double() * 0.02) @ (w_codes.double() * 0.01)
    size = (codes.double().abs() * 0.02) @ (w_codes.double().abs() * 0.01)
    assert ((got.double() - want).abs() <= (C + 4) * 2.0**-24 * size).all()
    codes, scales = ops.rms_norm(x, gamma, out_dtype=e4m3)
    got = ops.gemm_fp8(codes, w_codes, 1.0, 0.01, out_dtype=f32) * scales[:, None]
    _, y, _, _ = ref.rms_norm(x.cpu(), gamma.cpu(), 1e-5)
    exact = y @ (w_codes.cpu().double() * 0.01)
    size = y.abs() @ (w_codes.cpu().double().abs() * 0.01)
    assert ((got.cpu().double() - exact).abs() <= (2.0**-4 + 2.0**-9) * size + 1e-3).all()


def test_captured_and_replayed():
    x, r, gamma = rows(30, 768, bf16, 8), rows(30, 768, f32, 9), torch.ones(768, device="cuda")
    after = torch.empty_like(r)
    run = lambda: ops.rms_norm(x, gamma, residual=r, residual_out=after, out_dtype=e4m3)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        x.copy_(rows(30, 768, bf16, 20 + i))
        graph.replay()
        got = [as_bits(out[0]).clone(), out[1].clone(), after.clone()]
        want = run()
        torch.cuda.synchronize()
        assert torch.equal(got[0], as_bits(want[0])) and torch.equal(got[1], want[1]) and torch.equal(got[2], after)


@pytest.mark.parametrize("out_dtype", [bf16, f32, e4m3])
def test_more_rows_than_a_launch_has(out_dtype):
    """2^26 rows of a wave each are 2^32 threads: around where the second launch begins and at the end every row is what it is by itself."""
    M = 2**26 + 9
    g = torch.Generator(device="cuda").manual_seed(7)
    x, residual = (torch.randn(M, 2, device="cuda", generator=g).to(bf16) for _ in range(2))
    gamma, after = torch.tensor([1.5, -0.25], device="cuda"), torch.empty_like(residual)
    got = ops.rms_norm(x, gamma, residual=residual, residual_out=after, out_dtype=out_dtype)
    for some in (slice(0, 64), slice(2**26 - 64, 2**26 + 9)):
        part_after = torch.empty_like(residual[some])
        part = ops.rms_norm(x[some], gamma, residual=residual[some], residual_out=part_after, out_dtype=out_dtype)
        assert torch.equal(after[some], part_after)
        for whole, piece in zip(got, part) if out_dtype == e4m3 else [(got, part)]:
            assert torch.equal(as_bits(whole[some]), as_bits(piece))


@pytest.mark.parametrize("C", [16, 2000, 20000])
def test_rows_whose_scale_would_be_no_number(C):
    """Results of a few times 2^-149, the smallest number: it is the row's scale, and their codes are those whole numbers; zeros stay zeros."""
    x = torch.zeros(3, C, device="cuda")
    x[0, ::2], x[0, 1], x[2, 3] = 1.0, -1.0, 4.0
    gamma = torch.full((C,), 2.0**-147, device="cuda")
    out, scales = ops.rms_norm(x, gamma, out_dtype=e4m3)
    whole = ops.rms_norm(x, gamma).cpu().double() / 2.0**-149
    assert (whole[0].abs() <= 8).all() and whole[0].abs().max() >= 1 and (whole[1] == 0).all()
    assert scales[:2].tolist() == [2.0**-149, 1.0]
    assert torch.equal(out[:2].cpu().double(), whole[:2])
    top = float(whole[2].abs().max())  # (4 sqrt(C): above 224 the quotient by 448 is a number again)
    assert float(scales[2].double()) / 2.0**-149 == max(1.0, round(top / 448)) and torch.isfinite(out.float()).all()
