"""Microscaled 4-bit floating point on the GPU against its definition in 64 bits.

Quantised rows are exact. Behind a norm, whose fp32 result is off by at most 2^-19 of a
value (32 squares added in fp32, 2^-20 of the root's, and three products), scales and
codes are those of values within that of the exact ones. Products are held to the 64-bit
result within the bound of fp32 sums (K additions) plus one rounding to the type."""

import pytest
import torch

from oracle.block_ref import half_step, within
from oracle.fp4_ref import (BLOCK, GRID, block_scales, nearest, over_scale, pack, product_ref, quantize_ref, rows_scales,
                            scale_values, values_ref)
from sglite_b200 import ops

pytestmark = pytest.mark.gpu

FORMATS = ["nvfp4", "mxfp4"]
DTYPES = [torch.bfloat16, torch.float16]


def _normal(cuda, M, K, dtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed + 31 * M + K)
    x = torch.randn((M, K), generator=g, device=cuda)
    x *= torch.where(torch.rand(K, generator=g, device=cuda) < 0.02, 20.0, 1.0)
    return x.to(dtype)


def _scale(cuda, fmt, value=0.0137):
    return torch.full((1,), value, device=cuda) if fmt == "nvfp4" else None


def _held(codes, scales, fmt):
    K = 2 * codes.shape[1]
    return values_ref(codes, rows_scales(scales, K, fmt), fmt)


def _same(got, want):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def _check_quantized(codes, scales, x, fmt, scale):
    K = x.shape[-1]
    want, byte = quantize_ref(over_scale(x.cpu(), scale), fmt)
    assert torch.equal(rows_scales(scales, K, fmt), byte)
    _same(_held(codes, scales, fmt), want)
    past = scales.cpu().transpose(0, 1).flatten(1)[:, K // BLOCK[fmt]:]
    assert not past.any()


# ---------------------------------------------------------------- rows
@pytest.mark.parametrize("M,K", [(1, 32), (1, 4096), (3, 96), (7, 256), (5, 288), (33, 544), (2, 16384), (129, 768),
                                 (1000, 64), (17, 2880)])
@pytest.mark.parametrize("fmt,scale", [("nvfp4", None), ("nvfp4", 0.0137), ("nvfp4", 2.0 ** -6), ("mxfp4", None)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize(cuda, M, K, fmt, dtype, scale):
    x = _normal(cuda, M, K, dtype)
    s = None if scale is None else torch.full((1,), scale, device=cuda)
    codes, scales = ops.fp4_quantize(x, fmt, scale=s)
    _check_quantized(codes, scales, x, fmt, s)
    back = ops.fp4_dequantize(codes, scales, fmt, dtype, scale=s)
    held = _held(codes, scales, fmt)
    want = (held.float() * (s.cpu() if s is not None else 1.0)).to(dtype)
    assert torch.equal(back.cpu(), want)


def _edges(dtype, fmt):
    """Blocks at the edges: ties of every code, borders of the scales, zeros, tiny and huge
    values, infinities and NaN."""
    tiny = torch.finfo(dtype).smallest_normal
    top = torch.finfo(dtype).max
    mids = ((GRID[:-1] + GRID[1:]) / 2).tolist()
    rows = []
    n = BLOCK[fmt]
    for s in [1.0, 0.75, 1.5, 2.0 ** -9, 416.0, 0.40625]:
        ties = [6.0] + mids + [-m for m in mids] + GRID.tolist() + (-GRID).tolist()
        rows += [[t * s for t in ties[:n - 1]] + [6 * s], [t * s * (1 + 2.0 ** -7) for t in ties[:n - 1]] + [6 * s]]
    for most in [0.0, -0.0, tiny, -tiny, tiny / 16, top, -top, top / 2, 448 * 6.0, 449 * 6.0, 480 * 6.0, 2.0 ** -10 * 6,
                 2.0 ** -10 * 6 * (1 + 2.0 ** -7), 2.0 ** -11, 1.0, 1.9921875, 2.0, 7.0, 8.0, 6.25, 6.375, 6.5]:
        rows.append([most] + [most * (i / 40 - 0.3) for i in range(n - 1)])
        rows.append([0.0] * (n - 1) + [most])
    for bad in [float("inf"), -float("inf"), float("nan")]:
        for at in (0, n // 2 + 1, n - 1):
            r = [0.25 * i for i in range(n)]
            r[at] = bad
            rows.append(r)
    while len(rows) * n % 32:
        rows.append([1.0] * n)
    return torch.tensor(rows, dtype=torch.float64).flatten().to(dtype)


@pytest.mark.parametrize("fmt,scale", [("nvfp4", None), ("nvfp4", 2.0 ** -3), ("nvfp4", 0.3), ("nvfp4", 1e-30),
                                       ("mxfp4", None)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_edges(cuda, fmt, dtype, scale):
    x = _edges(dtype, fmt)[None].to(cuda)
    s = None if scale is None else torch.full((1,), scale, device=cuda)
    codes, scales = ops.fp4_quantize(x, fmt, scale=s)
    _check_quantized(codes, scales, x, fmt, s)
    assert torch.isnan(ops.fp4_dequantize(codes, scales, fmt, dtype, scale=s)).any()


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_value_of_sixteen_bits(cuda, fmt):
    """Each finite bf16 beside a larger one: all scales and codes."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    bits = bits[torch.isfinite(bits.float())]
    n = bits.numel() // 64 * 64
    x = torch.cat([bits[:n], bits[torch.randperm(n, generator=torch.Generator().manual_seed(1))]]).view(-1, 64).to(cuda)
    codes, scales = ops.fp4_quantize(x, fmt)
    _check_quantized(codes, scales, x, fmt, None)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_strided_and_batched(cuda, fmt):
    wide = _normal(cuda, 9, 640, torch.bfloat16)
    x = wide[:, 64:64 + 288]
    _check_quantized(*ops.fp4_quantize(x, fmt), x, fmt, None)
    y = _normal(cuda, 12, 96, torch.float16).view(3, 4, 96)
    codes, scales = ops.fp4_quantize(y, fmt)
    assert codes.shape == (12, 48)
    _check_quantized(codes, scales, y.view(12, 96), fmt, None)
    for empty in (torch.empty((0, 64), dtype=torch.float16, device=cuda),):
        codes, scales = ops.fp4_quantize(empty, fmt)
        assert codes.shape == (0, 32) and ops.fp4_dequantize(codes, scales, fmt, torch.float16).shape == (0, 64)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("per_row", [1, 3, 8])
def test_quantize_gathered(cuda, fmt, per_row):
    M, K = 21, 800
    x = _normal(cuda, M, K, torch.bfloat16)
    g = torch.Generator().manual_seed(per_row)
    index = torch.randperm(M * per_row, generator=g).to(torch.int32)
    index[4], index[5], index[6], index[7] = -1, M * per_row, 2 ** 31 - 1, -2 ** 31
    s = _scale(cuda, fmt)
    out = ops.fp4_rows_empty(M * per_row, K, fmt, cuda)
    for t in out:
        t.fill_(77)
    count = torch.tensor([M * per_row - 5], dtype=torch.int32, device=cuda)
    codes, scales = ops.fp4_quantize(x, fmt, scale=s, index=index.to(cuda), per_row=per_row, count=count, out=out)
    live = torch.ones(M * per_row, dtype=torch.bool)
    live[4:8] = False
    live[-5:] = False
    src = x[(index.long()[live] // per_row).to(cuda)]
    _check_quantized(codes[live.to(cuda)], scales[:, live.to(cuda)], src, fmt, s)
    assert bool((codes[~live.to(cuda)] == 77).all()) and bool((scales[:, ~live.to(cuda)] == 77).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_by_an_empty_index(cuda, fmt):
    x = _normal(cuda, 5, 96, torch.float16)
    index = torch.zeros(4, dtype=torch.int32, device=cuda)
    for empty in (torch.empty(0, dtype=torch.int32, device=cuda), index[4:]):
        for kw in ({}, {"per_row": 3, "count": index[:1]}):
            codes, scales = ops.fp4_quantize(x, fmt, index=empty, **kw)
            assert codes.shape == (0, 48) and scales.shape[1:] == (0, 16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("count", [-3, 0, 1, 6, 9, 100])
def test_quantize_up_to_a_count_on_the_device(cuda, fmt, count):
    x = _normal(cuda, 9, 96, torch.float16)
    out = ops.fp4_rows_empty(9, 96, fmt, cuda)
    for t in out:
        t.fill_(77)
    codes, scales = ops.fp4_quantize(x, fmt, count=torch.tensor([count], dtype=torch.int32, device=cuda), out=out)
    n = min(max(count, 0), 9)
    _check_quantized(codes[:n], scales[:, :n], x[:n], fmt, None)
    assert bool((codes[n:] == 77).all()) and bool((scales[:, n:] == 77).all())


# ---------------------------------------------------------------- norm
@pytest.mark.parametrize("M,K", [(1, 32), (1, 4096), (5, 96), (3, 544), (64, 2048), (2, 8192), (3, 8224), (2, 16384),
                                 (300, 2880)])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("add", [True, False])
def test_add_rmsnorm(cuda, M, K, fmt, dtype, add):
    x, r = _normal(cuda, M, K, dtype), _normal(cuda, M, K, dtype, seed=5)
    w = (torch.rand(K, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda) + 0.5).to(dtype)
    s = _scale(cuda, fmt, 0.011)
    codes, scales, h = ops.fp4_add_rmsnorm(x, r if add else None, w, 1e-6, fmt, scale=s)
    wide = x.double().cpu() + (r.double().cpu() if add else 0)
    # the fp32 sum of two 16-bit values, rounded to 16 bits
    assert torch.equal(h.cpu(), (x.float() + r.float()).to(dtype).cpu() if add else x.cpu())
    y = wide / (wide.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double().cpu()
    y = y / (1.0 if s is None else float(s))
    d = 2.0 ** -19
    byte = rows_scales(scales, K, fmt)
    most = y.unflatten(-1, (-1, BLOCK[fmt])).abs().amax(-1)
    low, high = block_scales(most * (1 - d), fmt), block_scales(most * (1 + d), fmt)
    assert bool(((byte == low) | (byte == high)).all())
    sv = scale_values(byte, fmt).repeat_interleave(BLOCK[fmt], dim=-1)
    got = _held(codes, scales, fmt)
    q = torch.where(sv > 0, y.abs() / sv, 0.0)
    least, largest = GRID[nearest(q * (1 - d), GRID)] * sv, GRID[nearest(q * (1 + d), GRID)] * sv
    assert bool(((got.abs() >= least) & (got.abs() <= largest)).all())
    assert bool(((got == 0) | (torch.sign(got) == torch.sign(y))).all())


@pytest.mark.parametrize("scale,weight,size", [(1.5 * 2.0 ** 126, 2.0 ** 126, 2.0 ** -6), (2.0 ** -120, 2.0 ** -118, 1.0),
                                               (1.0, 1.0, 1.0)])
def test_add_rmsnorm_scales_near_the_ends_of_fp32(cuda, scale, weight, size):
    """1 / scale is right where a fast fp32 division gives zero. The factor's low half may
    be subnormal here: off by 2^-149 where it is 2^-121, far within the 2^-19 allowed."""
    x = (_normal(cuda, 5, 1024, torch.bfloat16).float() * size).to(torch.bfloat16)
    g = torch.Generator(device=cuda).manual_seed(2)
    w = ((torch.rand(1024, generator=g, device=cuda) + 0.5) * weight).to(torch.bfloat16)
    codes, scales, _ = ops.fp4_add_rmsnorm(x, None, w, 1e-9, "nvfp4", scale=torch.full((1,), scale, device=cuda))
    wide = x.double().cpu()
    y = wide / (wide.pow(2).mean(-1, keepdim=True) + 1e-9).sqrt() * w.double().cpu() / scale
    d = 2.0 ** -19
    byte = rows_scales(scales, 1024, "nvfp4")
    most = y.unflatten(-1, (-1, 16)).abs().amax(-1)
    low, high = block_scales(most * (1 - d), "nvfp4"), block_scales(most * (1 + d), "nvfp4")
    assert bool(((byte == low) | (byte == high)).all()) and bool((byte > 0).all())
    sv = scale_values(byte, "nvfp4").repeat_interleave(16, dim=-1)
    got, q = _held(codes, scales, "nvfp4").abs(), y.abs() / sv
    assert bool(((got >= GRID[nearest(q * (1 - d), GRID)] * sv) & (got <= GRID[nearest(q * (1 + d), GRID)] * sv)).all())


@pytest.mark.parametrize("power,eps", [(-126, 0.0), (-100, 0.0), (-100, 2.0 ** -190), (-60, 2.0 ** -110), (-40, 0.0),
                                       (58, 1e-6), (63, 1e-6), (66, 1e-6), (100, 1e-6), (120, 0.0)])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K", [96, 2048, 16384])
def test_add_rmsnorm_of_very_large_and_small_rows(cuda, K, fmt, power, eps):
    """Squares past both ends of fp32, beside an ordinary row: the formula's values."""
    x = _normal(cuda, 3, K, torch.bfloat16)
    x[1:] = (x[1:].double() * 2.0 ** power).to(torch.bfloat16)
    r = torch.zeros_like(x)
    r[1] = (_normal(cuda, 1, K, torch.bfloat16, seed=5)[0].double() * 2.0 ** power).to(torch.bfloat16)
    w = (torch.rand(K, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda) + 0.5).to(torch.bfloat16)
    s = _scale(cuda, fmt, 0.011)
    codes, scales, h = ops.fp4_add_rmsnorm(x, r, w, eps, fmt, scale=s)
    assert bool(torch.isfinite(h).all())
    eps = float(torch.tensor(eps, dtype=torch.float32))  # as the call takes it: 2^-190 is 0 there
    wide = x.double().cpu() + r.double().cpu()
    y = wide / (wide.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu() / (1.0 if s is None else float(s))
    d = 2.0 ** -19
    byte = rows_scales(scales, K, fmt)
    most = y.unflatten(-1, (-1, BLOCK[fmt])).abs().amax(-1)
    low, high = block_scales(most * (1 - d), fmt), block_scales(most * (1 + d), fmt)
    assert bool(((byte == low) | (byte == high)).all())
    sv = scale_values(byte, fmt).repeat_interleave(BLOCK[fmt], dim=-1)
    got, q = _held(codes, scales, fmt).abs(), torch.where(sv > 0, y.abs() / sv, 0.0)
    assert bool(((got >= GRID[nearest(q * (1 - d), GRID)] * sv) & (got <= GRID[nearest(q * (1 + d), GRID)] * sv)).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_add_rmsnorm_of_a_row_with_an_infinity(cuda, dtype, fmt):
    """Over an infinite root mean square everything finite is 0 and an infinity is NaN, in
    its block only; a NaN makes its whole row NaN."""
    K = 544
    x = _normal(cuda, 3, K, dtype)
    x[0, 40], x[1, 100] = float("inf"), float("nan")
    codes, scales, _ = ops.fp4_add_rmsnorm(x, None, torch.ones(K, dtype=dtype, device=cuda), 1e-6, fmt)
    got = _held(codes, scales, fmt)
    block = torch.arange(K) // BLOCK[fmt] == 40 // BLOCK[fmt]
    assert bool(torch.isnan(got[0, block]).all()) and not got[0, ~block].any()
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isfinite(got[2]).all())


def test_add_rmsnorm_in_place_and_strided(cuda):
    x, r = _normal(cuda, 7, 512, torch.bfloat16)[:, :288], _normal(cuda, 7, 640, torch.bfloat16)[:, 64:352]
    w = torch.ones(288, dtype=torch.bfloat16, device=cuda)
    want = ops.fp4_add_rmsnorm(x, r, w, 1e-5, "mxfp4")
    got = ops.fp4_add_rmsnorm(x, r, w, 1e-5, "mxfp4", residual_out=r)
    assert got[2].data_ptr() == r.data_ptr()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- products
def _weight(cuda, E, N, K, fmt, seed=0):
    g = torch.Generator().manual_seed(seed + N + K)
    w = torch.randn((E, N, K), generator=g) * K ** -0.5
    if fmt == "nvfp4":
        scale = (torch.rand(E, generator=g) + 0.5) * 2.0 ** -9
        values, byte = quantize_ref(over_scale(w, scale[:, None, None]), fmt)
    else:
        scale = None
        values, byte = quantize_ref(w, fmt)
    codes = pack(values, byte, fmt)
    return codes.to(cuda), byte, values, None if scale is None else scale.to(cuda)


def _rows(cuda, M, K, fmt, seed=0):
    x = _normal(cuda, M, K, torch.float16, seed)
    s = _scale(cuda, fmt)
    codes, scales = ops.fp4_quantize(x, fmt, scale=s)
    return codes, scales, s, _held(codes, scales, fmt)


def _product(cuda, M, K, N, fmt, dtype, silu=False, bias=False, ldo=0, seed=0):
    codes, scales, xs, x = _rows(cuda, M, K, fmt, seed)
    w, byte, wv, ws = _weight(cuda, 1, N, K, fmt, seed)
    b = torch.randn(N, generator=torch.Generator().manual_seed(9)).to(dtype) if bias else None
    n_out = N // 2 if silu else N
    out = torch.full((M, n_out + ldo), 3.0, dtype=dtype, device=cuda)
    got = ops.fp4_gemm(codes, scales, w[0], ops.fp4_lay_out_scales(byte[0], fmt).to(cuda), fmt, dtype, x_scale=xs,
                       w_scale=ws, bias=None if b is None else b.to(cuda), silu_mul=silu, out=out[:, :n_out])
    y, bound = product_ref(x, wv[0], xs, ws, b, silu)
    assert ops.device_error() == 0
    assert within(got.cpu(), y, bound, dtype) <= 0
    assert bool((out[:, n_out:] == 3).all())
    return got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,N", [(1, 256, 128), (1, 32, 8), (16, 512, 128), (3, 64, 16), (2, 96, 24), (17, 288, 136),
                                   (64, 1024, 264), (65, 768, 520), (33, 2080, 128), (128, 544, 384), (200, 512, 640),
                                   (7, 4128, 1000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gemm(cuda, M, K, N, fmt, dtype):
    _product(cuda, M, K, N, fmt, dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,N", [(1, 256, 128), (5, 96, 16), (70, 800, 272), (33, 512, 48)])
@pytest.mark.parametrize("silu,bias", [(True, False), (False, True), (True, True)])
def test_gemm_epilogues(cuda, M, K, N, fmt, silu, bias):
    _product(cuda, M, K, N, fmt, torch.bfloat16, silu, bias, ldo=8)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 5, 31, 33, 64, 65, 100, 230, 333, 449])
@pytest.mark.parametrize("K,N,silu", [(1056, 264, False), (4128, 136, False), (8192, 400, True), (2304, 16, True)])
def test_gemm_shared_k(cuda, M, K, N, silu, fmt):
    """Few tiles and a long K, which several CTAs then share."""
    got = _product(cuda, M, K, N, fmt, torch.bfloat16, silu, bias=True, ldo=8)
    assert torch.equal(got, _product(cuda, M, K, N, fmt, torch.bfloat16, silu, bias=True, ldo=8))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("silu,bias,dtype", [(False, True, torch.bfloat16), (True, False, torch.float16)])
@pytest.mark.parametrize("M,K,N", [(65, 2304, 3712), (100, 4128, 3600), (40, 1056, 5008), (33, 8192, 9488), (209, 800, 2608),
                                   (333, 2080, 2320), (208, 512, 2400), (416, 1312, 1936), (1000, 32, 1200),
                                   (417, 96, 1040)])
def test_gemm_many_rows(cuda, M, K, N, fmt, silu, bias, dtype):
    """The kernel of CTA pairs at odd sizes, K whole and shared by two or four pairs."""
    codes, scales, xs, x = _rows(cuda, M, K, fmt)
    w, byte, wv, ws = _weight(cuda, 1, N, K, fmt)
    b = torch.randn(N, generator=torch.Generator().manual_seed(9)).to(dtype).to(cuda) if bias else None
    n_out = N // 2 if silu else N
    out = torch.full((M + 1, n_out + 8), 3.0, dtype=dtype, device=cuda)
    laid = ops.fp4_lay_out_scales(byte[0], fmt).to(cuda)
    got = ops.fp4_gemm(codes, scales, w[0], laid, fmt, dtype, x_scale=xs, w_scale=ws, bias=b, silu_mul=silu,
                       out=out[:M, :n_out])
    y, bound = product_ref(x.to(cuda), wv[0].to(cuda), xs, ws, b, silu)
    assert ops.device_error() == 0
    assert within(got, y, bound, dtype) <= 0
    assert bool((out[M] == 3).all()) and bool((out[:, n_out:] == 3).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,N", [(128, 2048, 28672), (450, 1536, 9000), (9, 4096, 28672), (2000, 800, 2056)])
def test_gemm_many_tiles_over_and_over(cuda, M, K, N, fmt):
    """Several tiles to a CTA, back to back without waiting between: the same bits each time,
    right on columns spread over the tiles."""
    codes, scales, xs, x = _rows(cuda, M, K, fmt)
    g = torch.Generator(device=cuda).manual_seed(3)
    w = torch.randint(0, 256, (N, K // 2), generator=g, device=cuda, dtype=torch.uint8)
    byte = torch.randint(40 if fmt == "nvfp4" else 118, 60 if fmt == "nvfp4" else 122, (N, K // BLOCK[fmt]), generator=g,
                         device=cuda, dtype=torch.uint8)
    laid = ops.fp4_lay_out_scales(byte, fmt)
    y = [ops.fp4_gemm(codes, scales, w, laid, fmt, torch.bfloat16, x_scale=xs) for _ in range(30)]
    assert ops.device_error() == 0
    assert all(torch.equal(t, y[0]) for t in y[1:])
    at = torch.arange(7, N, 97)
    want, bound = product_ref(x, values_ref(w[at.to(cuda)], byte[at.to(cuda)], fmt), xs)
    assert within(y[0][:, at.to(cuda)].cpu(), want, bound, torch.bfloat16) <= 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,N", [(65, 2304, 3712), (80, 4096, 4096), (100, 2048, 3840), (208, 8192, 2048), (209, 1024, 6000)])
def test_gemm_pairs_share_k_over_and_over(cuda, M, K, N, fmt):
    """K shared by two or four CTA pairs, whose warps have one turn, two or none to sum:
    the same bits each time, right on columns spread over the tiles."""
    codes, scales, xs, x = _rows(cuda, M, K, fmt)
    w, byte, wv, ws = _weight(cuda, 1, N, K, fmt)
    laid = ops.fp4_lay_out_scales(byte[0], fmt).to(cuda)
    first = ops.fp4_gemm(codes, scales, w[0], laid, fmt, torch.bfloat16, x_scale=xs, w_scale=ws)
    for _ in range(50):
        assert torch.equal(ops.fp4_gemm(codes, scales, w[0], laid, fmt, torch.bfloat16, x_scale=xs, w_scale=ws), first)
    assert ops.device_error() == 0
    at = torch.arange(3, N, 37)
    want, bound = product_ref(x, wv[0][at], xs, ws)
    assert within(first[:, at.to(cuda)].cpu(), want, bound, torch.bfloat16) <= 0


@pytest.mark.parametrize("M", [1, 2, 8, 15, 16, 31, 32, 48, 63, 96, 127, 129, 255, 256, 257, 400, 511, 600])
def test_gemm_row_counts(cuda, M):
    _product(cuda, M, 320, 272, "nvfp4", torch.bfloat16)
    _product(cuda, M, 320, 272, "mxfp4", torch.float16, silu=True)


def _grouped(cuda, sizes, K, N, fmt, dtype, silu=False, pad=0, first=0, scatter=False, seed=0, ldo=0):
    E, rows = len(sizes), first + sum(sizes) + pad
    codes, scales, xs, x = _rows(cuda, rows, K, fmt, seed)
    w, byte, wv, ws = _weight(cuda, E, N, K, fmt, seed)
    off = torch.tensor([first] + sizes).cumsum(0).to(torch.int32)
    n_out = N // 2 if silu else N
    out = torch.full((rows, n_out + ldo), 3.0, dtype=dtype, device=cuda)
    g = torch.Generator().manual_seed(rows)
    to = torch.randperm(rows, generator=g).to(torch.int32) if scatter else None
    factor = torch.rand(rows, generator=g) if scatter else None
    got = ops.fp4_grouped_gemm(codes, scales, w, ops.fp4_lay_out_scales(byte, fmt).to(cuda), off.to(cuda), fmt, dtype,
                               x_scale=xs, w_scale=ws, out=out[:, :n_out], silu_mul=silu,
                               row_map=None if to is None else to.to(cuda),
                               row_scale=None if factor is None else factor.to(cuda)).cpu()
    assert ops.device_error() == 0
    left = torch.ones(rows, dtype=torch.bool)
    for e in range(E):
        r = torch.arange(int(off[e]), int(off[e + 1]))
        if not r.numel():
            continue
        y, bound = product_ref(x[r], wv[e], xs, None if ws is None else ws[e], None, silu)
        at = r if to is None else to[r].long()
        if factor is not None:
            f = factor[at].double()[:, None]
            y, bound = y * f, bound * f + 2.0 ** -23 * (y * f).abs()
        assert within(got[at], y, bound, dtype) <= 0
        left[at] = False
    assert bool((out.cpu()[left] == 3).all()) and bool((out[:, n_out:] == 3).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K,N", [(64, 64), (32, 8), (96, 264), (768, 256), (544, 136)])
@pytest.mark.parametrize("sizes", [[1], [0, 0, 5], [1, 0, 127, 128, 129], [300, 1, 0, 2, 257, 0], [16] * 9, [700],
                                   [3, 61, 33, 7, 500, 225, 224, 223]])
def test_grouped(cuda, sizes, K, N, fmt):
    _grouped(cuda, sizes, K, N, fmt, torch.bfloat16, pad=5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("silu,scatter,first", [(True, False, 0), (False, True, 0), (True, False, 3), (False, False, 7),
                                                (True, True, 1)])
@pytest.mark.parametrize("sizes", [[1, 0, 40, 2], [100, 300, 0, 33], [2, 1, 1, 1, 0, 0, 3]])
def test_grouped_epilogues(cuda, sizes, silu, scatter, first, fmt):
    _grouped(cuda, sizes, 288, 272, fmt, torch.float16, silu, pad=9, first=first, scatter=scatter, ldo=8)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("silu,scatter", [(False, True), (True, False)])
@pytest.mark.parametrize("K,sizes", [(2048, [1, 0, 2, 1]), (288, [0, 3, 0, 0]), (1024, [0, 0, 0, 0])])
def test_grouped_few_live_rows_of_a_large_buffer(cuda, K, sizes, silu, scatter, fmt):
    """A rank whose experts got few of the buffer's rows: the kernel for many rows with a few."""
    _grouped(cuda, sizes, K, 272, fmt, torch.bfloat16, silu, pad=500, scatter=scatter)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("sizes", [[1] * 1024, [0] * 1000 + [3] * 24, [100] + [0] * 1023])
def test_grouped_of_a_thousand_experts(cuda, sizes, fmt):
    _grouped(cuda, sizes, 64, 24, fmt, torch.float16, pad=2)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K", [32, 256, 512, 768])
def test_grouped_many_short_tiles(cuda, K, fmt):
    """Dozens of tiles of one to three stages to a CTA pair: tiles that one of the two warps
    that turn scales has nothing to do for. The same bits each time, right on columns spread
    over the tiles."""
    E, N, per = 64, 16384, 50
    codes, scales, xs, x = _rows(cuda, E * per, K, fmt)
    g = torch.Generator(device=cuda).manual_seed(K)
    w = torch.randint(0, 256, (E, N, K // 2), generator=g, device=cuda, dtype=torch.uint8)
    byte = torch.randint(40 if fmt == "nvfp4" else 118, 60 if fmt == "nvfp4" else 122, (E, N, K // BLOCK[fmt]),
                         generator=g, device=cuda, dtype=torch.uint8)
    laid = ops.fp4_lay_out_scales(byte, fmt)
    off = (torch.arange(E + 1, device=cuda) * per).to(torch.int32)
    first = ops.fp4_grouped_gemm(codes, scales, w, laid, off, fmt, torch.bfloat16, x_scale=xs)
    for _ in range(30):
        assert torch.equal(ops.fp4_grouped_gemm(codes, scales, w, laid, off, fmt, torch.bfloat16, x_scale=xs), first)
    assert ops.device_error() == 0
    at = torch.arange(7, N, 397, device=cuda)
    for e in range(E):
        rows = slice(e * per, (e + 1) * per)
        want, bound = product_ref(x[rows], values_ref(w[e][at], byte[e][at], fmt), xs)
        assert within(first[rows][:, at].cpu(), want, bound, torch.bfloat16) <= 0


@pytest.mark.parametrize("sizes", [[3, 0, 5], [90, 120]])
def test_grouped_rows_that_map_nowhere(cuda, sizes):
    """Rows whose place is outside out are dropped, and so is what offsets say past the rows."""
    rows, K, N = sum(sizes), 128, 136
    codes, scales, xs, x = _rows(cuda, rows, K, "nvfp4")
    w, byte, wv, ws = _weight(cuda, len(sizes), N, K, "nvfp4")
    to = torch.arange(rows, dtype=torch.int32).flip(0)
    to[1], to[2], to[rows - 1] = -1, 2 ** 31 - 1, rows + 4
    off = torch.tensor([0] + sizes).cumsum(0).to(torch.int32)
    off[-1] += 1000
    out = torch.full((rows + 4, N), 3.0, dtype=torch.bfloat16, device=cuda)
    factor = torch.rand(rows + 4, generator=torch.Generator().manual_seed(4))
    got = ops.fp4_grouped_gemm(codes, scales, w, ops.fp4_lay_out_scales(byte, "nvfp4").to(cuda), off.to(cuda), "nvfp4",
                               torch.bfloat16, x_scale=xs, w_scale=ws, out=out, row_map=to.to(cuda),
                               row_scale=factor.to(cuda)).cpu()
    left = torch.ones(rows + 4, dtype=torch.bool)
    for e in range(len(sizes)):
        for r in range(int(off[e]), min(int(off[e + 1]), rows)):
            at = int(to[r])
            if not 0 <= at < rows + 4:
                continue
            y, bound = product_ref(x[r:r + 1], wv[e], xs, ws[e])
            f = float(factor[at])
            assert within(got[at:at + 1], y * f, bound * f + 2.0 ** -23 * (y * f).abs(), torch.bfloat16) <= 0
            left[at] = False
    assert bool((got[left] == 3).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_nan_in_rows_and_weights_stays_visible(cuda, fmt):
    """A block that holds a NaN or an infinity makes its row of the product NaN, and only it."""
    x = _normal(cuda, 5, 320, torch.bfloat16)
    x[1, 300] = float("nan")
    x[3, 7] = float("inf")
    codes, scales = ops.fp4_quantize(x, fmt)
    w, byte, _, ws = _weight(cuda, 1, 136, 320, fmt)
    y = ops.fp4_gemm(codes, scales, w[0], ops.fp4_lay_out_scales(byte[0], fmt).to(cuda), fmt, torch.bfloat16)
    bad = torch.tensor([False, True, False, True, False])
    assert bool(torch.isnan(y[bad.to(cuda)]).all()) and bool(torch.isfinite(y[~bad.to(cuda)]).all())
    byte = byte.clone()
    byte[0, 130, 2] = 127 if fmt == "nvfp4" else 255
    y = ops.fp4_gemm(codes, scales, w[0], ops.fp4_lay_out_scales(byte[0], fmt).to(cuda), fmt, torch.bfloat16)
    assert bool(torch.isnan(y[:, 130]).all()) and bool(torch.isfinite(y[0, :130]).all())
