"""MXFP4: quantisation, dequantisation, the fp32 matvec and the block-scaled product against a float64 restatement of
the format, and their refusals."""
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from conftest import ROOT
from oracle import mxfp4_np as mx

gpu = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def layout(codes, scales):
    return dev(codes), dev(mx.tile_scales(scales))


# ---- the restatement itself and what needs no GPU ----


def test_digits_of_the_oracle_points():
    codes, scales = mx.quantize(np.array([[0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25, -5.01, 4.0] + [0.0] * 20]))
    assert scales[0, 0] == 127                            # the largest value lies in [4, 8): the factor is 1
    nib = np.stack([codes & 15, codes >> 4], axis=-1).reshape(-1)
    assert list(nib[:12]) == [0, 0, 2, 2, 4, 4, 6, 6, 7, 8, 15, 6]   # ties to the even code, 7.9 saturates


def test_scale_bytes(ffi, ops):
    L = ffi.lib()
    for rows, nb in ((0, 5), (5, 0), (1, 1), (128, 4), (129, 5), (1 << 20, 1024)):
        want = -(-rows // 128) * (-(-nb // 4)) * 512
        assert L.axc_cuda_mxfp4_scale_bytes(rows, nb) == want == ops.mxfp4_scale_bytes(rows, nb)


def test_c_entries_refuse_before_any_launch(ffi):
    L, bad = ffi.lib(), ffi.AXC_ERR_INVALID_ARGUMENT
    f32, bf16, i64 = ffi.AXC_TY_F32, ffi.AXC_TY_BF16, ffi.AXC_TY_I64
    assert L.axc_cuda_mxfp4_quantize(16, ffi.AXC_TY_U8, 32, 1, 32, 32, 48, None) == bad
    assert L.axc_cuda_mxfp4_quantize(None, f32, 32, 1, 32, 32, 48, None) == bad
    assert L.axc_cuda_mxfp4_quantize(18, f32, 32, 1, 32, 32, 48, None) == bad            # x not aligned to its elements
    assert L.axc_cuda_mxfp4_quantize(16, f32, 32, 1, 32, 40, 48, None) == bad            # codes not 16-byte aligned
    assert L.axc_cuda_mxfp4_quantize(16, f32, 31, 2, 32, 32, 48, None) == bad            # rows overlap
    assert "row stride" in ffi.last_error_detail()
    assert L.axc_cuda_mxfp4_quantize(None, f32, 0, 0, 32, None, None, None) == ffi.AXC_OK
    assert L.axc_cuda_mxfp4_dequant(16, 32, 48, i64, 1, 1, None) == bad
    assert L.axc_cuda_mxfp4_dequant(16, 40, 48, f32, 1, 1, None) == bad
    assert L.axc_cuda_mxfp4_matvec(16, 32, 48, 64, 9, 1, 1, None, None) == bad
    assert "1..8 tokens" in ffi.last_error_detail()
    assert L.axc_cuda_mxfp4_matvec(16, 32, 48, 66, 1, 1, 1, None, None) == bad
    assert L.axc_cuda_mxfp4_matvec(16, 32, None, 64, 1, 1, 1, None, None) == bad
    assert L.axc_cuda_mxfp4_matvec(16, 32, 48, 64, 1, 1 << 31, 1, None, None) == bad
    assert L.axc_cuda_mxfp4_matvec(None, None, None, None, 0, 5, 5, None, None) == ffi.AXC_OK
    assert L.axc_cuda_mxfp4_prefill(16, 32, 48, 64, 80, i64, 1, 1, 1, None, None) == bad
    assert L.axc_cuda_mxfp4_prefill(16, 32, 48, 66, 80, bf16, 1, 1, 1, None, None) == bad
    assert L.axc_cuda_mxfp4_prefill(16, 32, 48, 64, 81, bf16, 1, 1, 1, None, None) == bad
    assert L.axc_cuda_mxfp4_prefill(16, 32, 48, 64, 80, bf16, 1 << 24, 1, 1, None, None) == bad
    assert L.axc_cuda_mxfp4_prefill(None, None, None, None, None, bf16, 0, 1, 1, None, None) == ffi.AXC_OK


def test_python_entries_refuse_cpu_tensors(ops):
    z = torch.zeros(1024, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.mxfp4_quantize(torch.zeros(4, 32))
    with pytest.raises(ValueError, match="CUDA"):
        ops.mxfp4_matvec(z, z, torch.zeros(32), 1, 1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.mxfp4_prefill(z, z, z, z, 1, 1, 1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.mxfp4_dequant(z, z, 1, 1)


@gpu
def test_python_entries_refuse_what_does_not_fit(ops):
    codes, scales = ops.mxfp4_quantize(torch.randn(130, 96, device="cuda"))
    x = torch.randn(2, 96, device="cuda")
    with pytest.raises(ValueError, match="scales has"):
        ops.mxfp4_matvec(codes, scales[:-1], x, 130, 3, m_tokens=2)
    with pytest.raises(ValueError, match="codes has"):
        ops.mxfp4_matvec(codes, scales, x, 131, 3, m_tokens=2)
    with pytest.raises(ValueError, match="x has"):
        ops.mxfp4_matvec(codes, scales, x, 130, 3, m_tokens=3)
    with pytest.raises(ValueError, match="m_tokens"):
        ops.mxfp4_matvec(codes, scales, x, 130, 3, m_tokens=0)
    with pytest.raises(Exception, match="1..8 tokens"):
        ops.mxfp4_matvec(codes, scales, torch.randn(9, 96, device="cuda"), 130, 3, m_tokens=9)
    with pytest.raises(ValueError, match="y has"):
        ops.mxfp4_matvec(codes, scales, x, 130, 3, m_tokens=2, y=torch.empty(259, device="cuda"))
    with pytest.raises(ValueError, match="out_dtype"):
        ops.mxfp4_dequant(codes, scales, 130, 3, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="last dimension"):
        ops.mxfp4_quantize(torch.randn(96, 130, device="cuda").t())
    with pytest.raises(ValueError, match="overlap"):
        ops.mxfp4_quantize(torch.randn(1, 64, device="cuda").expand(4, 64))
    with pytest.raises(ValueError, match="dimensions"):
        ops.mxfp4_quantize(torch.randn(2, 2, 32, device="cuda"))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        ops.mxfp4_quantize(torch.zeros(2, 32, dtype=torch.float64, device="cuda"))


# ---- quantisation ----


def spread_rows(rows, cols, rng):
    """Normal values times row factors from 2^-20 to 2^20 and column factors up to 16, some zeros."""
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-20, 21, (rows, 1))) * np.exp2(rng.integers(0, 5, (1, cols)))
    x[rng.random((rows, cols)) < 0.02] = 0.0
    return x


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 256), (127, 100), (128, 128), (129, 4097), (300, 1000),
                                       (1, 14336)])
def test_quantise_has_the_bytes_of_the_definition(ops, rows, cols, dtype):
    x = torch.from_numpy(spread_rows(rows, cols, np.random.default_rng(rows * 7 + cols))).clamp(-6e4, 6e4).to(dtype)
    codes, scales = ops.mxfp4_quantize(x.cuda())
    want_codes, want_scales = mx.quantize(x.double().numpy())
    assert np.array_equal(codes.cpu().numpy(), want_codes)
    assert np.array_equal(scales.cpu().numpy(), mx.tile_scales(want_scales))   # the bytes that fill up tiles are zero
    w = ops.mxfp4_dequant(codes, scales, rows, want_scales.shape[1])
    assert np.array_equal(w.cpu().numpy().astype(np.float64), mx.values(want_codes, want_scales))


@gpu
def test_quantise_ties_extremes_and_non_finite_blocks(ops):
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99], np.float32)
    x = np.zeros((10, 64), np.float32)
    x[0, :10], x[0, 10:20], x[0, 20] = ties, -ties, 4.0
    x[1, :10], x[1, 10:20], x[1, 20] = np.nextafter(ties, 0), np.nextafter(ties, 9), 4.0
    x[2, 0] = np.finfo(np.float32).max
    x[3, 0], x[3, 1] = np.finfo(np.float32).smallest_subnormal, -np.finfo(np.float32).smallest_subnormal
    x[4, :32] = np.float32(2.0 ** -126) * np.arange(32, dtype=np.float32) / 31       # scale at its lower end
    x[5, 3] = np.nan
    x[6, 40], x[6, 41] = np.inf, 1.0
    x[7, :] = -0.0
    x[8, 0], x[8, 33] = -np.inf, 3.0
    x[9, :4] = np.float32(2.0 ** -125) * np.array([1, 3, 5.5, 7.99])
    codes, scales = ops.mxfp4_quantize(dev(x))
    want_codes, want_scales = mx.quantize(x)
    assert np.array_equal(codes.cpu().numpy(), want_codes) and np.array_equal(scales.cpu().numpy(), mx.tile_scales(want_scales))
    w = ops.mxfp4_dequant(codes, scales, 10, 2).cpu().numpy()
    ref = mx.values(want_codes, want_scales)
    assert np.array_equal(np.isnan(w), np.isnan(ref)) and np.isnan(w[5, :32]).all() and not np.isnan(w[5, 32:]).any()
    assert np.array_equal(w[~np.isnan(ref)].astype(np.float64), ref[~np.isnan(ref)])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,stride", [(0, 200), (1, 200), (8, 208), (3, 131), (0, 100)])
def test_quantise_of_strided_rows(ops, dtype, offset, stride):
    """A slice of a wider buffer: any start and any row distance, with wide loads or without."""
    buf = torch.from_numpy(spread_rows(1, 40 * stride + 16, np.random.default_rng(3)))[0].to(dtype).cuda()
    x = buf.as_strided((40, 100), (stride, 1), offset)
    codes, scales = ops.mxfp4_quantize(x)
    again = ops.mxfp4_quantize(x.clone(memory_format=torch.contiguous_format))
    assert torch.equal(codes, again[0]) and torch.equal(scales, again[1])
    assert np.array_equal(codes.cpu().numpy(), mx.quantize(x.double().cpu().numpy())[0])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dequant_rounds_once_and_covers_every_scale(ops, dtype):
    scales = np.arange(256, dtype=np.uint8).reshape(64, 4)
    codes = np.tile(np.arange(256, dtype=np.uint8), 16).reshape(64, 64)
    w = ops.mxfp4_dequant(*layout(codes, scales), 64, 4, out_dtype=dtype).cpu()
    with np.errstate(over="ignore"):
        ref = torch.from_numpy(mx.values(codes, scales).astype(np.float32)).to(dtype)   # exact in fp32, or infinite
    assert torch.equal(torch.isnan(w), torch.isnan(ref))
    assert torch.equal(torch.nan_to_num(w, nan=0.0), torch.nan_to_num(ref, nan=0.0))


@gpu
def test_quantise_into_the_callers_buffers_leaves_the_rest(ops):
    x = torch.randn(5, 70, device="cuda")
    n = 5 * 3 * 16
    codes = torch.full((n + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    scales = torch.full((512 + 64,), 0xCD, dtype=torch.uint8, device="cuda")
    ops.mxfp4_quantize(x, codes=codes, scales=scales)
    want = ops.mxfp4_quantize(x)
    assert torch.equal(codes[:n], want[0].view(-1)) and torch.equal(scales[:512], want[1])
    assert bool((codes[n:] == 0xAB).all()) and bool((scales[512:] == 0xCD).all())


# ---- products ----


def chain_bound(blocks):
    """Relative to sum |a w|: every product is exact; a chain of MMAs of 64 columns truncates the running sum once per
    MMA, and inside an MMA the addends are aligned to the largest and truncated: two times 2^-23 per step; the sums of
    the parts are a few roundings of 2^-24 more."""
    return (2 * ((blocks + 1) // 2) + 8) * 2.0 ** -23


def check_prefill(ops, m, n, nb, dtype, seed, low=118, high=124):
    rng = np.random.default_rng(seed)
    w_codes, w_scales, w_tiles, w = mx.random_matrix(n, nb, rng, low, high)
    a_codes, a_scales, a_tiles, a = mx.random_matrix(m, nb, rng, low, high)
    st = ops.new_status()
    c = ops.mxfp4_prefill(dev(w_codes), dev(w_tiles), dev(a_codes), dev(a_tiles), m, n, nb, out_dtype=dtype, status=st)
    assert c.shape == (m, n) and c.dtype == dtype and int(st.item()) == 0
    ref, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    got = c.double().cpu().numpy()
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    assert (np.abs(got - ref) <= chain_bound(nb) * mag * (1 + half) + half * np.abs(ref)).all()
    return c


@gpu
@pytest.mark.parametrize("m,n,nb", [(1, 1, 1), (1, 128, 2), (5, 300, 7), (16, 128, 8), (17, 130, 3), (37, 513, 33), (64, 96, 128),
                                    (128, 128, 16), (256, 256, 8), (257, 129, 9), (300, 200, 4), (513, 384, 11), (600, 640, 5),
                                    (520, 3000, 6), (1000, 2310, 10), (80, 19200, 5), (128, 700, 40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_prefill_matches_float64(ops, m, n, nb, dtype):
    check_prefill(ops, m, n, nb, dtype, m * 1000 + n + nb)


@gpu
@pytest.mark.parametrize("m,n,nb", [(3, 200, 448), (40, 128, 300), (130, 257, 897), (300, 512, 129)])
def test_prefill_long_rows_and_scales_far_apart(ops, m, n, nb):
    check_prefill(ops, m, n, nb, torch.float32, m + n + nb, low=112, high=136)


@gpu
@pytest.mark.parametrize("m,n", [(4, 200), (300, 300)])
def test_prefill_nan_scale_reaches_its_row_only(ops, m, n):
    rng = np.random.default_rng(5)
    w_codes, w_scales, _t, w = mx.random_matrix(n, 5, rng)
    a_codes, a_scales, _t, a = mx.random_matrix(m, 5, rng)
    w_scales[130, 2] = 255
    a_scales[m - 1, 4] = 255
    c = ops.mxfp4_prefill(*layout(w_codes, w_scales), *layout(a_codes, a_scales), m, n, 5).cpu().numpy()
    want = np.zeros((m, n), bool)
    want[m - 1, :] = want[:, 130] = True
    assert np.array_equal(np.isnan(c), want)


@gpu
def test_prefill_writes_only_its_rows(ops):
    m, n, nb = 5, 130, 3
    rng = np.random.default_rng(6)
    w, a = mx.random_matrix(n, nb, rng), mx.random_matrix(m, nb, rng)
    c = torch.full((m * n + 256,), 7.0, device="cuda")
    ops.mxfp4_prefill(dev(w[0]), dev(w[2]), dev(a[0]), dev(a[2]), m, n, nb, c=c)
    assert bool((c[m * n:] == 7.0).all())
    assert torch.equal(c[:m * n].view(m, n), ops.mxfp4_prefill(dev(w[0]), dev(w[2]), dev(a[0]), dev(a[2]), m, n, nb))


def check_matvec(ops, m, rows, nb, seed, x=None, low=118, high=124):
    rng = np.random.default_rng(seed)
    codes, _s, tiles, w = mx.random_matrix(rows, nb, rng, low, high)
    if x is None:
        x = (rng.standard_normal((m, nb * 32)) * np.exp2(rng.integers(-8, 9, (m, 1)))).astype(np.float32)
        x[:, rng.random(nb * 32) < 0.01] *= 12
    st = ops.new_status()
    y = ops.mxfp4_matvec(dev(codes), dev(tiles), dev(x), rows, nb, m_tokens=m, status=st)
    assert int(st.item()) == 0
    x64 = x.astype(np.float64)
    ref, mag = x64 @ w.T, np.abs(x64) @ np.abs(w).T
    # x in a block is a multiple of a unit of at most 2^-21 of the block's largest |x|, rounded to nearest; the digits
    # of an integer X sum to at most 4 |X| + 4 in magnitude, and each digit's column is summed as in chain_bound
    top = np.repeat(np.abs(x64).reshape(m, nb, 32).max(axis=2), 32, axis=1)
    fixed = 2.0 ** -22 * (top @ np.abs(w).T)
    err = np.abs(y.double().cpu().numpy().reshape(m, rows) - ref)
    assert (err <= fixed + chain_bound(nb) * (4 * mag + 8 * fixed)).all(), (err / np.maximum(mag, 1e-300)).max()
    return y


@gpu
@pytest.mark.parametrize("m", [1, 2, 3, 8])
@pytest.mark.parametrize("rows,nb", [(1, 1), (7, 3), (128, 8), (129, 9), (300, 33), (1000, 128), (20000, 5), (16, 448)])
def test_matvec_matches_float64(ops, m, rows, nb):
    check_matvec(ops, m, rows, nb, m * 100000 + rows + nb)


@gpu
@pytest.mark.parametrize("m,rows,nb", [(1, 200, 897), (5, 64, 1400), (8, 300, 260), (7, 150, 512)])
def test_matvec_long_rows_and_scales_far_apart(ops, m, rows, nb):
    check_matvec(ops, m, rows, nb, m + rows + nb, low=112, high=136)


@gpu
def test_matvec_is_norm_wise_as_close_as_fp32(ops):
    """Normal x: the fixed point and the sums together stay below 1e-6 of the result's norm."""
    rng = np.random.default_rng(11)
    codes, _s, tiles, w = mx.random_matrix(2048, 128, rng)
    x = rng.standard_normal((1, 4096)).astype(np.float32)
    y = ops.mxfp4_matvec(dev(codes), dev(tiles), dev(x), 2048, 128).double().cpu().numpy()
    ref = (x.astype(np.float64) @ w.T).reshape(y.shape)
    assert np.linalg.norm(y - ref) <= 1e-6 * np.linalg.norm(ref)


@gpu
def test_matvec_every_digit_pattern(ops):
    """x = integers of up to 22 bits against the identity: comes back exactly."""
    nb, rows = 4, 128
    codes = np.zeros((rows, nb * 16), np.uint8)
    for r in range(rows):
        codes[r, r // 2] = 2 << (4 * (r % 2))             # the value 1 at column r
    rng = np.random.default_rng(12)
    x = rng.integers(-(1 << 22), (1 << 22) + 1, (8, 128)).astype(np.float32)
    x[0, :8] = [0, 1, -1, 4, -4, 1 << 22, -(1 << 22), 0o4444444]
    x[:, ::32] = 1 << 22                                   # every block has the same unit: 1/2 or 1
    y = ops.mxfp4_matvec(*layout(codes, np.full((rows, nb), 127, np.uint8)), dev(x), rows, nb, m_tokens=8)
    assert np.abs(y.cpu().numpy().astype(np.float64) - x).max() <= 1.0   # 2^22 is the lower end of its binade: unit 2
    y = ops.mxfp4_matvec(*layout(codes, np.full((rows, nb), 127, np.uint8)), dev(np.clip(x, 1 - (1 << 22), (1 << 22) - 1)),
                         rows, nb, m_tokens=8)
    assert np.array_equal(y.cpu().numpy(), np.clip(x, 1 - (1 << 22), (1 << 22) - 1))


@gpu
@pytest.mark.parametrize("power", [-149, -126, -106, -100, 0, 100, 126])
def test_matvec_magnitudes_of_x(ops, power):
    nb, rows = 2, 40
    rng = np.random.default_rng(13)
    codes, _s, tiles, w = mx.random_matrix(rows, nb, rng, 116, 118)
    with np.errstate(under="ignore"):
        x = (rng.uniform(0.5, 0.99, (1, 64)) * np.exp2(float(power) + 1)).astype(np.float32)
    y = ops.mxfp4_matvec(dev(codes), dev(tiles), dev(x), rows, nb).double().cpu().numpy().reshape(-1)
    x64 = x.astype(np.float64)
    unit = max(2.0 ** -21 * np.abs(x64).max(), 2.0 ** -127)
    fixed = unit / 2 * np.abs(w).sum(axis=1)
    mag = (np.abs(w) @ np.abs(x64).T)[:, 0]
    small = 64 * 2.0 ** -126                              # sums below the smallest normal number may be flushed
    assert (np.abs(y - (w @ x64.T)[:, 0]) <= fixed + chain_bound(nb) * (4 * mag + 8 * fixed) + small).all()


@gpu
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 3e38])
def test_matvec_non_finite_x_makes_its_token_nan(ops, value):
    rng = np.random.default_rng(14)
    codes, _s, tiles, _w = mx.random_matrix(50, 9, rng)
    x = rng.standard_normal((3, 288)).astype(np.float32)
    clean = ops.mxfp4_matvec(dev(codes), dev(tiles), dev(x), 50, 9, m_tokens=3)
    x[1, 100] = value
    y = ops.mxfp4_matvec(dev(codes), dev(tiles), dev(x), 50, 9, m_tokens=3)
    assert bool(torch.isnan(y[1]).all()) and torch.equal(y[0], clean[0]) and torch.equal(y[2], clean[2])


@gpu
def test_matvec_nan_weights_reach_their_row_only(ops):
    rng = np.random.default_rng(17)
    codes, scales, _t, _w = mx.random_matrix(300, 9, rng)
    scales[200, 4] = 255
    y = ops.mxfp4_matvec(*layout(codes, scales), torch.randn(2, 288, device="cuda"), 300, 9, m_tokens=2).cpu().numpy()
    want = np.zeros((2, 300), bool)
    want[:, 200] = True
    assert np.array_equal(np.isnan(y), want)


@gpu
def test_a_range_of_rows_is_a_matrix(ops):
    """From a multiple of 128 on, rows can be used by themselves (a shard of a matrix)."""
    codes, scales, w = large_operands(ops, 500, 20, 5)
    x = torch.randn(640, device="cuda")
    whole = ops.mxfp4_matvec(codes, scales, x, 500, 20)
    part = ops.mxfp4_matvec(codes[256:], scales[2 * 5 * 512:], x, 244, 20)
    assert bool(((part - whole[256:]).abs() <= chain_bound(20) * 8 * (w.float().abs() @ x.abs())[256:]).all())
    assert torch.equal(ops.mxfp4_dequant(codes[128:], scales[5 * 512:], 372, 20).double(), w[128:])


@gpu
def test_sizes_beyond_four_gigabytes(ops):
    """x, codes and the product pass 2^32 bytes, x and the product 2^32 elements too."""
    rows, nb, m = 1_060_000, 256, 4100
    ends = torch.cat([torch.arange(300), torch.arange(rows - 300, rows)]).cuda()
    x = torch.zeros(rows, nb * 32, dtype=torch.bfloat16, device="cuda")
    x[ends] = torch.randn(600, nb * 32, device="cuda").to(torch.bfloat16)
    codes, scales = ops.mxfp4_quantize(x)
    few = ops.mxfp4_quantize(x[ends])
    del x
    w = ops.mxfp4_dequant(*few, 600, nb)
    assert torch.equal(codes[ends], few[0])
    assert torch.equal(ops.mxfp4_embed(codes, scales, ends, rows, nb), w)
    a_codes, a_scales = ops.mxfp4_quantize(torch.randn(m, nb * 32, device="cuda"))
    a = ops.mxfp4_dequant(a_codes, a_scales, m, nb)[-300:].double()
    half = torch.finfo(torch.bfloat16).eps / 2
    for tokens in (m, 100):                               # many and few tokens
        operand = (a_codes, a_scales) if tokens == m else ops.mxfp4_quantize(a[-tokens:].float())
        c = ops.mxfp4_prefill(codes, scales, *operand, tokens, rows, nb, out_dtype=torch.bfloat16)
        last = min(tokens, 300)
        ref, mag = a[-last:] @ w.double().t(), a[-last:].abs() @ w.double().abs().t()
        assert bool(((c[-last:, ends].double() - ref).abs() <= chain_bound(nb) * mag * (1 + half) + half * ref.abs()).all())
        assert bool((c[-last:, 300:rows - 300] == 0).all())
        del c


@gpu
def test_calls_from_several_threads(ops):
    codes, scales, w = large_operands(ops, 2000, 64, 6)
    x = torch.randn(300, 2048, device="cuda")
    a_codes, a_scales = ops.mxfp4_quantize(x)
    want = (ops.mxfp4_matvec(codes, scales, x[:4], 2000, 64, m_tokens=4),
            ops.mxfp4_prefill(codes, scales, a_codes, a_scales, 300, 2000, 64),
            ops.mxfp4_prefill(codes, scales, a_codes, a_scales, 30, 2000, 64))
    torch.cuda.synchronize()

    def work(_):
        with torch.cuda.stream(torch.cuda.Stream()):
            good = True
            for _i in range(20):
                c, s = ops.mxfp4_quantize(x)
                got = (ops.mxfp4_matvec(codes, scales, x[:4], 2000, 64, m_tokens=4),
                       ops.mxfp4_prefill(codes, scales, c, s, 300, 2000, 64),
                       ops.mxfp4_prefill(codes, scales, c, s, 30, 2000, 64))
                torch.cuda.current_stream().synchronize()
                good = good and all(torch.equal(g, e) for g, e in zip(got, want))
            return good

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))


@gpu
def test_zero_sizes(ops):
    st = ops.new_status()
    e = torch.empty(0, dtype=torch.uint8, device="cuda")
    assert ops.mxfp4_quantize(torch.empty(0, 64, device="cuda"))[0].shape == (0, 32)
    assert ops.mxfp4_quantize(torch.empty(3, 0, device="cuda"))[0].shape == (3, 0)
    assert ops.mxfp4_dequant(e, e, 4, 0).shape == (4, 0)
    y = ops.mxfp4_matvec(e, e, torch.empty(0, device="cuda"), 5, 0, y=torch.full((5,), 3.0, device="cuda"), status=st)
    assert bool((y == 0).all())
    c = ops.mxfp4_prefill(e, e, e, e, 3, 5, 0, c=torch.full((3, 5), 3.0, device="cuda"), status=st)
    assert bool((c == 0).all())
    assert ops.mxfp4_matvec(e, e, torch.zeros(32, device="cuda"), 0, 1).shape == (0,)
    assert ops.mxfp4_prefill(torch.zeros(5 * 48, dtype=torch.uint8, device="cuda"), torch.zeros(512, dtype=torch.uint8, device="cuda"),
                             e, e, 0, 5, 3).shape == (0, 5)
    assert int(st.item()) == 0


def large_operands(ops, rows, nb, seed, spread=0.02):
    """A matrix quantised on the device and its values (exact in fp32) as float64."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes, scales = ops.mxfp4_quantize(torch.randn(rows, nb * 32, generator=g, device="cuda") * spread)
    return codes, scales, ops.mxfp4_dequant(codes, scales, rows, nb).double()


@gpu
@pytest.mark.parametrize("rows,nb", [(1100, 600), (9000, 200), (4096, 128), (14336, 40), (40000, 16), (700, 1000), (129, 2100),
                                     (20000, 30), (1024, 25), (1024, 24)])
def test_matvec_over_the_forms_of_the_kernel(ops, rows, nb):
    """One and two row tiles, 1 to 8 CTAs per row, rings that wrap, every number of tokens."""
    codes, scales, w = large_operands(ops, rows, nb, rows + nb)
    x = torch.randn(8, nb * 32, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    x64 = x.double()
    ref, mag = x64 @ w.t(), x64.abs() @ w.abs().t()
    top = x64.abs().view(8, nb, 32).amax(dim=2).repeat_interleave(32, dim=1)
    fixed = 2.0 ** -22 * (top @ w.abs().t())
    all8 = ops.mxfp4_matvec(codes, scales, x, rows, nb, m_tokens=8)
    assert bool(((all8.double() - ref).abs() <= fixed + chain_bound(nb) * (4 * mag + 8 * fixed)).all())
    for m in range(1, 8):                                 # the same bits whatever other tokens the call serves
        st = ops.new_status()
        assert torch.equal(ops.mxfp4_matvec(codes, scales, x[8 - m:], rows, nb, m_tokens=m, status=st), all8[8 - m:]), m
        assert int(st.item()) == 0


@gpu
@pytest.mark.parametrize("rows,nb", [(300, 32), (300, 100), (1024, 128), (2048, 64), (2048, 128), (2048, 256), (3500, 448),
                                     (4096, 64), (4096, 448), (5120, 64), (18900, 24), (19000, 32), (40000, 24)])
def test_matvec_where_the_split_of_the_work_changes(ops, rows, nb):
    """One and two row tiles on either side of the rules that choose them: right, and the same bits for every number of
    tokens."""
    codes, scales, w = large_operands(ops, rows, nb, rows + nb)
    x = torch.randn(8, nb * 32, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    x64 = x.double()
    top = x64.abs().view(8, nb, 32).amax(dim=2).repeat_interleave(32, dim=1)
    fixed, mag = 2.0 ** -22 * (top @ w.abs().t()), x64.abs() @ w.abs().t()
    st = ops.new_status()
    all8 = ops.mxfp4_matvec(codes, scales, x, rows, nb, m_tokens=8, status=st)
    assert bool(((all8.double() - x64 @ w.t()).abs() <= fixed + chain_bound(nb) * (4 * mag + 8 * fixed)).all())
    for m in (1, 2, 3, 4, 5):
        assert torch.equal(ops.mxfp4_matvec(codes, scales, x[:m], rows, nb, m_tokens=m, status=st).view(m, rows), all8[:m]), m
    assert int(st.item()) == 0


@gpu
@pytest.mark.parametrize("m,n,nb", [(129, 4096, 128), (160, 300, 130), (200, 1000, 448), (257, 2100, 256), (300, 4500, 127), (513, 260, 130),
                                    (640, 900, 200), (1000, 129, 300), (2000, 128, 128), (4096, 100, 140), (130, 9400, 128), (130, 9500, 128)])
def test_prefill_of_rows_split_over_the_sms(ops, m, n, nb):
    """More than 128 tokens and few rows: on either side of the rule that splits K, and nothing beyond the output."""
    w_codes, w_scales, w = large_operands(ops, n, nb, n + nb)
    a_codes, a_scales, a = large_operands(ops, m, nb, m + nb, 3.0)
    st = ops.new_status()
    out = torch.full((m * n + 300,), 7.0, device="cuda")
    ops.mxfp4_prefill(w_codes, w_scales, a_codes, a_scales, m, n, nb, c=out, status=st)
    c = out[:m * n].view(m, n)
    assert int(st.item()) == 0 and bool((out[m * n:] == 7.0).all())
    assert bool(((c.double() - a @ w.t()).abs() <= chain_bound(nb) * (a.abs() @ w.abs().t())).all())
    for dtype in (torch.bfloat16, torch.float16):         # the same sums, rounded once
        assert torch.equal(ops.mxfp4_prefill(w_codes, w_scales, a_codes, a_scales, m, n, nb, out_dtype=dtype), c.to(dtype))


@gpu
@pytest.mark.parametrize("m,n,nb", [(40, 1100, 600), (64, 9000, 200), (33, 25000, 16), (64, 20000, 50), (100, 3000, 300), (128, 1000, 900),
                                    (128, 19500, 20), (65, 9600, 40), (129, 4000, 130), (1000, 5000, 100), (2048, 9500, 24),
                                    (3, 60000, 9)])
def test_prefill_over_the_forms_of_the_kernels(ops, m, n, nb):
    w_codes, w_scales, w = large_operands(ops, n, nb, n + nb)
    a_codes, a_scales, a = large_operands(ops, m, nb, m + nb, 3.0)
    st = ops.new_status()
    c = ops.mxfp4_prefill(w_codes, w_scales, a_codes, a_scales, m, n, nb, status=st)
    assert int(st.item()) == 0
    assert bool(((c.double() - a @ w.t()).abs() <= chain_bound(nb) * (a.abs() @ w.abs().t())).all())
    for dtype in (torch.bfloat16, torch.float16):         # the same sums, rounded once
        assert torch.equal(ops.mxfp4_prefill(w_codes, w_scales, a_codes, a_scales, m, n, nb, out_dtype=dtype), c.to(dtype))


@gpu
def test_first_call_may_be_captured():
    """In a process that has not used the library yet, every call goes into a graph at once."""
    code = """
import importlib, torch
ops = importlib.import_module("axiom-compute_b200.ops")
x = torch.randn(300, 640, device="cuda"); w = torch.randn(1100, 640, device="cuda"); ids = torch.arange(5, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    wc, ws = ops.mxfp4_quantize(w)
    xc, xs = ops.mxfp4_quantize(x)
    c = ops.mxfp4_prefill(wc, ws, xc, xs, 300, 1100, 20)
    few = ops.mxfp4_prefill(wc, ws, xc, xs, 40, 1100, 20)
    y = ops.mxfp4_matvec(wc, ws, x[:3], 1100, 20, m_tokens=3)
    e = ops.mxfp4_embed(wc, ws, ids, 1100, 20)
    v = ops.mxfp4_dequant(wc, ws, 1100, 20)
g.replay(); torch.cuda.synchronize()
assert torch.equal(e, v[:5]) and torch.equal(few, ops.mxfp4_prefill(wc, ws, xc, xs, 40, 1100, 20))
assert torch.equal(c, ops.mxfp4_prefill(wc, ws, xc, xs, 300, 1100, 20))
assert torch.equal(y, ops.mxfp4_matvec(wc, ws, x[:3], 1100, 20, m_tokens=3))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@gpu
def test_results_do_not_change_from_run_to_run(ops):
    rng = np.random.default_rng(15)
    w, a = mx.random_matrix(2000, 100, rng, 110, 135), mx.random_matrix(300, 100, rng, 110, 135)
    wd, ws, ad, as_ = dev(w[0]), dev(w[2]), dev(a[0]), dev(a[2])
    x = torch.randn(8, 3200, device="cuda")
    c, y = ops.mxfp4_prefill(wd, ws, ad, as_, 300, 2000, 100), ops.mxfp4_matvec(wd, ws, x, 2000, 100, m_tokens=8)
    for _ in range(5):
        assert torch.equal(ops.mxfp4_prefill(wd, ws, ad, as_, 300, 2000, 100), c)
        assert torch.equal(ops.mxfp4_matvec(wd, ws, x, 2000, 100, m_tokens=8), y)


@gpu
def test_quantise_then_product_in_one_stream_and_in_a_graph(ops):
    """Weights and tokens quantised right before the products that read them, back to back and without waits, on a side
    stream and replayed from a graph with new inputs."""
    w, x = torch.randn(1000, 640, device="cuda"), torch.randn(40, 640, device="cuda")

    def step():
        wc, ws = ops.mxfp4_quantize(w)
        xc, xs = ops.mxfp4_quantize(x)
        c = ops.mxfp4_prefill(wc, ws, xc, xs, 40, 1000, 20)
        y = ops.mxfp4_matvec(wc, ws, x[:3], 1000, 20, m_tokens=3)
        return c, y, ops.mxfp4_dequant(wc, ws, 1000, 20), ops.mxfp4_dequant(xc, xs, 40, 20)

    def check(c, y, wv, xv):
        torch.cuda.synchronize()
        ref = xv.double() @ wv.double().t()
        mag = xv.double().abs() @ wv.double().abs().t()
        assert bool(((c.double() - ref).abs() <= chain_bound(20) * mag).all())
        ref = x[:3].double() @ wv.double().t()
        mag = x[:3].double().abs().max() * wv.double().abs().sum(dim=1)
        assert bool(((y.double() - ref).abs() <= (2.0 ** -22 + 12 * chain_bound(20)) * mag).all())

    check(*step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            out = step()
    check(*out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        w.copy_(torch.randn(w.shape, device="cuda") * seed), x.copy_(torch.randn(x.shape, device="cuda"))
        graph.replay()
        check(*out)


@gpu
def test_two_streams_at_once(ops):
    rng = np.random.default_rng(16)
    w, a = mx.random_matrix(4096, 128, rng), mx.random_matrix(300, 128, rng)
    wd, ws, ad, as_ = dev(w[0]), dev(w[2]), dev(a[0]), dev(a[2])
    x = torch.randn(8, 4096, device="cuda")
    c, y = ops.mxfp4_prefill(wd, ws, ad, as_, 300, 4096, 128), ops.mxfp4_matvec(wd, ws, x, 4096, 128, m_tokens=8)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            got.append(("c", ops.mxfp4_prefill(wd, ws, ad, as_, 300, 4096, 128)))
        with torch.cuda.stream(s2):
            got.append(("y", ops.mxfp4_matvec(wd, ws, x, 4096, 128, m_tokens=8)))
    torch.cuda.synchronize()
    assert all(torch.equal(v, c if k == "c" else y) for k, v in got)


# ---- the ends of the ranges, with results that are normal numbers ----


def pick_columns(rows, blocks, byte):
    """Codes and scale bytes of a matrix whose row r is 2^(byte - 127) at column r and zero elsewhere."""
    codes = np.zeros((rows, blocks * 16), np.uint8)
    r = np.arange(rows)
    codes[r, r // 2] = 2 << (4 * (r % 2))
    return codes, np.full((rows, blocks), byte, np.uint8)


def held(x):
    """x as the matvec holds it: per block of 32 columns a whole number of units of 2^(floor(log2 max |x|) - 21), at
    least 2^-127, ties to even.  The unit is a power of two, so the division is exact in float64."""
    v = x.astype(np.float64).reshape(x.shape[0], -1, 32)
    top = np.abs(v).max(axis=2, keepdims=True)
    _m, e = np.frexp(np.where(top == 0, 1.0, top))
    unit = np.maximum(np.exp2(np.where(top == 0, -127.0, e - 22.0)), 2.0 ** -127)
    return (np.rint(v / unit) * unit).reshape(x.shape)


@gpu
@pytest.mark.parametrize("rows,nb,byte", [(128, 4, 147), (128, 5, 254), (300, 64, 150), (2048, 64, 160), (2048, 900, 147)])
def test_matvec_holds_x_to_its_block_unit(ops, rows, nb, byte):
    """Each y is one value of x times a power of two, a normal number that the sums hold exactly: tiny and subnormal
    blocks beside ordinary ones, blocks on either side of 2^-105, and blocks with one value that dwarfs the others."""
    rng = np.random.default_rng(rows + nb + byte)
    up = 40 if byte == 254 else 126                       # 2^127 times the largest result stays finite
    kinds = [(-149, -149), (-149, -126), (-149, -106), (-127, -105), (-106, -104), (-20, 0), (-1, up - 40)]
    if byte == 254:
        kinds = kinds[:5] + [(-120, -100), (-60, -20)]
    x = np.zeros((8, nb, 32))
    for t in range(8):
        for b in range(nb):
            low, high = kinds[(b + t) % len(kinds)]
            x[t, b] = rng.uniform(-1, 1, 32) * np.exp2(rng.uniform(low, high, 32))
            x[t, b, rng.integers(32)] = np.exp2(float(high)) * (1.0 if (b + t) % 2 else 0.999)
    with np.errstate(under="ignore"):
        x = x.reshape(8, nb * 32).astype(np.float32)
    codes, tiles = layout(*pick_columns(rows, nb, byte))
    want = held(x)[:, :rows] * 2.0 ** (byte - 127)
    assert (np.abs(want[want != 0]) >= 2.0 ** -126).all() and np.abs(want).max() < 2.0 ** 127
    for m in (1, 3, 8):
        y = ops.mxfp4_matvec(codes, tiles, dev(x[:m]), rows, nb, m_tokens=m).double().cpu().numpy().reshape(m, rows)
        assert np.array_equal(y, want[:m]), (m, np.argwhere(y != want[:m])[:5])


@gpu
@pytest.mark.parametrize("power", [-128, -127, -118, -110, -106])
def test_matvec_of_tiny_x_keeps_the_unit(ops, power):
    """Sums over whole rows of blocks below 2^-105: the error is half a unit of 2^-127 per column, with a result that an
    answer of zero would miss (every product is positive)."""
    rng = np.random.default_rng(21 - power)
    nb, rows = 6, 200
    codes, scales, _t, w = mx.random_matrix(rows, nb, rng, 150, 152)
    codes &= 0x77
    codes |= 0x22                                         # magnitudes of at least 1
    w = mx.values(codes, scales)
    x = (rng.uniform(0.6, 0.99, (2, nb * 32)) * np.exp2(float(power) + 1)).astype(np.float32)
    y = ops.mxfp4_matvec(*layout(codes, scales), dev(x), rows, nb, m_tokens=2).double().cpu().numpy()
    x64 = x.astype(np.float64)
    ref, fixed = x64 @ w.T, 2.0 ** -128 * np.abs(w).sum(axis=1)
    assert (ref > 1.2 * fixed + chain_bound(nb) * (4 * ref + 8 * fixed)).all()   # so zeros fail
    assert (np.abs(y - ref) <= fixed + chain_bound(nb) * (4 * ref + 8 * fixed)).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dequant_and_lookup_overflow_to_infinity(ops, dtype):
    """Values beyond the output type's range are infinite, not its largest number; every scale byte, every code."""
    scales = np.arange(256, dtype=np.uint8).reshape(64, 4)
    codes = np.tile(np.arange(256, dtype=np.uint8), 16).reshape(64, 64)
    w = ops.mxfp4_dequant(*layout(codes, scales), 64, 4, out_dtype=dtype).cpu()
    with np.errstate(over="ignore"):
        ref = torch.from_numpy(mx.values(codes, scales).astype(np.float32)).to(dtype)
    ok = ~torch.isnan(ref)
    assert torch.equal(torch.isnan(w), ~ok) and torch.equal(w[ok], ref[ok]) and bool(torch.isinf(ref).any())
    assert torch.equal(torch.signbit(w[ok]), torch.signbit(ref[ok]))
    ids = torch.arange(63, -1, -1, device="cuda")
    e = ops.mxfp4_embed(*layout(codes, scales), ids, 64, 4, out_dtype=dtype).cpu().flip(0)
    assert torch.equal(torch.isnan(e), ~ok) and torch.equal(e[ok], ref[ok])


@gpu
@pytest.mark.parametrize("m,n,nb", [(5, 130, 3), (40, 300, 40), (300, 600, 5), (200, 300, 130)])
def test_prefill_overflows_to_infinity(ops, m, n, nb):
    """Sums beyond fp16 are infinite with the sum's sign, in every form of the product."""
    rng = np.random.default_rng(m + n)
    w, a = mx.random_matrix(n, nb, rng, 130, 134), mx.random_matrix(m, nb, rng, 130, 134)
    args = (dev(w[0]), dev(w[2]), dev(a[0]), dev(a[2]), m, n, nb)
    c = ops.mxfp4_prefill(*args)
    half = ops.mxfp4_prefill(*args, out_dtype=torch.float16)
    assert bool((c.abs() > 65520).any()) and bool((c.abs() < 65504).any())
    assert torch.equal(half, c.to(torch.float16)) and bool(torch.isinf(half).any())


def test_the_limit_of_tokens_is_one_number(ffi, ops):
    """The header's, the binding's and the kernel's limit of the matvec agree (the C entry names the kernel's)."""
    with open(f"{ROOT}/include/axc_cuda.h") as f:
        assert f"#define AXC_MXFP4_MATVEC_TOKENS {ops.MX_MATVEC_TOKENS}\n" in f.read()
    n = ffi.AXC_MXFP4_MATVEC_TOKENS + 1
    assert ffi.lib().axc_cuda_mxfp4_matvec(16, 32, 48, 64, n, 1, 1, None, None) == ffi.AXC_ERR_INVALID_ARGUMENT
    assert f"1..{ops.MX_MATVEC_TOKENS} tokens" in ffi.last_error_detail()
