"""Device-layer entry points on torch CUDA tensors (weights and activations resident in HBM).

torch is used for device memory and streams only; every function forwards raw device pointers
and the current stream to ``libaxc_cuda.so``.  No function here computes anything itself and
none has a CPU path: a non-CUDA tensor is an error.  Nothing is recorded for a backward pass:
outputs do not require gradients, whatever the inputs do.

Kernels report through `status` (``new_status``) only: bit 0 says that a bounded wait inside the
kernel ran out and the output is not complete.  A call without `status` does not report it.
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import Optional

import torch

from . import _ffi
from .runtime import _raise_for

Q4K_SB_BYTES, Q4K_SB_ELEMS = 144, 256
Q4_0_BLK_BYTES, Q4_0_BLK_ELEMS = 18, 32


def _stream_ptr() -> int:
    return int(torch.cuda.current_stream().cuda_stream)


def _chk(t: torch.Tensor, dtype, name: str, min_elems: int) -> int:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this backend has no CPU path)")
    if t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype}")
    if t.numel() < min_elems:
        raise ValueError(f"{name} has {t.numel()} elements, needs >= {min_elems}")
    return t.data_ptr()


def make_tuning(ctas_per_sm: int = 0, tile_rows: int = 0, stages: int = 0, threads: int = 0,
                evict_first: int = -1, pdl: int = 2, resident: int = 0) -> _ffi.AxcTuning:
    return _ffi.AxcTuning(ctas_per_sm, tile_rows, stages, threads, evict_first, pdl, resident)


def new_status(device=None) -> torch.Tensor:
    """Device word that receives kernel error bits (0 = clean)."""
    return torch.zeros(1, dtype=torch.int32, device=device or "cuda")


def _matvec(fn_name, blk_bytes, blk_elems, q, x, rows, n, y, status, tuning):
    qp = _chk(q, torch.uint8, "q", rows * n * blk_bytes)
    xp = _chk(x, torch.float32, "x", n * blk_elems)
    if y is None:
        y = torch.empty(rows, dtype=torch.float32, device=q.device)
    yp = _chk(y, torch.float32, "y", rows)
    sp = _chk(status, torch.int32, "status", 1) if status is not None else None
    with torch.cuda.device(q.device):
        rc = getattr(_ffi.lib(), fn_name)(qp, xp, yp, rows, n, _stream_ptr(), sp,
                                          C.byref(tuning) if tuning is not None else None)
    _raise_for(rc)
    return y


def q4k_matvec(q: torch.Tensor, x: torch.Tensor, rows: int, n_superblocks: int,
               y: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None,
               tuning: Optional[_ffi.AxcTuning] = None) -> torch.Tensor:
    """y[r] = q4km_dequant_matvec(q row r, x): ``rows`` reference calls
    (examples/q4km_dequant_matvec.axc) in one launch."""
    return _matvec("axc_cuda_q4k_matvec", Q4K_SB_BYTES, Q4K_SB_ELEMS, q, x, rows, n_superblocks,
                   y, status, tuning)


def q4_0_matvec(q: torch.Tensor, x: torch.Tensor, rows: int, n_blocks: int,
                y: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None,
                tuning: Optional[_ffi.AxcTuning] = None) -> torch.Tensor:
    """y[r] = q4_0_dequant_matvec(q row r, x) (examples/q4_0_dequant_matvec.axc)."""
    return _matvec("axc_cuda_q4_0_matvec", Q4_0_BLK_BYTES, Q4_0_BLK_ELEMS, q, x, rows, n_blocks,
                   y, status, tuning)


def _matvec_seq(fn_name, blk_bytes, blk_elems, q, x, rows, n, y):
    qp = _chk(q, torch.uint8, "q", rows * n * blk_bytes)
    xp = _chk(x, torch.float32, "x", n * blk_elems)
    if y is None:
        y = torch.empty(rows, dtype=torch.float32, device=q.device)
    yp = _chk(y, torch.float32, "y", rows)
    with torch.cuda.device(q.device):
        rc = getattr(_ffi.lib(), fn_name)(qp, xp, yp, rows, n, _stream_ptr())
    _raise_for(rc)
    return y


def q4k_matvec_seq(q, x, rows: int, n_superblocks: int, y=None) -> torch.Tensor:
    """Reference operation order; y is bit-identical to ``q4km_dequant_matvec_cpu``."""
    return _matvec_seq("axc_cuda_q4k_matvec_seq", Q4K_SB_BYTES, Q4K_SB_ELEMS, q, x, rows,
                       n_superblocks, y)


def q4_0_matvec_seq(q, x, rows: int, n_blocks: int, y=None) -> torch.Tensor:
    """Reference operation order; y is bit-identical to ``q4_0_dequant_matvec_cpu``."""
    return _matvec_seq("axc_cuda_q4_0_matvec_seq", Q4_0_BLK_BYTES, Q4_0_BLK_ELEMS, q, x, rows,
                       n_blocks, y)


def _dequant(fn_name, blk_bytes, blk_elems, q, rows, n):
    qp = _chk(q, torch.uint8, "q", rows * n * blk_bytes)
    w = torch.empty((rows, n * blk_elems), dtype=torch.float32, device=q.device)
    with torch.cuda.device(q.device):
        rc = getattr(_ffi.lib(), fn_name)(qp, w.data_ptr(), rows, n, _stream_ptr())
    _raise_for(rc)
    return w


def q4k_dequant(q: torch.Tensor, rows: int, n_superblocks: int) -> torch.Tensor:
    """Bit-exact dequantised weights, shape (rows, n_superblocks * 256)."""
    return _dequant("axc_cuda_q4k_dequant", Q4K_SB_BYTES, Q4K_SB_ELEMS, q, rows, n_superblocks)


def q4_0_dequant(q: torch.Tensor, rows: int, n_blocks: int) -> torch.Tensor:
    """Bit-exact dequantised weights, shape (rows, n_blocks * 32)."""
    return _dequant("axc_cuda_q4_0_dequant", Q4_0_BLK_BYTES, Q4_0_BLK_ELEMS, q, rows, n_blocks)


def q4k_matvec_plan(rows: int, n_superblocks: int, tuning=None, sm_count: int = 148) -> dict:
    """Launch geometry the Q4_K_M matvec would use (no GPU needed)."""
    out = (C.c_int32 * 5)()
    rc = _ffi.lib().axc_cuda_q4k_matvec_plan(rows, n_superblocks,
                                             C.byref(tuning) if tuning is not None else None,
                                             sm_count, out)
    _raise_for(rc)
    return {"grid": out[0], "block": out[1], "smem": out[2], "tile_rows": out[3], "stages": out[4]}


def q4k_prefill(q: torch.Tensor, a_bf16: torch.Tensor, m_tokens: int, n_rows: int, n_superblocks: int,
                c: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None, form: int = 0,
                independent: bool = False) -> torch.Tensor:
    """C[m, n] = sum_k A[m, k] * bf16(W[n, k]) on the tensor cores (tcgen05); A is a bf16 tensor of
    shape (m_tokens, n_superblocks * 256), the result fp32 of shape (m_tokens, n_rows).  `form`:
    0 = the library's choice, 1 = one CTA per tile, 2 = a CTA pair per 256 rows.  `independent`: q and a
    are not written and c not touched by the launch directly before (lets the call overlap it)."""
    qp = _chk(q, torch.uint8, "q", n_rows * n_superblocks * Q4K_SB_BYTES)
    ap = _chk(a_bf16, torch.bfloat16, "a", m_tokens * n_superblocks * Q4K_SB_ELEMS)
    if c is None:
        c = torch.empty((m_tokens, n_rows), dtype=torch.float32, device=q.device)
    cp = _chk(c, torch.float32, "c", m_tokens * n_rows)
    with torch.cuda.device(q.device):
        rc = _ffi.lib().axc_cuda_q4k_prefill_form(qp, ap, cp, m_tokens, n_rows, n_superblocks, _stream_ptr(),
                                                  status.data_ptr() if status is not None else None, int(form),
                                                  1 if independent else 0)
    _raise_for(rc)
    return c


# ---- MXFP4 and rows of quantised tables ----

MX_BLOCK_BYTES, MX_BLOCK_ELEMS = 16, 32
MX_MATVEC_TOKENS = _ffi.AXC_MXFP4_MATVEC_TOKENS
_FLOAT_TYPES = {torch.float32: _ffi.AXC_TY_F32, torch.bfloat16: _ffi.AXC_TY_BF16, torch.float16: _ffi.AXC_TY_F16}
_ID_TYPES = {torch.int32: _ffi.AXC_TY_I32, torch.int64: _ffi.AXC_TY_I64}


def _float_type(dtype, name: str) -> int:
    code = _FLOAT_TYPES.get(dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16")
    return code


def _count(value, name: str, least: int = 0) -> int:
    if type(value) is int and least <= value < 0x80000000:
        return value
    value = operator.index(value)
    if not least <= value < 0x80000000:
        raise ValueError(f"{name} must be in [{least}, 2^31), got {value}")
    return value


_current_device = getattr(torch._C, "_cuda_getDevice", None)          # what torch.cuda.current_device() and
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)    # current_stream(i).cuda_stream read


def _lib():
    return _ffi._lib or _ffi.lib()


def _ptr(t: torch.Tensor, dtype, name: str, min_elems: int, device: int) -> int:
    """``_chk``, and on CUDA device `device`.  (A small call is bound by the host: the checks that pass are kept to a
    few attribute reads.)"""
    if t.dtype is dtype and t.get_device() == device and t.is_contiguous() and t.numel() >= min_elems:
        return t.data_ptr()
    _chk(t, dtype, name, min_elems)      # says what is wrong
    raise ValueError(f"{name} is on {t.device}, the first operand on cuda:{device}")


def _device_of(t: torch.Tensor, name: str) -> int:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this backend has no CPU path)")
    return t.get_device()


def _call(device: int, fn, *args) -> None:
    """fn(*args) with CUDA device `device` current; a status other than OK raises."""
    if device == _current_device():
        rc = fn(*args)
    else:
        with torch.cuda.device(device):
            rc = fn(*args)
    if rc:
        _raise_for(rc)


def _status_ptr(status: torch.Tensor, device: int) -> int:
    return _ptr(status, torch.int32, "status", 1, device)


def mxfp4_scale_bytes(rows: int, n_blocks: int) -> int:
    """Bytes of the scale tiles of an MXFP4 matrix (tiles of 128 rows x 4 blocks; the address of each byte is in
    include/axc_cuda.h).  ``mxfp4_quantize`` writes all of them.  Whoever fills such a buffer otherwise sets the bytes
    that belong to no row and block to zero: no call checks them, and a NaN scale there reaches the products."""
    return _tile_bytes(_count(rows, "rows"), _count(n_blocks, "n_blocks"))


def _tile_bytes(rows: int, n_blocks: int) -> int:
    return (rows + 127) // 128 * ((n_blocks + 3) // 4) * 512


def _codes_ptr(codes, rows: int, n_blocks: int, device: int, name: str = "codes") -> int:
    return _ptr(codes, torch.uint8, name, rows * n_blocks * MX_BLOCK_BYTES, device)


def _scales_ptr(scales, rows: int, n_blocks: int, device: int, name: str = "scales") -> int:
    return _ptr(scales, torch.uint8, name, _tile_bytes(rows, n_blocks), device)


def mxfp4_quantize(x: torch.Tensor, codes: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None):
    """Rows of a float32, bfloat16 or float16 tensor to MXFP4: returns (codes, scales), uint8 tensors of
    rows x ceil(cols / 32) * 16 bytes and of ``mxfp4_scale_bytes`` (layout: include/axc_cuda.h).  x has shape
    (rows, cols) or (cols,); its last dimension is contiguous, rows may be any stride apart."""
    device = _device_of(x, "x")
    xt = _float_type(x.dtype, "x")
    shape, strides = x.shape, x.stride()
    if len(shape) == 2:
        rows, cols = shape
        stride = strides[0] if rows > 1 else cols
    elif len(shape) == 1:
        rows, cols = 1, shape[0]
        stride = cols
    else:
        raise ValueError(f"x must have one or two dimensions, got {x.dim()}")
    if cols > 1 and strides[-1] != 1:
        raise ValueError("the last dimension of x must be contiguous")
    if stride < cols:
        raise ValueError("the rows of x overlap")
    _count(rows, "rows"), _count(cols, "cols")
    n_blocks = (cols + 31) // 32
    if codes is None:
        codes = torch.empty(rows, n_blocks * MX_BLOCK_BYTES, dtype=torch.uint8, device=x.device)
        cp = codes.data_ptr()
    else:
        cp = _codes_ptr(codes, rows, n_blocks, device)
    if scales is None:
        scales = torch.empty(_tile_bytes(rows, n_blocks), dtype=torch.uint8, device=x.device)
        sp = scales.data_ptr()
    else:
        sp = _scales_ptr(scales, rows, n_blocks, device)
    _call(device, _lib().axc_cuda_mxfp4_quantize, x.data_ptr(), xt, stride, rows, cols, cp, sp, _raw_stream(device))
    return codes, scales


def mxfp4_dequant(codes: torch.Tensor, scales: torch.Tensor, rows: int, n_blocks: int,
                  out_dtype: torch.dtype = torch.float32, w: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values of an MXFP4 matrix, shape (rows, n_blocks * 32): exact in float32, rounded to nearest even in
    bfloat16 / float16."""
    device = _device_of(codes, "codes")
    rows, n_blocks = _count(rows, "rows"), _count(n_blocks, "n_blocks")
    cp, sp = _codes_ptr(codes, rows, n_blocks, device), _scales_ptr(scales, rows, n_blocks, device)
    wt = _float_type(out_dtype, "out_dtype")
    if w is None:
        w = torch.empty(rows, n_blocks * MX_BLOCK_ELEMS, dtype=out_dtype, device=codes.device)
        wp = w.data_ptr()
    else:
        wp = _ptr(w, out_dtype, "w", rows * n_blocks * MX_BLOCK_ELEMS, device)
    _call(device, _lib().axc_cuda_mxfp4_dequant, cp, sp, wp, wt, rows, n_blocks, _raw_stream(device))
    return w


def mxfp4_matvec(codes: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, rows: int, n_blocks: int,
                 y: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None, m_tokens: int = 1) -> torch.Tensor:
    """y[t, r] = sum_k W[r, k] x[t, k] with W in MXFP4, for 1 to 8 float32 vectors x of n_blocks * 32 values.  x is held
    in fixed point, 23 bits with sign per block of 32: each value is off by at most 2^-22 of the block's largest |x|, so
    small values beside a very large one lose bits that float32 has.  A block with a NaN, an infinity or a magnitude of
    2^127 or more makes its token NaN.  y has shape (rows,) for one vector, (m_tokens, rows) where x has more
    dimensions than one or there are several."""
    device = _device_of(codes, "codes")
    rows, n_blocks, m_tokens = _count(rows, "rows"), _count(n_blocks, "n_blocks"), _count(m_tokens, "m_tokens", 1)
    cp, sp = _codes_ptr(codes, rows, n_blocks, device), _scales_ptr(scales, rows, n_blocks, device)
    xp = _ptr(x, torch.float32, "x", m_tokens * n_blocks * MX_BLOCK_ELEMS, device)
    if y is None:
        y = torch.empty(rows, dtype=torch.float32, device=x.device) if m_tokens == 1 and x.dim() <= 1 else \
            torch.empty(m_tokens, rows, dtype=torch.float32, device=x.device)
        yp = y.data_ptr()
    else:
        yp = _ptr(y, torch.float32, "y", m_tokens * rows, device)
    _call(device, _lib().axc_cuda_mxfp4_matvec, cp, sp, xp, yp, m_tokens, rows, n_blocks, _raw_stream(device),
          None if status is None else _status_ptr(status, device))
    return y


def mxfp4_prefill(w_codes: torch.Tensor, w_scales: torch.Tensor, a_codes: torch.Tensor, a_scales: torch.Tensor,
                  m_tokens: int, n_rows: int, n_blocks: int, c: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """C[m, n] = sum_k A[m, k] W[n, k] on the tensor cores, both operands in MXFP4 (tokens through
    ``mxfp4_quantize``): C has shape (m_tokens, n_rows) in out_dtype, fp32 accumulation, one rounding.
    The tensor cores' accumulation cuts off where fp32 addition rounds: an error of up to 2^-22 of sum |A W| per 64 columns
    where scales lie far apart (include/axc_cuda.h)."""
    device = _device_of(w_codes, "w_codes")
    m_tokens, n_rows, n_blocks = _count(m_tokens, "m_tokens"), _count(n_rows, "n_rows"), _count(n_blocks, "n_blocks")
    wp, wsp = _codes_ptr(w_codes, n_rows, n_blocks, device, "w_codes"), _scales_ptr(w_scales, n_rows, n_blocks, device, "w_scales")
    ap, asp = _codes_ptr(a_codes, m_tokens, n_blocks, device, "a_codes"), _scales_ptr(a_scales, m_tokens, n_blocks, device, "a_scales")
    ct = _float_type(out_dtype, "out_dtype")
    if c is None:
        c = torch.empty(m_tokens, n_rows, dtype=out_dtype, device=w_codes.device)
        cp = c.data_ptr()
    else:
        cp = _ptr(c, out_dtype, "c", m_tokens * n_rows, device)
    _call(device, _lib().axc_cuda_mxfp4_prefill, wp, wsp, ap, asp, cp, ct, m_tokens, n_rows, n_blocks, _raw_stream(device),
          None if status is None else _status_ptr(status, device))
    return c


def _embed(fn, ptrs, device: int, ids, rows: int, n: int, elems: int, scale, out, out_dtype, status):
    it, ot = _ID_TYPES.get(ids.dtype), _FLOAT_TYPES.get(out_dtype)
    if it is None or not ids.is_cuda or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous int32 or int64 CUDA tensor")
    if ids.get_device() != device:
        raise ValueError(f"ids is on {ids.device}, the first operand on cuda:{device}")
    if ot is None:
        _float_type(out_dtype, "out_dtype")
    n_ids = _count(ids.numel(), "the number of ids")
    if out is None:
        out = torch.empty(*ids.shape, n * elems, dtype=out_dtype, device=ids.device)
        op = out.data_ptr()
    else:
        op = _ptr(out, out_dtype, "out", n_ids * n * elems, device)
    _call(device, fn, *ptrs, ids.data_ptr(), it, n_ids, op, ot, rows, n, scale, _raw_stream(device),
          None if status is None else _status_ptr(status, device))
    return out


def q4k_embed(q: torch.Tensor, ids: torch.Tensor, rows: int, n_superblocks: int, scale: float = 1.0,
              out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32,
              status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[..., :] = dequant(row ids[...] of a Q4_K_M matrix) * scale, rounded once to out_dtype.  An id outside
    [0, rows) gives a row of zeros and sets bit 1 (value 2) of status."""
    device = _device_of(q, "q")
    rows, n = _count(rows, "rows"), _count(n_superblocks, "n_superblocks")
    qp = _ptr(q, torch.uint8, "q", rows * n * Q4K_SB_BYTES, device)
    return _embed(_lib().axc_cuda_q4k_embed, (qp,), device, ids, rows, n, Q4K_SB_ELEMS, scale, out, out_dtype, status)


def q4_0_embed(q: torch.Tensor, ids: torch.Tensor, rows: int, n_blocks: int, scale: float = 1.0,
               out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32,
               status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``q4k_embed`` for a Q4_0 matrix."""
    device = _device_of(q, "q")
    rows, n = _count(rows, "rows"), _count(n_blocks, "n_blocks")
    qp = _ptr(q, torch.uint8, "q", rows * n * Q4_0_BLK_BYTES, device)
    return _embed(_lib().axc_cuda_q4_0_embed, (qp,), device, ids, rows, n, Q4_0_BLK_ELEMS, scale, out, out_dtype, status)


def mxfp4_embed(codes: torch.Tensor, scales: torch.Tensor, ids: torch.Tensor, rows: int, n_blocks: int, scale: float = 1.0,
                out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32,
                status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``q4k_embed`` for an MXFP4 matrix."""
    device = _device_of(codes, "codes")
    rows, n = _count(rows, "rows"), _count(n_blocks, "n_blocks")
    ptrs = _codes_ptr(codes, rows, n, device), _scales_ptr(scales, rows, n, device)
    return _embed(_lib().axc_cuda_mxfp4_embed, ptrs, device, ids, rows, n, MX_BLOCK_ELEMS, scale, out, out_dtype, status)
