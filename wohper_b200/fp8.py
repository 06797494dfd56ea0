"""The Python side of wh_fp8_gemm (``gemm_fp8_e4m3_ue8m0``), imported with torch on
first use."""
from __future__ import annotations

import torch

from . import Context, _check, _ptr, lib
from .kvcache import (_INVALID_POINTER, _INVALID_SHAPE, _UNSUPPORTED, _dense, _dtype_code, _fail,
                      _handle, _int, _on, _on_gpu)


def _rows(x, rows: int, cols: int, what: str) -> int:
    """The stride between the rows of x [rows, cols]."""
    if x.dim() != 2 or x.shape != (rows, cols):
        _fail(_INVALID_SHAPE, f"{what}: {tuple(x.shape)}, not {(rows, cols)}")
    a, b = x.stride()
    if b != 1 and cols > 1:
        _fail(_INVALID_SHAPE, f"{what}: contiguous rows")
    if rows <= 1:  # a size-1 dimension's stride is free
        return cols
    if a < cols:
        _fail(_INVALID_SHAPE, f"{what}: rows that share memory")
    return a


_scratch_sizes: dict = {}


def _scratch_bytes(cols: int, tokens: int) -> int:
    """wh_fp8_gemm_scratch_bytes, asked once for the same sizes."""
    size = _scratch_sizes.get((cols, tokens))
    if size is None:
        if len(_scratch_sizes) >= 256:
            _scratch_sizes.clear()
        size = _scratch_sizes[cols, tokens] = int(lib().wh_fp8_gemm_scratch_bytes(cols, tokens))
    return size


def gemm_fp8_e4m3_ue8m0(ctx: Context, weight, scale, x, act_quant_block: int = 64, out_dtype=None,
                        out=None, scratch=None, stream=None):
    """The product of many tokens on the tensor cores (wh_fp8_gemm): weight uint8
    [rows, cols] (E4M3; cols % 16 == 0) and scale uint8 [ceil(rows / 128),
    ceil(cols / 128)] (UE8M0), both dense; x [tokens, cols] f32, bf16 or f16, whose
    rows may lie apart (on 16 bytes).  x is quantised to E4M3 per act_quant_block
    (32, 64 or 128) values of a row, as fp8_act_quant_dequant_in_place does.
    Returns out [tokens, rows] of out_dtype (by default x's), f32 sums: those of the
    GEMV in another order.  out may not overlap an input; its rows may lie apart."""
    dev = weight.device
    if weight.dim() != 2 or scale.dim() != 2 or x.dim() != 2:
        _fail(_INVALID_SHAPE, "weight [rows, cols], scale, x [tokens, cols]")
    rows, cols = weight.shape
    tokens = x.shape[0]
    _int(max(rows, cols), "weight")
    _int(tokens, "x")
    _on_gpu(ctx, dev, "weight")
    _dense(weight, torch.uint8, rows * cols, dev, "weight")
    srows, scols = scale.shape
    if srows != (rows + 127) // 128 or scols != (cols + 127) // 128:
        _fail(_INVALID_SHAPE, f"scale: {(srows, scols)}, one for each block of 128 x 128")
    _dense(scale, torch.uint8, srows * scols, dev, "scale")
    code = _dtype_code(x.dtype)
    ldx = _rows(x, tokens, cols, "x")
    if x.device != dev:
        _fail(_INVALID_POINTER, f"x: on {x.device}, not {dev}")
    if not isinstance(act_quant_block, int) or act_quant_block not in (32, 64, 128):
        _fail(_UNSUPPORTED, f"act_quant_block {act_quant_block}: 32, 64 or 128")
    if out is None:
        out_dtype = x.dtype if out_dtype is None else out_dtype
        out_code, ldy = _dtype_code(out_dtype), rows
    else:
        if out_dtype is not None and out.dtype is not out_dtype:
            _fail(_UNSUPPORTED, f"out: {out.dtype}, not {out_dtype}")
        if out.device != dev:
            _fail(_INVALID_POINTER, f"out: on {out.device}, not {dev}")
        out_code, ldy = _dtype_code(out.dtype), _rows(out, tokens, rows, "out")
    with _on(stream):
        if out is None:
            out = torch.empty((tokens, rows), dtype=out_dtype, device=dev)
        if scratch is None:
            size = _scratch_bytes(cols, tokens)
            if size:
                scratch = torch.empty(size, dtype=torch.uint8, device=dev)
        else:
            _dense(scratch, scratch.dtype, scratch.numel(), dev, "scratch")
            size = scratch.numel() * scratch.element_size()
    _check(lib().wh_fp8_gemm(ctx.handle, weight.data_ptr(), scale.data_ptr(), rows, cols, srows,
                             scols, x.data_ptr(), code, tokens, ldx, out.data_ptr(), out_code, ldy,
                             act_quant_block, _ptr(scratch), size, _handle(stream, dev)))
    return out
