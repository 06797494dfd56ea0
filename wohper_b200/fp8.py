"""The Python side of wh_fp8_gemm (``gemm_fp8_e4m3_ue8m0``), imported with torch on
first use."""
from __future__ import annotations

import torch

from . import Context, _check, lib
from .kvcache import (_INVALID_POINTER, _INVALID_SHAPE, _UNSUPPORTED, _dense, _dtype_code, _fail,
                      _handle, _on, _on_gpu)


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


def gemm(ctx: Context, weight, scale, x, act_quant_block, out_dtype, out, scratch, stream):
    dev = weight.device
    _on_gpu(ctx, dev, "weight")
    if weight.dim() != 2 or scale.dim() != 2 or x.dim() != 2:
        _fail(_INVALID_SHAPE, "weight [rows, cols], scale, x [tokens, cols]")
    rows, cols = weight.shape
    tokens = x.shape[0]
    _dense(weight, torch.uint8, rows * cols, dev, "weight")
    if scale.shape != (-(-rows // 128), -(-cols // 128)):
        _fail(_INVALID_SHAPE, f"scale: {tuple(scale.shape)}, one for each block of 128 x 128")
    _dense(scale, torch.uint8, scale.numel(), dev, "scale")
    code = _dtype_code(x.dtype)
    ldx = _rows(x, tokens, cols, "x")
    if x.device != dev:
        _fail(_INVALID_POINTER, f"x: on {x.device}, not {dev}")
    if not isinstance(act_quant_block, int) or act_quant_block not in (32, 64, 128):
        _fail(_UNSUPPORTED, f"act_quant_block {act_quant_block}: 32, 64 or 128")
    if out is not None:
        if out_dtype is not None and out.dtype is not out_dtype:
            _fail(_UNSUPPORTED, f"out: {out.dtype}, not {out_dtype}")
        if out.device != dev:
            _fail(_INVALID_POINTER, f"out: on {out.device}, not {dev}")
    elif out_dtype is None:
        out_dtype = x.dtype
    out_code = _dtype_code(out_dtype if out is None else out.dtype)
    with _on(stream):
        if out is None:
            out = torch.empty((tokens, rows), dtype=out_dtype, device=dev)
        if scratch is None:
            scratch = torch.empty(lib().wh_fp8_gemm_scratch_bytes(cols, tokens), dtype=torch.uint8,
                                  device=dev)
        else:
            _dense(scratch, scratch.dtype, scratch.numel(), dev, "scratch")
    ldy = _rows(out, tokens, rows, "out")
    _check(lib().wh_fp8_gemm(ctx.handle, weight.data_ptr(), scale.data_ptr(), rows, cols,
                             scale.shape[0], scale.shape[1], x.data_ptr(), code, tokens, ldx,
                             out.data_ptr(), out_code, ldy, act_quant_block, scratch.data_ptr(),
                             scratch.numel() * scratch.element_size(), _handle(stream, dev)))
    return out
