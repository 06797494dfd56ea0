"""The paged key/value cache in 4 bits: its pool, a serving step's plan, writes,
reads and attention (``wh_kv_*`` in ``include/wohper_b200.h``).

One step of a server, per layer and without a host synchronisation:

    plan = kv_plan(ctx, page, kv_lens, q_lens, block_table, free_blocks, free_top, tokens)
    kv_append(ctx, cache, plan.slots, k)                       # the step's new rows
    out = kv_attention(ctx, cache, q, plan.cu_q, plan.kv_lens, block_table)

A row is E2M1 codes (OCP values, low nibble = even column) with one UE8M0 scale
per 32.  The reference engine keeps f32 rows and has no counterpart.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from . import Context, WohperError, _check, _ptr, lib

_INVALID_SHAPE, _INVALID_POINTER, _UNSUPPORTED = 2, 9, 10
_INT_MAX = 0x7FFFFFFF  # ctypes would wrap what the C calls' int does not hold
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _current_stream(index: int) -> int:
    return int(torch.cuda.current_stream(index).cuda_stream)


# torch's own short cut to the same handle, where this torch has it
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


class KvCacheSpec(C.Structure):
    """wh_kv_cache."""
    _fields_ = [("blocks", C.c_int), ("page", C.c_int), ("kv_heads", C.c_int),
                ("head_dim", C.c_int), ("keys", C.c_void_p), ("key_scales", C.c_void_p),
                ("values", C.c_void_p), ("value_scales", C.c_void_p),
                ("block_stride", C.c_longlong), ("scale_block_stride", C.c_longlong)]


def _fail(status: int, why: str):
    raise WohperError(status, why)


def _dtype_code(dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        _fail(_UNSUPPORTED, f"dtype {dtype}: float32, bfloat16 or float16")
    return code


def _dense(t, dtype, n, device, what: str) -> None:
    """Raises unless t is a dense tensor of n elements of `dtype` on `device`."""
    if t.dtype is dtype and t.numel() == n and t.is_contiguous() and t.device == device:
        return
    if t.dtype is not dtype:
        _fail(_UNSUPPORTED, f"{what}: {t.dtype}, not {dtype}")
    if t.device != device:
        _fail(_INVALID_POINTER, f"{what}: on {t.device}, not {device}")
    _fail(_INVALID_SHAPE, f"{what}: {n} dense elements")


def _on_gpu(ctx: Context, device, what: str) -> None:
    """Raises unless `device` is the context's GPU."""
    if device.type != "cuda" or device.index != ctx.device:
        _fail(_INVALID_POINTER, f"{what}: on {device}, not on the context's cuda:{ctx.device}")


def _handle(stream, device) -> int:
    """The cudaStream_t of stream, or of the current stream (in one call of torch's)."""
    if stream is not None:
        return int(stream.cuda_stream)
    return _current_stream(device.index)


def _on(stream):
    """Allocations inside belong to the stream that the call runs on."""
    return _HERE if stream is None else torch.cuda.stream(stream)


_HERE = contextlib.nullcontext()


@dataclass(frozen=True)
class PagedKvCache:
    """A pool of blocks: uint8 CUDA tensors keys [blocks, kv_heads, page,
    head_dim / 2] and key_scales [blocks, kv_heads, page, head_dim / 32]; values
    and value_scales alike, or None where the values are the keys (a latent
    cache).  The outermost stride may be wider than dense (a layer's slice of a
    pool that holds several); it must be the same for keys and values.  A cache
    keeps the tensors that it was made of: other tensors are another cache."""
    keys: object
    key_scales: object
    values: Optional[object] = None
    value_scales: Optional[object] = None

    def __post_init__(self):
        k, ks, v, vs = self.keys, self.key_scales, self.values, self.value_scales
        if (v is None) != (vs is None):
            _fail(_INVALID_POINTER, "values and value_scales go together")
        if k.dim() != 4:
            _fail(_INVALID_SHAPE, "keys: [blocks, kv_heads, page, head_dim / 2]")
        b, h, p, half = k.shape
        if half % 16:
            _fail(_INVALID_SHAPE, f"keys: {tuple(k.shape)}: head_dim % 32 != 0")
        rest, scales = (b, h, p, half), (b, h, p, half // 16)
        for t, shape, what in ((k, rest, "keys"), (ks, scales, "key_scales"), (v, rest, "values"),
                               (vs, scales, "value_scales")):
            if t is None:
                continue
            if t.dtype is not torch.uint8:
                _fail(_UNSUPPORTED, f"{what}: {t.dtype}, not torch.uint8")
            if t.shape != shape:
                _fail(_INVALID_SHAPE, f"{what}: {tuple(t.shape)}, not {shape}")
            if not t.is_contiguous() and not t[0].is_contiguous():
                _fail(_INVALID_SHAPE, f"{what}: dense inside a block")
            if t.device != k.device:
                _fail(_INVALID_POINTER, f"{what}: on {t.device}, not {k.device}")
        step, scale_step = k.stride(0), ks.stride(0)
        if v is not None and (v.stride(0) != step or vs.stride(0) != scale_step):
            _fail(_INVALID_SHAPE, "keys and values: one block stride")
        if b == 1:  # a stride means nothing where there is a single block
            step = scale_step = 0
        elif step < h * p * half or scale_step < h * p * (half // 16):
            # 0 (an expanded tensor) would read as a dense pool
            _fail(_INVALID_SHAPE, "keys, scales: a block stride below a block's size")
        spec = KvCacheSpec(b, p, h, 2 * half, k.data_ptr(), ks.data_ptr(), _ptr(v), _ptr(vs), step,
                           scale_step)
        object.__setattr__(self, "_spec", spec)
        object.__setattr__(self, "_ref", C.byref(spec))

    @classmethod
    def empty(cls, blocks: int, page: int, kv_heads: int, head_dim: int,
              separate_values: bool = False, device="cuda") -> "PagedKvCache":
        """A zeroed pool (every row reads as zeros)."""
        def z(last):
            return torch.zeros(blocks, kv_heads, page, last, dtype=torch.uint8, device=device)

        if head_dim % 32:
            _fail(_INVALID_SHAPE, "head_dim % 32 != 0")
        args = [z(head_dim // 2), z(head_dim // 32)]
        if separate_values:
            args += [z(head_dim // 2), z(head_dim // 32)]
        return cls(*args)

    def spec(self) -> KvCacheSpec:
        return self._spec

    @property
    def blocks(self) -> int:
        return self._spec.blocks

    @property
    def page(self) -> int:
        return self._spec.page

    @property
    def kv_heads(self) -> int:
        return self._spec.kv_heads

    @property
    def head_dim(self) -> int:
        return self._spec.head_dim


@dataclass
class KvPlan:
    """What kv_plan gives: int32 device tensors kv_lens [requests], cu_q
    [requests + 1], positions and requests [tokens], free_top [1], and int64
    slots [tokens] (-1 past the last new token)."""
    kv_lens: object
    cu_q: object
    slots: object
    positions: object
    requests: object
    free_top: object


def kv_plan(ctx: Context, page: int, kv_lens, q_lens, block_table, free_blocks, free_top,
            tokens: int, finished=None, stream=None) -> KvPlan:
    """The bookkeeping of one serving step on the device (wh_kv_plan): request r
    has kv_lens[r] rows and gets q_lens[r] tokens (int32 device tensors);
    requests marked in finished (uint8 or bool, or None) give their blocks back.
    block_table [requests, max_blocks] and the stack free_blocks (height
    free_top [1]) are updated in place; tokens is the step's token count, or a
    larger fixed one (a captured graph).  A step that does not fit changes
    nothing, gives no tokens, and ctx.sync() raises DeviceArg."""
    n, dev = kv_lens.numel(), kv_lens.device
    _on_gpu(ctx, dev, "kv_lens")
    i32 = torch.int32
    _dense(kv_lens, i32, n, dev, "kv_lens")
    _dense(q_lens, i32, n, dev, "q_lens")
    if block_table.dim() != 2 or block_table.shape[0] != n:
        _fail(_INVALID_SHAPE, "block_table: [requests, max_blocks]")
    _dense(block_table, i32, block_table.numel(), dev, "block_table")
    capacity = free_blocks.numel()
    _dense(free_blocks, i32, capacity, dev, "free_blocks")
    _dense(free_top, i32, 1, dev, "free_top")
    if finished is not None:
        if finished.dtype is not torch.uint8 and finished.dtype is not torch.bool:
            _fail(_UNSUPPORTED, "finished: uint8 or bool")
        _dense(finished, finished.dtype, n, dev, "finished")
    if not 0 <= tokens <= _INT_MAX or not 0 <= page <= _INT_MAX:
        _fail(_INVALID_SHAPE, f"tokens {tokens}, page {page}")
    with _on(stream):
        # lens | cu_q | top | positions | requests | scratch in one allocation, the slots in another
        ints = kv_lens.new_empty(3 * n + 2 + 2 * tokens)
        slots = torch.empty(tokens, dtype=torch.int64, device=dev)
    lens, cu, top, pos, who, _ = ints.split_with_sizes((n, n + 1, 1, tokens, tokens, n))
    at = ints.data_ptr()
    cu_at = at + 4 * n
    pos_at = cu_at + 4 * (n + 2)
    _check(lib().wh_kv_plan(ctx.handle, n, page, block_table.shape[1], tokens, kv_lens.data_ptr(),
                            q_lens.data_ptr(), _ptr(finished), block_table.data_ptr(),
                            free_blocks.data_ptr(), capacity, free_top.data_ptr(),
                            cu_at + 4 * (n + 1), at, cu_at, slots.data_ptr(), pos_at,
                            pos_at + 4 * tokens, pos_at + 8 * tokens, 4 * n,
                            _handle(stream, dev)))
    return KvPlan(lens, cu, slots, pos, who, top)


def _row_strides(x, cache: PagedKvCache, rows: int, what: str):
    """Strides of [rows, kv_heads, head_dim]; a size-1 dimension's stride is free."""
    shape = (rows, cache.kv_heads, cache.head_dim)
    if x.shape != shape:
        _fail(_INVALID_SHAPE, f"{what}: {tuple(x.shape)}, not {shape}")
    a, b, c = x.stride()
    if c != 1:
        _fail(_INVALID_SHAPE, f"{what}: contiguous rows")
    if x.device != cache.keys.device:
        _fail(_INVALID_POINTER, f"{what}: on {x.device}")
    return (a if rows > 1 else 0, b if shape[1] > 1 else 0)


def kv_append(ctx: Context, cache: PagedKvCache, slots, keys, values=None, stream=None) -> None:
    """Quantises keys (and values) [rows, kv_heads, head_dim], f32, bf16 or f16,
    into the cache's slots (int64 [rows]; negative: skipped; twice the same: its row
    is undefined)."""
    rows, dev = slots.numel(), cache.keys.device
    _on_gpu(ctx, dev, "cache")
    _dense(slots, torch.int64, rows, dev, "slots")
    if (values is None) != (cache.values is None):
        _fail(_INVALID_POINTER, "values exactly when the cache has values")
    ks = _row_strides(keys, cache, rows, "keys")
    vs = (0, 0)
    if values is not None:
        if values.dtype is not keys.dtype:
            _fail(_UNSUPPORTED, "keys and values: one dtype")
        vs = _row_strides(values, cache, rows, "values")
    _check(lib().wh_kv_append(ctx.handle, cache._ref, slots.data_ptr(), rows, keys.data_ptr(),
                              _ptr(values), _dtype_code(keys.dtype), *ks, *vs,
                              _handle(stream, dev)))


def kv_gather(ctx: Context, cache: PagedKvCache, slots, dtype=None, stream=None):
    """The rows of slots (int64 [rows]; negative: zeros) as values: (keys, values)
    [rows, kv_heads, head_dim] of dtype (float32 by default); values is None for
    a cache whose values are its keys."""
    rows, dev = slots.numel(), cache.keys.device
    _on_gpu(ctx, dev, "cache")
    _dense(slots, torch.int64, rows, dev, "slots")
    dtype = torch.float32 if dtype is None else dtype
    code = _dtype_code(dtype)
    shape = (rows, cache.kv_heads, cache.head_dim)
    with _on(stream):
        k = torch.empty(shape, dtype=dtype, device=dev)
        v = None if cache.values is None else torch.empty(shape, dtype=dtype, device=dev)
    _check(lib().wh_kv_gather(ctx.handle, cache._ref, slots.data_ptr(), rows, k.data_ptr(),
                              _ptr(v), code, _handle(stream, dev)))
    return k, v


_scratch_sizes: dict = {}


def _scratch_bytes(ctx: Context, cache: PagedKvCache, tokens: int, heads: int, requests: int,
                   code: int) -> int:
    """wh_kv_attention_scratch_bytes, asked once for the same device and sizes."""
    s = cache._spec
    key = (ctx.device, s.kv_heads, s.head_dim, tokens, heads, requests, code)
    size = _scratch_sizes.get(key)
    if size is None:
        if len(_scratch_sizes) >= 256:
            _scratch_sizes.clear()
        size = _scratch_sizes[key] = int(lib().wh_kv_attention_scratch_bytes(
            ctx.handle, cache._ref, tokens, heads, requests, code))
    return size


def kv_attention(ctx: Context, cache: PagedKvCache, q, cu_q, kv_lens, block_table,
                 scale: Optional[float] = None, window: int = 0, first: int = 0, sink=None,
                 out=None, scratch=None, stream=None):
    """Attention of the queries q [tokens, heads, head_dim] over the cached rows
    (wh_kv_attention): request r owns the queries cu_q[r] .. cu_q[r + 1] - 1
    (cu_q None: one each) and kv_lens[r] rows, the new ones included; the last
    query sits at position kv_lens[r] - 1.  A query at p sees rows i <= p and,
    with a window, only i > p - window or i < first.  sink: f32 [heads] or None.
    scale defaults to head_dim ** -0.5.  Returns out, like q; out may be q itself,
    but may not overlap it in another way.  Rows of tokens past cu_q[-1] are not
    written: with out=None they hold whatever the memory held (all of them, after a
    step that did not fit).  f32 queries give the accuracy of f32 products; weights
    of 16-bit queries are held in 11 bits."""
    dev = cache.keys.device
    _on_gpu(ctx, dev, "cache")
    if q.dim() != 3 or q.shape[2] != cache.head_dim:
        _fail(_INVALID_SHAPE, "q: [tokens, heads, head_dim]")
    code = _dtype_code(q.dtype)
    tokens, heads, d = q.shape
    n = kv_lens.numel()
    if q.device != dev:
        _fail(_INVALID_POINTER, f"q: on {q.device}, not {dev}")
    _dense(kv_lens, torch.int32, n, dev, "kv_lens")
    if cu_q is not None:
        _dense(cu_q, torch.int32, n + 1, dev, "cu_q")
    if block_table.dim() != 2 or block_table.shape[0] != n:
        _fail(_INVALID_SHAPE, "block_table: [requests, max_blocks]")
    _dense(block_table, torch.int32, block_table.numel(), dev, "block_table")
    if sink is not None:
        _dense(sink, torch.float32, heads, dev, "sink")
    if not 0 <= window <= _INT_MAX or not 0 <= first <= _INT_MAX:
        _fail(_INVALID_SHAPE, f"window {window}, first {first}")
    with _on(stream):
        if out is None:
            out = torch.empty((tokens, heads, d), dtype=q.dtype, device=dev)
        if scratch is None:
            scratch = torch.empty(_scratch_bytes(ctx, cache, tokens, heads, n, code),
                                  dtype=torch.uint8, device=dev)
        else:
            _dense(scratch, scratch.dtype, scratch.numel(), dev, "scratch")
    if out.shape != q.shape or out.dtype is not q.dtype or out.device != dev:
        _fail(_INVALID_SHAPE, "out: like q")
    q0, q1, q2 = q.stride()
    o0, o1, o2 = out.stride()
    if q2 != 1 or o2 != 1:
        _fail(_INVALID_SHAPE, "q, out: contiguous rows")
    if (tokens > 1 and o0 == 0) or (heads > 1 and o1 == 0):
        _fail(_INVALID_SHAPE, "out: rows that share memory")
    if tokens == 1:  # a size-1 dimension's stride is free
        q0 = o0 = 0
    if heads == 1:
        q1 = o1 = 0
    _check(lib().wh_kv_attention(ctx.handle, cache._ref, q.data_ptr(), code, tokens, heads, q0, q1,
                                 n, _ptr(cu_q), kv_lens.data_ptr(), block_table.data_ptr(),
                                 block_table.shape[1], d ** -0.5 if scale is None else scale,
                                 window, first, _ptr(sink), out.data_ptr(), o0, o1,
                                 scratch.data_ptr(), scratch.numel() * scratch.element_size(),
                                 _handle(stream, dev)))
    return out
