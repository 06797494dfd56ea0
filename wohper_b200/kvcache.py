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

import ctypes as C
from dataclasses import dataclass
from typing import Optional

from . import Context, WohperError, _check, _ptr, _stream, lib

_INVALID_SHAPE, _INVALID_POINTER, _UNSUPPORTED = 2, 9, 10


class KvCacheSpec(C.Structure):
    """wh_kv_cache."""
    _fields_ = [("blocks", C.c_int), ("page", C.c_int), ("kv_heads", C.c_int),
                ("head_dim", C.c_int), ("keys", C.c_void_p), ("key_scales", C.c_void_p),
                ("values", C.c_void_p), ("value_scales", C.c_void_p),
                ("block_stride", C.c_longlong), ("scale_block_stride", C.c_longlong)]


def _need(ok: bool, status: int, why: str) -> None:
    if not ok:
        raise WohperError(status, why)


def _dtype_code(dtype) -> int:
    import torch

    codes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    _need(dtype in codes, _UNSUPPORTED, f"dtype {dtype}: float32, bfloat16 or float16")
    return codes[dtype]


def _ints(t, dtype, n, device, what: str) -> None:
    """A dense CUDA tensor of n elements of `dtype` on `device`."""
    _need(t.dtype == dtype, _UNSUPPORTED, f"{what}: {t.dtype}, not {dtype}")
    _need(t.numel() == n and t.is_contiguous(), _INVALID_SHAPE, f"{what}: {n} dense elements")
    _need(t.device == device, _INVALID_POINTER, f"{what}: on {t.device}, not {device}")


def _on(stream):
    """Allocations inside belong to the stream that the call runs on."""
    import contextlib

    import torch

    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


@dataclass
class PagedKvCache:
    """A pool of blocks: uint8 CUDA tensors keys [blocks, kv_heads, page,
    head_dim / 2] and key_scales [blocks, kv_heads, page, head_dim / 32]; values
    and value_scales alike, or None where the values are the keys (a latent
    cache).  The outermost stride may be wider than dense (a layer's slice of a
    pool that holds several); it must be the same for keys and values."""
    keys: object
    key_scales: object
    values: Optional[object] = None
    value_scales: Optional[object] = None

    def __post_init__(self):
        import torch

        _need((self.values is None) == (self.value_scales is None), _INVALID_POINTER,
              "values and value_scales go together")
        _need(self.keys.dim() == 4, _INVALID_SHAPE, "keys: [blocks, kv_heads, page, head_dim / 2]")
        b, h, p, half = self.keys.shape
        for t, last, what in ((self.keys, half, "keys"), (self.key_scales, half // 16, "key_scales"),
                              (self.values, half, "values"),
                              (self.value_scales, half // 16, "value_scales")):
            if t is None:
                continue
            _need(t.dtype == torch.uint8, _UNSUPPORTED, f"{what}: {t.dtype}, not torch.uint8")
            _need(half % 16 == 0 and tuple(t.shape) == (b, h, p, last), _INVALID_SHAPE,
                  f"{what}: {tuple(t.shape)}")
            _need(t[0].is_contiguous(), _INVALID_SHAPE, f"{what}: dense inside a block")
            _need(t.device == self.keys.device, _INVALID_POINTER, f"{what}: on {t.device}")
        if self.values is not None:
            _need(self.values.stride(0) == self.keys.stride(0) and
                  self.value_scales.stride(0) == self.key_scales.stride(0), _INVALID_SHAPE,
                  "keys and values: one block stride")
        # a stride means nothing where there is a single block
        wide = b > 1
        self._spec = KvCacheSpec(b, p, h, 2 * half, _ptr(self.keys), _ptr(self.key_scales),
                                 _ptr(self.values), _ptr(self.value_scales),
                                 self.keys.stride(0) if wide else 0,
                                 self.key_scales.stride(0) if wide else 0)

    @classmethod
    def empty(cls, blocks: int, page: int, kv_heads: int, head_dim: int,
              separate_values: bool = False, device="cuda") -> "PagedKvCache":
        """A zeroed pool (every row reads as zeros)."""
        import torch

        def z(last):
            return torch.zeros(blocks, kv_heads, page, last, dtype=torch.uint8, device=device)

        _need(head_dim % 32 == 0, _INVALID_SHAPE, "head_dim % 32 != 0")
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
    import torch

    n, dev = kv_lens.numel(), kv_lens.device
    _ints(kv_lens, torch.int32, n, dev, "kv_lens")
    _ints(q_lens, torch.int32, n, dev, "q_lens")
    _need(block_table.dim() == 2 and block_table.shape[0] == n, _INVALID_SHAPE,
          "block_table: [requests, max_blocks]")
    _ints(block_table, torch.int32, block_table.numel(), dev, "block_table")
    _ints(free_blocks, torch.int32, free_blocks.numel(), dev, "free_blocks")
    _ints(free_top, torch.int32, 1, dev, "free_top")
    if finished is not None:
        _need(finished.dtype in (torch.uint8, torch.bool), _UNSUPPORTED, "finished: uint8 or bool")
        _ints(finished, finished.dtype, n, dev, "finished")
    _need(tokens >= 0, _INVALID_SHAPE, "tokens < 0")
    with _on(stream):
        # one allocation: lens | cu_q | top | positions | requests | scratch, then the slots
        ints = torch.empty(3 * n + 2 + 2 * tokens, dtype=torch.int32, device=dev)
        slots = torch.empty(tokens, dtype=torch.int64, device=dev)
    lens, cu, top, pos, who, scratch = ints.split((n, n + 1, 1, tokens, tokens, n))
    base = ints.data_ptr()
    at = [base + 4 * o for o in (0, n, 2 * n + 1, 2 * n + 2, 2 * n + 2 + tokens,
                                 2 * n + 2 + 2 * tokens)]
    _check(lib().wh_kv_plan(ctx.handle, n, page, block_table.shape[1], tokens, _ptr(kv_lens),
                            _ptr(q_lens), _ptr(finished), _ptr(block_table), _ptr(free_blocks),
                            free_blocks.numel(), _ptr(free_top), at[2], at[0], at[1],
                            _ptr(slots), at[3], at[4], at[5], 4 * n, _stream(stream)))
    return KvPlan(lens, cu, slots, pos, who, top)


def _row_strides(x, cache: PagedKvCache, rows: int, what: str):
    """Strides of [rows, kv_heads, head_dim]; a size-1 dimension's stride is free."""
    _need(tuple(x.shape) == (rows, cache.kv_heads, cache.head_dim), _INVALID_SHAPE,
          f"{what}: {tuple(x.shape)}, not {(rows, cache.kv_heads, cache.head_dim)}")
    _need(x.stride(2) == 1, _INVALID_SHAPE, f"{what}: contiguous rows")
    _need(x.device == cache.keys.device, _INVALID_POINTER, f"{what}: on {x.device}")
    return (x.stride(0) if x.shape[0] > 1 else 0, x.stride(1) if x.shape[1] > 1 else 0)


def kv_append(ctx: Context, cache: PagedKvCache, slots, keys, values=None, stream=None) -> None:
    """Quantises keys (and values) [rows, kv_heads, head_dim], f32, bf16 or f16,
    into the cache's slots (int64 [rows]; negative: skipped)."""
    import torch

    rows = slots.numel()
    _ints(slots, torch.int64, rows, cache.keys.device, "slots")
    _need((values is None) == (cache.values is None), _INVALID_POINTER,
          "values exactly when the cache has values")
    ks = _row_strides(keys, cache, rows, "keys")
    vs = (0, 0)
    if values is not None:
        _need(values.dtype == keys.dtype, _UNSUPPORTED, "keys and values: one dtype")
        vs = _row_strides(values, cache, rows, "values")
    _check(lib().wh_kv_append(ctx.handle, C.byref(cache.spec()), _ptr(slots), rows, _ptr(keys),
                              _ptr(values), _dtype_code(keys.dtype), *ks, *vs, _stream(stream)))


def kv_gather(ctx: Context, cache: PagedKvCache, slots, dtype=None, stream=None):
    """The rows of slots (int64 [rows]; negative: zeros) as values: (keys, values)
    [rows, kv_heads, head_dim] of dtype (float32 by default); values is None for
    a cache whose values are its keys."""
    import torch

    rows = slots.numel()
    _ints(slots, torch.int64, rows, cache.keys.device, "slots")
    dtype = torch.float32 if dtype is None else dtype
    code = _dtype_code(dtype)
    shape = (rows, cache.kv_heads, cache.head_dim)
    with _on(stream):
        k = torch.empty(shape, dtype=dtype, device=slots.device)
        v = None if cache.values is None else torch.empty(shape, dtype=dtype, device=slots.device)
    _check(lib().wh_kv_gather(ctx.handle, C.byref(cache.spec()), _ptr(slots), rows, _ptr(k),
                              _ptr(v), code, _stream(stream)))
    return k, v


def kv_attention(ctx: Context, cache: PagedKvCache, q, cu_q, kv_lens, block_table,
                 scale: Optional[float] = None, window: int = 0, first: int = 0, sink=None,
                 out=None, scratch=None, stream=None):
    """Attention of the queries q [tokens, heads, head_dim] over the cached rows
    (wh_kv_attention): request r owns the queries cu_q[r] .. cu_q[r + 1] - 1
    (cu_q None: one each) and kv_lens[r] rows, the new ones included; the last
    query sits at position kv_lens[r] - 1.  A query at p sees rows i <= p and,
    with a window, only i > p - window or i < first.  sink: f32 [heads] or None.
    scale defaults to head_dim ** -0.5.  Returns out, like q."""
    import torch

    dev = cache.keys.device
    _need(q.dim() == 3 and q.shape[2] == cache.head_dim, _INVALID_SHAPE,
          "q: [tokens, heads, head_dim]")
    code = _dtype_code(q.dtype)
    tokens, heads, d = q.shape
    n = kv_lens.numel()
    _need(q.device == dev, _INVALID_POINTER, f"q: on {q.device}, not {dev}")
    _ints(kv_lens, torch.int32, n, dev, "kv_lens")
    if cu_q is not None:
        _ints(cu_q, torch.int32, n + 1, dev, "cu_q")
    _need(block_table.dim() == 2 and block_table.shape[0] == n, _INVALID_SHAPE,
          "block_table: [requests, max_blocks]")
    _ints(block_table, torch.int32, block_table.numel(), dev, "block_table")
    if sink is not None:
        _ints(sink, torch.float32, heads, dev, "sink")
    with _on(stream):
        if out is None:
            out = torch.empty((tokens, heads, d), dtype=q.dtype, device=dev)
        need = int(lib().wh_kv_attention_scratch_bytes(ctx.handle, C.byref(cache.spec()), tokens,
                                                       heads, n, code))
        if scratch is None:
            scratch = torch.empty(need, dtype=torch.uint8, device=dev)
    _need(out.shape == q.shape and out.dtype == q.dtype and out.device == dev, _INVALID_SHAPE,
          "out: like q")
    _need(q.stride(2) == 1 and out.stride(2) == 1, _INVALID_SHAPE, "q, out: contiguous rows")
    st = [t.stride(i) if t.shape[i] > 1 else 0 for t in (q, out) for i in (0, 1)]
    _check(lib().wh_kv_attention(ctx.handle, C.byref(cache.spec()), _ptr(q), code, tokens, heads,
                                 st[0], st[1], n, _ptr(cu_q), _ptr(kv_lens), _ptr(block_table),
                                 block_table.shape[1], d ** -0.5 if scale is None else scale,
                                 window, first, _ptr(sink), _ptr(out), st[2], st[3],
                                 _ptr(scratch), scratch.numel() * scratch.element_size(),
                                 _stream(stream)))
    return out
