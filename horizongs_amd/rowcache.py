"""A cache of rows held in 8 bits (csrc/rowcache.hip): quantised as they are written into their
slots, read back by slot.

    cache = rowcache_alloc(capacity, dim, "int8", group=32, device="cuda")
    rowcache_write(cache, rows, slots)           # rows [n, dim], slots [n]; None: slots 0 .. n - 1
    rows = rowcache_read(cache, slots)           # None: every slot

A cache is (codes, scales, group): codes int8 or float8_e4m3fn [capacity, dim], one float32 scale for
each `group` columns in scales [capacity, ceil(dim / group)].  A row x is held as
s = max(max |x| over the group * (1 / 127) (e4m3: 1 / 448), 2^-100) in f32 and x / s rounded to the nearest
code, ties to even; x' = code * s reads back within s / 2 (int8), or within 2^-4 of each value and 2^-10 s (e4m3).  A
group that holds a NaN or an infinity reads back as NaN.  decode.decode() takes a cache for the anchor
features: the visible anchors' rows are read back for each view (a quarter of their float32 bytes are
kept, plus the scales).  No derivative passes through a cache, in reverse or in forward mode, and
its calls cannot be traced.  There is no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from .embedding import (_TYPES, check_device, check_ids, id_stride, increment_version, refuse_trace, row_stride,
                        type_code)

_FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}
_NAMES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
GROUPS = (16, 32, 64, 128)


class RowCache(NamedTuple):
    codes: torch.Tensor
    scales: torch.Tensor
    group: int = 32


def rowcache_alloc(capacity, dim, fmt="int8", group=32, device="cuda"):
    """An empty cache: every slot reads back as zeros until it is written."""
    if fmt not in _NAMES:
        raise ValueError(f"hgsr row cache: format {fmt!r}: 'int8' or 'e4m3'")
    if group not in GROUPS:
        raise ValueError(f"hgsr row cache: group of {group} columns: one of {GROUPS}")
    if capacity < 0 or dim < 1:
        raise ValueError(f"hgsr row cache: {capacity} slots of {dim} columns")
    codes = torch.zeros(capacity, dim, dtype=torch.uint8, device=device).view(_NAMES[fmt])
    return RowCache(codes, torch.zeros(capacity, -(-dim // group), device=device), group)


def _cache(cache):
    refuse_trace()
    codes, scales, group = cache
    if group not in GROUPS:
        raise ValueError(f"hgsr row cache: group of {group} columns: one of {GROUPS}")
    if codes.dtype not in _FORMATS or codes.dim() != 2 or codes.shape[1] < 1:
        raise ValueError(f"hgsr row cache: codes {tuple(codes.shape)} of {codes.dtype}: [capacity, columns] of int8 or "
                         "float8_e4m3fn are needed")
    capacity, dim = codes.shape
    groups = -(-dim // group)
    if scales.dtype != torch.float32 or scales.shape != (capacity, groups):
        raise ValueError(f"hgsr row cache: scales {tuple(scales.shape)} of {scales.dtype} do not fit codes "
                         f"{tuple(codes.shape)} in groups of {group}")
    cs, ss = row_stride(codes, "codes"), row_stride(scales, "scales")
    if cs < dim or ss < groups:
        raise ValueError("hgsr row cache: its rows overlap")
    return codes, scales, group, capacity, dim, cs, ss


def _slot_args(slots):
    if slots is None:
        return None, 0, 1
    return slots.data_ptr(), int(slots.dtype == torch.int64), id_stride(slots)


def _check_slots(slots, n):
    if slots.dim() != 1 or (n is not None and slots.shape[0] != n):
        raise ValueError(f"hgsr row cache: slots {tuple(slots.shape)}: [n] is needed, one number for each row")
    check_ids(slots)


def rowcache_write(cache, rows, slots=None):
    """Quantise rows [n, dim] (float32, float16 or bfloat16, contiguous columns) into their slots (int32 /
    int64 [n]; None: slots 0 .. n - 1).  A row whose slot lies outside the cache (-1 by custom) is left
    out; where a slot is named twice, the last of its rows stays.  Other slots keep what they hold.  A
    write is ordered on the current stream like any kernel; two streams must not write one slot at once."""
    codes, scales, group, capacity, dim, cs, ss = _cache(cache)
    xt = type_code(rows.dtype)
    if rows.dim() != 2 or rows.shape[1] != dim:
        raise ValueError(f"hgsr row cache: rows {tuple(rows.shape)}: [n, {dim}] are needed")
    n = rows.shape[0]
    xs = row_stride(rows, "rows")
    if slots is None:
        if n > capacity:
            raise ValueError(f"hgsr row cache: {n} rows, {capacity} slots")
        index = check_device(codes, scales, rows)
    else:
        _check_slots(slots, n)
        index = check_device(codes, scales, rows, slots)
    if n == 0 or capacity == 0:
        return
    ws_b = N.size_query("hgsr_rowcache_write_ws_bytes", capacity, n, dim, int(slots is not None))
    ws = torch.empty(ws_b, dtype=torch.uint8, device=codes.device) if ws_b else None
    N.call_on(index, "hgsr_rowcache_write", capacity, n, dim, group, _FORMATS[codes.dtype], rows.data_ptr(), xt, xs,
              *_slot_args(slots), codes.data_ptr(), cs, scales.data_ptr(), ss, ws.data_ptr() if ws_b else None, ws_b)
    increment_version((codes, scales))  # a backward that saved them as they were must not go on with them


def rowcache_read(cache, slots=None, dtype=torch.float32):
    """Rows [n, dim] of the named slots (int32 / int64 [n]; None: every slot) in `dtype`: code * scale in
    f32, rounded once.  A slot outside the cache reads zeros."""
    codes, scales, group, capacity, dim, cs, ss = _cache(cache)
    ot = type_code(dtype)
    if slots is None:
        n, index = capacity, check_device(codes, scales)
    else:
        _check_slots(slots, None)
        n, index = slots.shape[0], check_device(codes, scales, slots)
    out = scales.new_empty((n, dim), dtype=dtype)
    if n:
        N.call_on(index, "hgsr_rowcache_read", capacity, n, dim, group, _FORMATS[codes.dtype], codes.data_ptr(), cs,
                  scales.data_ptr(), ss, *_slot_args(slots), out.data_ptr(), ot)
    return out
