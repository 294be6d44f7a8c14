"""The row tables' native entries by their formulas, on host memory (contiguous float32 rows, int8 codes): for
CPU tests of the Python boundary around them."""
import ctypes as ct

import numpy as np

from horizongs_amd import _native as N
from horizongs_amd import embedding as E
from horizongs_amd import rowcache as R


def at(ptr, ctype, *shape):
    if not all(shape):
        return np.empty(shape, ctype)  # such tensors have no memory
    return np.ctypeslib.as_array(ct.cast(ptr, ct.POINTER(ctype)), shape)


def numbers(ptr, n, is64):
    return at(ptr, ct.c_int64 if is64 else ct.c_int32, n)


def formulas(index, name, *a):
    if name == "hgsr_embed_fwd":
        V, n, D, w, _, _, ids, ids64, _, scale, out, _ = a
        at(out, ct.c_float, n, D)[:] = at(w, ct.c_float, V, D)[numbers(ids, n, ids64)] * scale
    elif name == "hgsr_embed_bwd":
        V, n, D, g, _, _, ids, ids64, _, scale, dw, _, _, accumulate, _, _ = a
        if not accumulate:
            at(dw, ct.c_float, V, D)[:] = 0
        np.add.at(at(dw, ct.c_float, V, D), numbers(ids, n, ids64), at(g, ct.c_float, n, D) * scale)
    elif name == "hgsr_rowcache_write":  # codes: the slot's last row rounded, scales 1
        cap, n, D, group, _, x, _, _, slots, slots64, _, codes, _, scales, _, _, _ = a
        k = numbers(slots, n, slots64) if slots else np.arange(n)
        at(codes, ct.c_int8, cap, D)[k] = np.rint(at(x, ct.c_float, n, D))
        at(scales, ct.c_float, cap, -(-D // group))[k] = 1
    else:
        assert name == "hgsr_rowcache_read"
        cap, n, D, group, _, codes, _, scales, _, slots, slots64, _, out, _ = a
        k = numbers(slots, n, slots64) if slots else np.arange(n)
        at(out, ct.c_float, n, D)[:] = at(codes, ct.c_int8, cap, D)[k] * at(scales, ct.c_float, cap, -(-D // group))[k][:, :1]


def install(monkeypatch):
    monkeypatch.setattr(N, "call_on", formulas)
    monkeypatch.setattr(N, "size_query", lambda *a: 0)
    for m in (E, R):
        monkeypatch.setattr(m, "check_device", lambda *ts: 0)
