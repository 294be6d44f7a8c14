"""Embedding lookup with scaling, and its gradient by sorted ids (csrc/embed.hip).

* `embedding(weight, ids, scale)`        out[..., :] = scale * weight[ids, :], differentiable
* `embedding_grad(grad, ids, num_rows)`  the gradient by itself, dense or added into a table's
* `Embedding`                            <- scene/embedding.py:50-79, the per-camera appearance
                                         rows that condition the colour head (decode.py)

Tables and rows may be float32, float16 or bfloat16; sums are f32, rounded once.  An id outside
[0, num_rows) (-1 by custom) is padding: its row is zeros and it takes no part in the gradient --
there is no host read that could raise.  Gradients are summed in an order that the ids alone set,
so they are the same bits on every run.  There is no CPU path.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from . import gradbuf

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def check_device(*ts):
    dev = ts[0].device
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError("hgsr: inputs must be HIP device tensors (no CPU fallback)")
        if t.device != dev:
            raise RuntimeError(f"hgsr: tensors on {dev} and {t.device}: one device is needed")


def type_code(dtype):
    code = _TYPES.get(dtype)
    if code is None:
        raise ValueError(f"hgsr: float32, float16 or bfloat16 rows are needed, not {dtype}")
    return code


def row_stride(t, what):
    """Elements between the rows of a 2-D tensor whose columns are contiguous."""
    if t.shape[1] > 1 and t.stride(1) != 1 and t.numel():
        raise ValueError(f"hgsr: the columns of {what} must be contiguous (stride {t.stride(1)})")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def rows_view(t, dim, what):
    """[n, dim] view of a tensor's rows with contiguous columns, copied only if there is none."""
    if t.shape[-1] != dim:
        raise ValueError(f"hgsr: rows of {what} have {t.shape[-1]} columns, not {dim}")
    t = t.reshape(-1, dim)
    return t if dim == 1 or t.stride(1) == 1 else t.contiguous()


def check_ids(ids):
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"hgsr: int32 or int64 ids are needed, not {ids.dtype}")


def id_args(ids):
    """(flat ids, whether they are int64, their stride)."""
    flat = ids.reshape(-1)
    return flat, int(ids.dtype == torch.int64), flat.stride(0) if flat.numel() > 1 else 1


def _lookup(weight, ids, scale, dtype):
    V, D = weight.shape
    out = torch.empty(*ids.shape, D, dtype=dtype, device=weight.device)
    n = ids.numel()
    if n and D:
        flat, is64, stride = id_args(ids)
        N.call_on(weight.device, "hgsr_embed_fwd", V, n, D, weight.data_ptr(), _TYPES[weight.dtype],
                  row_stride(weight, "weight"), flat.data_ptr(), is64, stride, scale, out.data_ptr(), _TYPES[dtype])
    return out


def _grad(grad, ids, out, scale, accumulate):
    V, D = out.shape
    n = ids.numel()
    if V == 0 or D == 0 or (n == 0 and accumulate):
        return out
    flat, is64, stride = id_args(ids)
    ws_b = N.size_query("hgsr_embed_bwd_ws_bytes", V, n, D)
    ws = torch.empty(max(ws_b, 1), dtype=torch.uint8, device=out.device)
    N.call_on(out.device, "hgsr_embed_bwd", V, n, D, grad.data_ptr(), _TYPES[grad.dtype], row_stride(grad, "grad"),
              flat.data_ptr(), is64, stride, scale, out.data_ptr(), _TYPES[out.dtype], row_stride(out, "out"),
              int(accumulate), ws.data_ptr(), ws_b)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, dtype):
        ctx.save_for_backward(ids)
        ctx.table = (weight.shape, weight.dtype, gradbuf.key(weight))
        ctx.scale = scale
        return _lookup(weight, ids, scale, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        shape, dtype, key = ctx.table
        out = gradbuf.take(key, shape, dtype)  # in place in a DDP bucket when one is registered
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=g.device)
        return _grad(rows_view(g, shape[1], "grad"), ids, out, ctx.scale, False), None, None, None


def embedding(weight, ids, scale=1.0, dtype=None):
    """scale * weight[ids]: weight [V, D] (any row stride, contiguous columns), ids int32 / int64 of
    any shape; returns [*ids.shape, D] in `dtype` (default: weight's).  The product is f32, rounded
    once.  Differentiable in weight; the gradient has weight's type and a row for each of its rows."""
    if weight.dim() != 2:
        raise ValueError(f"hgsr: weight must be [rows, columns], not {tuple(weight.shape)}")
    dtype = weight.dtype if dtype is None else dtype
    type_code(weight.dtype), type_code(dtype)
    row_stride(weight, "weight")
    check_ids(ids)
    check_device(weight, ids)
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(weight, ids, float(scale), dtype)
    return _lookup(weight, ids, float(scale), dtype)


@torch.no_grad()
def embedding_grad(grad, ids, num_rows, scale=1.0, dtype=None, out=None):
    """The lookup's gradient by itself: dw[v] = scale * sum of grad's rows whose id is v.

    grad [*ids.shape, D]; returns dw [num_rows, D] in `dtype` (default: grad's), zeros in rows that no
    id names.  With out [num_rows, D] (contiguous columns, rows that do not overlap) the sums are added
    to its named rows instead -- each row's sum and its old value are added in f32 and rounded once,
    the other rows are left as they are -- and out is returned."""
    type_code(grad.dtype)
    check_ids(ids)
    if grad.dim() < 1 or grad.shape[:-1] != ids.shape:
        raise ValueError(f"hgsr: grad {tuple(grad.shape)} does not hold one row per id of {tuple(ids.shape)}")
    num_rows, D = int(num_rows), grad.shape[-1]
    if num_rows < 0:
        raise ValueError("hgsr: num_rows is negative")
    if out is None:
        dtype = grad.dtype if dtype is None else dtype
        type_code(dtype)
        check_device(grad, ids)
        g = rows_view(grad, D, "grad") if D else grad
        return _grad(g, ids, torch.empty(num_rows, D, dtype=dtype, device=grad.device), float(scale), False)
    type_code(out.dtype)
    if tuple(out.shape) != (num_rows, D) or (dtype is not None and dtype != out.dtype):
        raise ValueError(f"hgsr: out is {tuple(out.shape)} of {out.dtype}, not {(num_rows, D)} of {dtype or 'its type'}")
    if row_stride(out, "out") < D:
        raise ValueError("hgsr: the rows of out overlap")
    check_device(grad, ids, out)
    g = rows_view(grad, D, "grad") if D else grad
    return _grad(g, ids, out, float(scale), True)


class Embedding(torch.nn.Module):
    """Learned rows, one per camera (reference scene/embedding.py:50-79): Embedding(in_dim, out_dim),
    called with ids; mean() is the average row.  The table is `embedding.weight`."""

    def __init__(self, in_dim, out_dim, scale=1.0, device=None, dtype=None):
        super().__init__()
        self.in_dim, self.out_dim, self.scale = int(in_dim), int(out_dim), float(scale)
        self.embedding = torch.nn.Embedding(self.in_dim, self.out_dim, device=device, dtype=dtype)

    def mean(self, dim=0):
        return self.embedding.weight.mean(dim)

    def forward(self, ids):
        return embedding(self.embedding.weight, ids, self.scale)
