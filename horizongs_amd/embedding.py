"""Embedding lookup with scaling, and its gradient by sorted ids (csrc/embed.hip).

* `embedding(weight, ids, scale)`        out[..., :] = scale * weight[ids, :], differentiable
* `embedding_grad(grad, ids, num_rows)`  the gradient by itself, dense or added into a table's
* `Embedding`                            <- scene/embedding.py:50-79, the per-camera appearance
                                         rows that condition the colour head (decode.py)

Tables and rows may be float32, float16 or bfloat16; sums are f32, rounded once.  An id outside
[0, num_rows) (-1 by custom) is padding: its row is zeros and it takes no part in the gradient --
there is no host read that could raise.  Gradients are summed in an order that the ids, the sizes
and the types set, so they are the same bits on every run, wherever the tensors lie.  Forward-mode
derivatives and torch.jit.trace are refused.  There is no CPU path.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _native as N
from . import gradbuf

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


_IDS = {torch.int32: 0, torch.int64: 1}

# the calls behind torch.jit.is_tracing and torch.autograd.graph.increment_version (0.1 and 0.3 us less)
_is_tracing, increment_version = torch._C._is_tracing, torch._C._increment_version


def check_device(*ts):
    """The device number of tensors that all lie on one HIP device."""
    index = ts[0].get_device()
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError("hgsr: inputs must be HIP device tensors (no CPU fallback)")
        if t.get_device() != index:
            raise RuntimeError(f"hgsr: tensors on devices {index} and {t.get_device()}: one is needed")
    return index


def type_code(dtype):
    code = _TYPES.get(dtype)
    if code is None:
        raise ValueError(f"hgsr: float32, float16 or bfloat16 rows are needed, not {dtype}")
    return code


def row_stride(t, what):
    """Elements between the rows of a 2-D tensor whose columns are contiguous."""
    n, d = t.shape
    s0, s1 = t.stride()
    if s1 != 1 and d > 1 and n:
        raise ValueError(f"hgsr: the columns of {what} must be contiguous (stride {s1})")
    return s0 if n > 1 else d


def rows_view(t, dim, what):
    """[n, dim] view of a tensor's rows with contiguous columns, copied only if there is none."""
    if t.shape[-1] != dim:
        raise ValueError(f"hgsr: rows of {what} have {t.shape[-1]} columns, not {dim}")
    if t.dim() != 2:
        t = t.reshape(t.shape[:-1].numel(), dim)  # spelt out: rows may have no columns
    return t if dim == 1 or t.stride(1) == 1 else t.contiguous()


def check_ids(ids):
    """1 for int64 ids, 0 for int32."""
    is64 = _IDS.get(ids.dtype)
    if is64 is None:
        raise ValueError(f"hgsr: int32 or int64 ids are needed, not {ids.dtype}")
    return is64


def flat_ids(ids):
    return ids if ids.dim() == 1 else ids.reshape(-1)


def id_stride(flat):
    return flat.stride(0) if flat.shape[0] > 1 else 1


def refuse_trace():
    """torch.jit.trace would record the allocation of a result and not the call that fills it."""
    if _is_tracing():
        raise NotImplementedError("hgsr: calls on row tables cannot be traced")


def _recorded(t):
    """Whether a call on t has to go through its Function: for a gradient, or for a tangent (a dual tensor's
    primal may need no gradient, and torch.no_grad() does not switch tangents off), which a Function refuses."""
    return (t.requires_grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0


def _lookup(weight, stride, flat, shape, scale, dtype, index):
    V, D = weight.shape
    out = weight.new_empty((*shape, D), dtype=dtype)
    n = flat.shape[0]
    if n and D:
        N.call_on(index, "hgsr_embed_fwd", V, n, D, weight.data_ptr(), _TYPES[weight.dtype],
                  stride, flat.data_ptr(), _IDS[flat.dtype], id_stride(flat), scale,
                  out.data_ptr(), _TYPES[dtype])
    return out


def _grad(grad, flat, out, scale, index, added=None):
    """The sums in out, which is contiguous, or added to out, whose rows lie `added` elements apart."""
    V, D = out.shape
    accumulate = added is not None
    n = flat.shape[0]
    if V == 0 or D == 0 or (n == 0 and accumulate):
        return out
    ws_b = N.size_query("hgsr_embed_bwd_ws_bytes", V, n, D)
    ws = torch.empty(ws_b, dtype=torch.uint8, device=out.device) if ws_b else None
    N.call_on(index, "hgsr_embed_bwd", V, n, D, grad.data_ptr(), _TYPES[grad.dtype], row_stride(grad, "grad"),
              flat.data_ptr(), _IDS[flat.dtype], id_stride(flat), scale, out.data_ptr(), _TYPES[out.dtype],
              added if accumulate else D, accumulate, ws.data_ptr() if ws_b else None, ws_b)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, flat, shape, scale, dtype, index):
        ctx.save_for_backward(flat)
        ctx.args = weight.shape, weight.dtype, (weight.data_ptr(), weight.numel()), scale, index
        return _lookup(weight, row_stride(weight, "weight"), flat, shape, scale, dtype, index)

    @staticmethod
    def backward(ctx, g):
        flat, = ctx.saved_tensors
        shape, dtype, key, scale, index = ctx.args
        # create_graph: the gradient is linear in g, and its own gradient a lookup
        if torch.is_grad_enabled() or _recorded(g):
            return _EmbeddingGrad.apply(g, flat, shape, dtype, scale, index), None, None, None, None, None
        out = gradbuf.take(key, shape, dtype)  # in place in a DDP bucket when one is registered
        if out is None:
            out = g.new_empty(shape, dtype=dtype)
        return _grad(rows_view(g, shape[1], "grad"), flat, out, scale, index), None, None, None, None, None


class _EmbeddingGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g, flat, shape, dtype, scale, index):
        ctx.save_for_backward(flat)
        ctx.args = (g.shape, g.dtype, scale, index)
        return _grad(rows_view(g, shape[1], "grad"), flat, g.new_empty(shape, dtype=dtype), scale, index)

    @staticmethod
    def backward(ctx, gg):
        (flat,) = ctx.saved_tensors
        shape, dtype, scale, index = ctx.args
        gg = rows_view(gg, gg.shape[1], "the gradient's gradient")
        if torch.is_grad_enabled() or _recorded(gg):
            return _Embedding.apply(gg, flat, shape[:-1], scale, dtype, index), None, None, None, None, None
        return _lookup(gg, row_stride(gg, "weight"), flat, shape[:-1], scale, dtype, index), None, None, None, None, None


def embedding(weight, ids, scale=1.0, dtype=None):
    """scale * weight[ids]: weight [V, D] (any row stride, contiguous columns), ids int32 / int64 of
    any shape; returns [*ids.shape, D] in `dtype` (default: weight's).  The product is f32, rounded
    once.  Differentiable in weight; the gradient has weight's type and a row for each of its rows."""
    refuse_trace()
    if weight.dim() != 2:
        raise ValueError(f"hgsr: weight must be [rows, columns], not {tuple(weight.shape)}")
    type_code(weight.dtype)
    if dtype is None:
        dtype = weight.dtype
    else:
        type_code(dtype)
    stride = row_stride(weight, "weight")
    check_ids(ids)
    index = check_device(weight, ids)
    flat = flat_ids(ids)
    if _recorded(weight):
        return _Embedding.apply(weight, flat, ids.shape, float(scale), dtype, index)
    return _lookup(weight, stride, flat, ids.shape, float(scale), dtype, index)


def embedding_grad(grad, ids, num_rows, scale=1.0, dtype=None, out=None):
    """The lookup's gradient by itself: dw[v] = scale * sum of grad's rows whose id is v.

    grad [*ids.shape, D]; returns dw [num_rows, D] in `dtype` (default: grad's), zeros in rows that no
    id names, differentiable in grad.  With out [num_rows, D] (contiguous columns, rows that do not overlap) the sums are added
    to its named rows instead -- each row's sum and its old value are added in f32 and rounded once,
    the other rows are left as they are -- and out, which must not share memory with grad, is
    returned; nothing is differentiated through that."""
    refuse_trace()
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
        index = check_device(grad, ids)
        if _recorded(grad):
            return _EmbeddingGrad.apply(grad, flat_ids(ids), (num_rows, D), dtype, float(scale), index)
        out, added = grad.new_empty((num_rows, D), dtype=dtype), None
    else:
        type_code(out.dtype)
        if tuple(out.shape) != (num_rows, D) or (dtype is not None and dtype != out.dtype):
            raise ValueError(f"hgsr: out is {tuple(out.shape)} of {out.dtype}, not {(num_rows, D)} of "
                             f"{dtype or 'its type'}")
        added = row_stride(out, "out")
        if added < D:
            raise ValueError("hgsr: the rows of out overlap")
        if torch.is_grad_enabled() and (grad.requires_grad or out.requires_grad):
            raise NotImplementedError("hgsr: sums added to out are not differentiable (torch.no_grad())")
        if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (grad, out)):
            raise NotImplementedError("hgsr: sums added to out are not differentiable, in forward mode neither")
        index = check_device(grad, ids, out)
    _grad(rows_view(grad, D, "grad"), flat_ids(ids), out, float(scale), index, added)
    if added is not None and grad.numel():
        increment_version((out,))  # a backward that saved out as it was must not go on with it
    return out


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
