"""Embedding lookup with scaling, and its gradient (trs_embedding, trs_embedding_grad).

The features of a graph whose nodes have none of their own are a learned table, looked up by id:
    out[i, :]  = scale * table[ids[i], :]
    grad[v, :] = scale * sum of dout[i, :] over the i with ids[i] = v
which are the products with the selection matrix of the ids and with its transpose.  The reference has neither (its
dataset classes draw random features, spmm/tr_csr_fp16/mdataset2_online.py:29-167).
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad

from . import _lib

TYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # TRS_TYPE_*
_NO_PADDING = -(1 << 63)


def _type_code(dtype, what: str) -> int:
    code = TYPE_CODES.get(dtype)
    if code is None:
        raise TypeError(f"{what} must be torch.float32, torch.float16 or torch.bfloat16")
    return code


def _row_stride(t: torch.Tensor, what: str) -> int:
    """Elements from one row to the next; rows may lie apart (a slice of a wider matrix) but not overlap."""
    rows, F = t.shape
    if F > 1 and t.stride(1) != 1 or rows > 1 and t.stride(0) < F:
        raise ValueError(f"{what} needs rows of neighbouring elements that do not overlap")
    return max(t.stride(0), F)


def _check_ids(ids: torch.Tensor, index: int) -> int:
    """1 for 64-bit ids, 0 for 32-bit ones."""
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise TypeError("ids must be torch.int64 or torch.int32")
    if ids.get_device() != index or not ids.is_contiguous():
        raise ValueError("ids must be contiguous and on the same CUDA device")
    return 1 if ids.dtype is torch.int64 else 0


def _special_id(value, what: str) -> int:
    """An id with a meaning of its own (the lowest of 64 bits tells the C entry that there is none)."""
    if not -(1 << 63) < value < 1 << 63:   # ctypes would cut it to 64 bits: another id
        raise ValueError(f"{what} must lie above -2^63 and below 2^63")
    return value


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory ranges of two strided matrices meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False

    def span(t):
        return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _no_tangents(what: str, *tensors) -> None:
    """Refuses tensors with a tangent: there is no forward-mode derivative, and the kernels would drop it in silence.  (Callers ask
    for the level first: outside one there are no tangents, and small calls notice every function.)"""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _written(out: torch.Tensor) -> None:
    """Tells autograd that the kernels write the caller's tensor: a graph that kept it raises in its backward pass."""
    torch.autograd.graph.increment_version(out)


def _check_out(what: str, out) -> None:
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} with out= is not differentiable: call it under torch.no_grad()")


def _lookup(table, ids, scale, padding_id, dtype, out):
    index = table.get_device()
    if index < 0:
        raise ValueError("embedding needs CUDA tensors (there is no CPU fallback)")
    if table.dim() != 2 or not table.numel():
        raise ValueError("the table must be [rows, F] with at least one row and one feature")
    wide = _check_ids(ids, index)
    rows, F = table.shape
    code = out_code = _type_code(table.dtype, "the table")
    stride, out_stride = F if table.is_contiguous() else _row_stride(table, "the table"), F
    if out is None:
        if dtype is None or dtype is table.dtype:
            out = table.new_empty((*ids.shape, F))
        else:
            out_code = _type_code(dtype, "the output")
            out = table.new_empty((*ids.shape, F), dtype=dtype)
    else:
        if out.shape != (*ids.shape, F) or out.get_device() != index or dtype is not None and out.dtype is not dtype:
            raise ValueError("out must be [*ids.shape, F] of the output type on the table's device")
        out_code = _type_code(out.dtype, "the output")
        if out.dim() == 2:
            out_stride = _row_stride(out, "out")
        elif not out.is_contiguous():
            raise ValueError("out must be contiguous unless ids is a vector")
        if _overlap(out, table) or _overlap(out, ids):
            raise ValueError("out may not overlap the table or the ids")
        _written(out)
    _lib.launch(index, _lib.load().trs_embedding, table.data_ptr(), code, rows, stride, ids.data_ptr(), wide, ids.numel(), F, scale,
                _NO_PADDING if padding_id is None else _special_id(padding_id, "padding_id"), out.data_ptr(), out_code, out_stride)
    return out


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, padding_id, dtype):
        ctx.save_for_backward(ids)
        ctx.args = table.shape[0], scale, padding_id, table.dtype
        return _lookup(table, ids, scale, padding_id, dtype, None)

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():   # under create_graph
            return _EmbeddingFn.once(ctx, dout)
        rows, scale, padding_id, dtype = ctx.args
        return embedding_grad(dout.contiguous(), ctx.saved_tensors[0], rows, scale, padding_id, dtype), None, None, None, None

    once = torch.autograd.function.once_differentiable(lambda ctx, dout: _EmbeddingFn.backward(ctx, dout))


def embedding(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding_id: int | None = None,
              out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """scale * table[ids], shape [*ids.shape, F], on the current stream.

    table: [rows, F] fp32, fp16 or bf16 (rows may lie apart).  ids: int64 or int32, any shape, contiguous; an id equal to
    `padding_id` gives zeros, one outside [0, rows) a row of NaN.  out_dtype: the table's type unless given - an fp32 table gives
    the fp16 features that the SpMM takes without a copy of the table.  `out` may be given instead (for a vector of ids its rows
    may lie apart).  Differentiable in the table where no `out` is given: the gradient is embedding_grad's, dense, in the
    table's type.  Forward-mode differentiation is refused."""
    if forward_ad._current_level >= 0:
        _no_tangents("embedding", table, out)
    if out is not None:
        _check_out("embedding", out)
    if table.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("embedding with out= is not differentiable: call it under torch.no_grad()")
        return _EmbeddingFn.apply(table, ids, scale, padding_id, out_dtype)
    return _lookup(table, ids, scale, padding_id, out_dtype, out)


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, n_rows: int, scale: float = 1.0, padding_id: int | None = None,
                   out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                   accumulate: bool = False) -> torch.Tensor:
    """The gradient of a table of `n_rows` rows from the gradient of the looked-up rows: [n_rows, F], row v the sum, times
    scale, of the rows of `grad` ([*ids.shape, F]) whose id is v.

    Ids are sorted within the call; sums are fp32 in an order that depends on the ids alone (the same bits every time), rounded
    once to out_dtype (the type of `grad` unless given).  Rows that no id names are zero.  With `accumulate` the sums
    are added to `out`, whose other rows stay as they are (micro-batches).  Padding ids and ids outside the table contribute
    nothing."""
    if forward_ad._current_level >= 0:
        _no_tangents("embedding_grad", grad, out)
    if out is not None:
        _check_out("embedding_grad", out)
    index = grad.get_device()
    if index < 0:
        raise ValueError("embedding_grad needs CUDA tensors (there is no CPU fallback)")
    wide = _check_ids(ids, index)
    if grad.dim() < 1 or grad.shape[:-1] != ids.shape or grad.shape[-1] < 1 or n_rows < 1:
        raise ValueError("grad must be [*ids.shape, F] with at least one feature, and the table have at least one row")
    F, n = grad.shape[-1], ids.numel()
    code = out_code = _type_code(grad.dtype, "the gradient")
    stride = out_stride = F
    if not grad.is_contiguous():
        if grad.dim() != 2:
            raise ValueError("the gradient must be contiguous unless ids is a vector")
        stride = _row_stride(grad, "the gradient")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs the out tensor to add to")
        if out_dtype is None or out_dtype is grad.dtype:
            out = grad.new_empty((n_rows, F))
        else:
            out_code = _type_code(out_dtype, "the output")
            out = grad.new_empty((n_rows, F), dtype=out_dtype)
    else:
        if out.shape != (n_rows, F) or out.get_device() != index or out_dtype is not None and out.dtype is not out_dtype:
            raise ValueError("out must be [n_rows, F] of the output type on the gradient's device")
        if _overlap(out, grad) or _overlap(out, ids):
            raise ValueError("out may not overlap the gradient or the ids")
        out_code, out_stride = _type_code(out.dtype, "the output"), _row_stride(out, "out")
        _written(out)
    lib, need = _lib.load(), C.c_size_t()
    _lib.check(lib.trs_embedding_grad_workspace_bytes(n, n_rows, F, C.byref(need)))
    # the workspace is this call's own: calls on several streams, and graphs, do not share one
    ws = grad.new_empty(need.value, dtype=torch.uint8) if need.value else None
    _lib.launch(index, lib.trs_embedding_grad, grad.data_ptr(), code, stride, ids.data_ptr(), wide, n, n_rows, F, scale,
                _NO_PADDING if padding_id is None else _special_id(padding_id, "padding_id"), out.data_ptr(), out_code, out_stride, 1 if accumulate else 0, None if ws is None else ws.data_ptr(), need.value)
    return out
