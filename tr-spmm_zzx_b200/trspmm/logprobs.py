"""Log probabilities of given classes, entropy and the best alternatives of rows of scores, with their gradient
(trs_logprobs, trs_logprobs_grad).

What the scores of a graph model are for: the loss of a node classifier is -logprobs of the labels, its answer the
alternatives; where links are predicted, a row holds the scores against all nodes.  The reference has no such operator
(its benchmarks end with the product, spmm/tr_csr_fp16/test_tr_csr_online.py:83-181).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .embedding import _check_out, _no_tangents, _overlap, _row_stride, _special_id, _type_code, _written

MAX_TOP = 32
_NO_IGNORE = -(1 << 63)


class ClassLogprobs(NamedTuple):
    """logprobs [n] (None without targets), entropy [n], top_logprobs [n, top] and top_ids [n, top] int32 (None for top = 0),
    stats [n, 2] (the row's largest score, the sum of exponentials relative to it); all but top_ids fp32."""
    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]
    stats: torch.Tensor


def _check(logits, targets, mask, scale, top):
    index = logits.get_device()
    if index < 0:
        raise ValueError("class_logprobs needs CUDA tensors (there is no CPU fallback)")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError("logits must be [n, classes] with at least one class")
    n, classes = logits.shape
    stride = classes if logits.is_contiguous() else _row_stride(logits, "logits")
    code = _type_code(logits.dtype, "logits")
    if targets is not None:
        if targets.dtype is not torch.int64 and targets.dtype is not torch.int32:
            raise TypeError("targets must be torch.int64 or torch.int32")
        if targets.shape != (n,) or targets.get_device() != index or not targets.is_contiguous():
            raise ValueError("targets must be contiguous [n] on the logits' device")
    mask_stride = 0
    if mask is not None:
        if mask.dtype is not torch.bool:
            raise TypeError("mask must be torch.bool")
        if mask.get_device() != index or mask.shape != (classes,) and mask.shape != (n, classes):
            raise ValueError("mask must be [classes] or [n, classes] on the logits' device")
        if mask.dim() == 2:
            mask_stride = _row_stride(mask, "mask")
        elif classes > 1 and mask.stride(0) != 1:
            raise ValueError("mask must be contiguous along the classes")
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale must be positive and finite")
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be 0 to {MAX_TOP}")
    return index, (logits.data_ptr(), code, n, classes, stride, None if targets is None else targets.data_ptr(),
                   1 if targets is not None and targets.dtype is torch.int64 else 0), \
        (None if mask is None else mask.data_ptr(), mask_stride, scale, top)


def _forward(logits, targets, top, mask, scale, ignore_id) -> ClassLogprobs:
    index, front, back = _check(logits, targets, mask, scale, top)
    n = logits.shape[0]
    if targets is None:
        logprobs, entropy = None, logits.new_empty(n, dtype=torch.float32)
    else:   # (an empty_like takes less time than an empty with a shape)
        logprobs, entropy = torch.empty_like(targets, dtype=torch.float32), torch.empty_like(targets, dtype=torch.float32)
    stats = entropy.new_empty((n, 2))
    top_logprobs = top_ids = None
    if top:
        top_logprobs = entropy.new_empty((n, top))
        top_ids = torch.empty_like(top_logprobs, dtype=torch.int32)
    _lib.launch(index, _lib.load().trs_logprobs, *front, _NO_IGNORE if ignore_id is None else _special_id(ignore_id, "ignore_id"), *back,
                None if logprobs is None else logprobs.data_ptr(), entropy.data_ptr(),
                None if top_logprobs is None else top_logprobs.data_ptr(), None if top_ids is None else top_ids.data_ptr(),
                stats.data_ptr())
    return ClassLogprobs(logprobs, entropy, top_logprobs, top_ids, stats)


def _launch_grad(index, front, back, ignore_id, top_ids, stats, entropy, g_logprobs, g_entropy, g_top, dx, dx_stride):
    _lib.launch(index, _lib.load().trs_logprobs_grad, *front, _NO_IGNORE if ignore_id is None else _special_id(ignore_id, "ignore_id"), *back,
                None if g_top is None else top_ids.data_ptr(), stats.data_ptr(), None if g_entropy is None else entropy.data_ptr(),
                None if g_logprobs is None else g_logprobs.data_ptr(), None if g_entropy is None else g_entropy.data_ptr(),
                None if g_top is None else g_top.data_ptr(), dx.data_ptr(), dx_stride)


class _LogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, mask, scale, ignore_id):
        r = _forward(logits, targets, top, mask, scale, ignore_id)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in (r.top_ids, r.stats) if t is not None])
        ctx.save_for_backward(logits, targets, mask, r.entropy, r.top_ids, r.stats)
        ctx.args = scale, ignore_id
        return tuple(r)

    @staticmethod
    def backward(ctx, g_logprobs, g_entropy, g_top, _ids, _stats):
        if torch.is_grad_enabled():   # under create_graph
            return _LogprobsFn.once(ctx, g_logprobs, g_entropy, g_top, _ids, _stats)
        if forward_ad._current_level >= 0:
            _no_tangents("the gradient of class_logprobs", g_logprobs, g_entropy, g_top)
        logits, targets, mask, entropy, top_ids, stats = ctx.saved_tensors
        scale, ignore_id = ctx.args
        if g_logprobs is None and g_entropy is None and g_top is None:
            return (None,) * 6
        top = 0 if g_top is None else g_top.shape[-1]
        index, front, back = _check(logits, targets, mask, scale, top)
        dx = torch.empty_like(logits, memory_format=torch.contiguous_format)
        _launch_grad(index, front, back, ignore_id, top_ids, stats, entropy, *[None if g is None else g.contiguous() for g in
                                                                              (g_logprobs, g_entropy, g_top)], dx, logits.shape[1])
        return dx, None, None, None, None, None

    once = torch.autograd.function.once_differentiable(lambda ctx, *g: _LogprobsFn.backward(ctx, *g))


def class_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, top: int = 0, mask: torch.Tensor | None = None,
                   scale: float = 1.0, ignore_id: int | None = None) -> ClassLogprobs:
    """Log probabilities of `targets`, entropies and the `top` best alternatives under softmax(scale * logits), row by row.

    logits: [n, classes] fp32, fp16 or bf16; rows may lie apart.  targets: [n] int64 or int32, or None; `ignore_id` marks rows without one (log
    probability 0, no gradient of it); a target outside the classes gives NaN.  mask: bool [classes] or [n, classes], True
    where a class may be chosen; what stands in masked places does not matter, and scores of -inf count as masked.  A row with nothing left has log probability
    -inf, entropy 0 and alternatives -1.  Alternatives (up to 32) descend by score, the lowest class first among equal ones.
    Computed in fp32, results are fp32 (top_ids int32).

    Differentiable in the logits through logprobs, entropy and top_logprobs (not through the choice of the alternatives).  Forward-mode
    differentiation is refused."""
    if forward_ad._current_level >= 0:
        _no_tangents("class_logprobs", logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return ClassLogprobs(*_LogprobsFn.apply(logits, targets, top, mask, scale, ignore_id))
    return _forward(logits, targets, top, mask, scale, ignore_id)


def class_logprobs_grad(logits: torch.Tensor, targets: torch.Tensor | None, result: ClassLogprobs,
                        g_logprobs: torch.Tensor | None = None, g_entropy: torch.Tensor | None = None,
                        g_top_logprobs: torch.Tensor | None = None, mask: torch.Tensor | None = None, scale: float = 1.0,
                        ignore_id: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of the logits, of their shape and type, from the gradients (fp32, contiguous) of what class_logprobs
    returned for the same arguments as `result` (its entropy is read where g_entropy is given, its top_ids where g_top_logprobs
    is, its stats always)."""
    if forward_ad._current_level >= 0:
        _no_tangents("class_logprobs_grad", logits, result.stats, result.entropy, g_logprobs, g_entropy, g_top_logprobs, out)
    if out is not None:
        _check_out("class_logprobs_grad", out)
    top = 0 if g_top_logprobs is None else g_top_logprobs.shape[-1]
    index, front, back = _check(logits, targets, mask, scale, top)
    n = logits.shape[0]
    if g_logprobs is not None and targets is None:
        raise ValueError("g_logprobs needs the targets")
    if g_top_logprobs is not None and result.top_ids is None:
        raise ValueError("g_top_logprobs needs the alternatives of the result")
    for t, shape, dtype in ((g_logprobs, (n,), torch.float32), (g_entropy, (n,), torch.float32),
                            (g_top_logprobs, (n, top), torch.float32),
                            (result.top_ids if top else None, (n, top), torch.int32),
                            (result.entropy if g_entropy is not None else None, (n,), torch.float32),
                            (result.stats, (n, 2), torch.float32)):
        if t is not None and (t.dtype is not dtype or t.shape != shape or t.get_device() != index or not t.is_contiguous()):
            raise ValueError("gradients and results must be contiguous fp32 (top_ids int32) of the result's shapes on the logits' device")
    dx_stride = logits.shape[1]
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    elif out.shape != logits.shape or out.dtype is not logits.dtype or out.get_device() != index:
        raise ValueError("out must have the logits' shape and type and be on their device")
    elif any(t is not None and _overlap(out, t) for t in (logits, targets, mask, g_logprobs, g_entropy, g_top_logprobs, result.entropy,
                                                          result.top_ids, result.stats)):
        raise ValueError("out may not overlap the logits or anything else that the call reads")
    else:
        dx_stride = _row_stride(out, "out")
        _written(out)

    _launch_grad(index, front, back, ignore_id, result.top_ids, result.stats, result.entropy, g_logprobs, g_entropy,
                 g_top_logprobs if top else None, out, dx_stride)
    return out
