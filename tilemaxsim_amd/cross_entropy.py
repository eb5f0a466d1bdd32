"""Softmax cross entropy over a large vocabulary, from the hidden states and the vocabulary's
weights, with gradients and without the logits.

The same loss trains a masked-token head (hidden states against the token embeddings) and a
one-vector retriever (query vectors against passage vectors, every other passage a negative,
``scale`` the inverse temperature). No reference counterpart (the reference does not train).
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _check, _lib

_REDUCTIONS = {"none": _lib.TMS_REDUCE_NONE, "sum": _lib.TMS_REDUCE_SUM, "mean": _lib.TMS_REDUCE_MEAN}


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, and at an address the kernels' 16-byte loads take."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _workspace(lib, N, d, V, code, backward, dev):
    nbytes = lib.tms_lce_workspace_size(N, d, V, code, backward)
    return (torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None), nbytes


def _forward(H, W, target, scale, ignore_index, reduction):
    N, d = H.shape
    V = W.shape[0]
    code = _lib.dtype_code(H.dtype)
    lib = _lib.load()
    loss = torch.empty(N if reduction == _lib.TMS_REDUCE_NONE else (), dtype=torch.float32, device=H.device)
    stats = torch.empty(lib.tms_lce_stats(N), dtype=torch.float32, device=H.device)
    ws, nbytes = _workspace(lib, N, d, V, code, 0, H.device)
    factor = ctypes.c_double(scale)
    status = _lib.launch(H.device, lib.tms_linear_cross_entropy, H.data_ptr(), N, d, W.data_ptr(), V, code, target.data_ptr(),
                         ignore_index, ctypes.addressof(factor), reduction, _lib.ptr(ws), nbytes, loss.data_ptr(),
                         stats.data_ptr())
    if status:
        _lib.check(status)
    return loss, stats


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, H, W, target, scale, ignore_index, reduction):
        loss, stats = _forward(H, W, target, scale, ignore_index, reduction)
        ctx.save_for_backward(H, W, target, stats)
        ctx.args = scale, ignore_index, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        H, W, target, stats = ctx.saved_tensors
        scale, ignore_index, reduction = ctx.args
        N, d = H.shape
        V = W.shape[0]
        want_h, want_w = ctx.needs_input_grad[:2]
        if N == 0:
            return (torch.zeros_like(H) if want_h else None, torch.zeros_like(W) if want_w else None) + (None,) * 4
        dH = torch.empty_like(H) if want_h else None
        dW = torch.empty_like(W) if want_w else None
        lib = _lib.load()
        code = _lib.dtype_code(H.dtype)
        grad = grad.contiguous()
        ws, nbytes = _workspace(lib, N, d, V, code, 1, H.device)
        factor = ctypes.c_double(scale)
        status = _lib.launch(H.device, lib.tms_linear_cross_entropy_grad, H.data_ptr(), N, d, W.data_ptr(), V, code,
                             target.data_ptr(), ignore_index, ctypes.addressof(factor), reduction, stats.data_ptr(),
                             grad.data_ptr(), _lib.ptr(ws), nbytes, _lib.ptr(dH), _lib.ptr(dW))
        if status:
            _lib.check(status)
        return dH, dW, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, scale: float = 1.0,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``softmax(scale * hidden @ weight.T)`` against ``target``, as
    ``torch.nn.functional.cross_entropy`` of those logits gives it, without forming them in
    memory; differentiable in ``hidden`` and ``weight``.

    Args:
        hidden: (..., d) hidden states or query vectors, float16, bfloat16 or float32.
        weight: (V, d), of hidden's dtype: token embeddings, or passage vectors.
        target: (...) integers in [0, V), or ``ignore_index``. Rows with that have loss 0
            and no gradient, and what stands in them is not seen by the others. A target
            outside the vocabulary gives NaN, in its row's loss and in the gradients.
        scale: multiplies the logits (positive).
        reduction: "mean" over the rows that are not ignored (NaN if there are none),
            "sum", or "none".

    Returns:
        float32: a scalar, or a tensor of target's shape.

    Logits, the softmax's statistics and all sums are fp32; the backward pass holds the
    softmax of one piece of the vocabulary at a time, in the inputs' type (three bf16 terms
    for float32).
    """
    fn = "linear_cross_entropy"
    _check.tensor("hidden", hidden)
    _check.tensor("weight", weight)
    _check.tensor("target", target)
    _check.no_tangents(fn, (hidden, weight))
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{fn}: hidden must be (..., d) and weight (V, d), got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"{fn}: target must be {tuple(hidden.shape[:-1])}, got {tuple(target.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{fn}: reduction must be one of {', '.join(_REDUCTIONS)} (got {reduction!r})")
    scale = float(scale)
    if not 0 < scale < 1e30:
        raise ValueError(f"{fn}: scale must be positive and finite (got {scale})")
    if target.is_floating_point() or target.is_complex() or target.dtype == torch.bool:
        raise TypeError(f"{fn}: target must be an integer tensor (got {target.dtype})")
    _check.embedding_dtype("hidden", hidden)
    if weight.dtype != hidden.dtype:
        raise TypeError(f"{fn}: hidden is {hidden.dtype}, weight is {weight.dtype}")
    if weight.shape[0] == 0 and target.numel():
        raise ValueError(f"{fn}: an empty vocabulary")
    _check.on_gpu("hidden", hidden)
    _check.on_gpu("weight", weight)
    _check.on_gpu("target", target)
    _check.same_device(hidden=hidden, weight=weight, target=target)
    H, W = _aligned(hidden.reshape(target.numel(), hidden.shape[-1])), _aligned(weight)
    t = target.reshape(-1).to(torch.int64).contiguous()
    code = _REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (H.requires_grad or W.requires_grad):
        loss = _LinearCrossEntropy.apply(H, W, t, scale, int(ignore_index), code)
    else:
        loss = _forward(H, W, t, scale, int(ignore_index), code)[0]
    return loss.view(target.shape) if reduction == "none" else loss
