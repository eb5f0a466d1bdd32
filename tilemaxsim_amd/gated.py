"""The gated projection of a feed-forward block, with gradients: both projections, the activation
and the product of the two in one kernel. No reference counterpart (the reference does not
encode or train).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _check, _lib

FEW_TOKENS = 64  # up to which the forward pass needs no workspace, whatever its rows
_ACTIVATIONS = {"silu": _lib.TMS_ACT_SILU, "gelu": _lib.TMS_ACT_GELU, "gelu_tanh": _lib.TMS_ACT_GELU_TANH}


def _workspace(lib, N, d, F, code, backward, dev):
    if N <= FEW_TOKENS and not backward:
        return None, 0
    nbytes = lib.tms_gated_workspace_size(N, d, F, code, backward)
    return (torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None), nbytes


def _forward(x, w_gate, w_up, act):
    N, d = x.shape
    F = w_gate.shape[0]
    code = _lib.DTYPE_CODES[x.dtype]
    lib = _lib.load()
    h = x.new_empty(N, F)
    ws, nbytes = _workspace(lib, N, d, F, code, 0, x.device)
    status = _lib.launch(x.device, lib.tms_gated_linear, x.data_ptr(), N, d, w_gate.data_ptr(), w_up.data_ptr(), F, code, act,
                         _lib.ptr(ws), nbytes, h.data_ptr())
    if status:
        _lib.check(status)
    return h


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        ctx.save_for_backward(x, w_gate, w_up)
        ctx.act = act
        return _forward(x, w_gate, w_up, act)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, w_gate, w_up = ctx.saved_tensors
        N, d = x.shape
        F = w_gate.shape[0]
        make = torch.empty_like if N and F else torch.zeros_like
        dx, dg, du = (make(t) if need else None for t, need in zip((x, w_gate, w_up), ctx.needs_input_grad))
        lib = _lib.load()
        code = _lib.DTYPE_CODES[x.dtype]
        grad = _check.aligned(grad)
        ws, nbytes = _workspace(lib, N, d, F, code, 1, x.device)
        status = _lib.launch(x.device, lib.tms_gated_linear_grad, x.data_ptr(), N, d, w_gate.data_ptr(), w_up.data_ptr(), F, code,
                             ctx.act, grad.data_ptr(), _lib.ptr(ws), nbytes, _lib.ptr(dx), _lib.ptr(dg), _lib.ptr(du))
        if status:
            _lib.check(status)
        return dx, dg, du, None


def _usual(x, w_gate, w_up) -> bool:
    """Whether the tensors are what a model has in hand, contiguous ones of one dtype on one GPU, and
    need none of the checks below (which cost a small call as much as its kernel)."""
    if not (isinstance(x, torch.Tensor) and isinstance(w_gate, torch.Tensor) and isinstance(w_up, torch.Tensor)):
        return False
    if not (x.is_cuda and x.dtype is w_gate.dtype and x.dtype is w_up.dtype and x.dtype in _lib.DTYPE_CODES and x.dim() > 0):
        return False
    shape, dev = w_gate.shape, x.get_device()
    return (len(shape) == 2 and shape == w_up.shape and shape[1] == x.shape[-1] > 0 and w_gate.get_device() == dev
            and w_up.get_device() == dev)


def _checked(fn: str, x, w_gate, w_up) -> None:
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up)):
        _check.tensor(name, t)
    if w_gate.dim() != 2 or w_up.shape != w_gate.shape or x.dim() < 1 or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"{fn}: x must be (..., d), w_gate and w_up (F, d), got {tuple(x.shape)}, {tuple(w_gate.shape)} and "
                         f"{tuple(w_up.shape)}")
    if x.shape[-1] == 0:
        raise ValueError(f"{fn}: rows of no elements")
    _check.embedding_dtype("x", x)
    if w_gate.dtype != x.dtype or w_up.dtype != x.dtype:
        raise TypeError(f"{fn}: x is {x.dtype}, w_gate is {w_gate.dtype}, w_up is {w_up.dtype}")


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """``act(x @ w_gate.T) * (x @ w_up.T)``, differentiable in all three.

    Args:
        x: (..., d) hidden states, float16, bfloat16 or float32.
        w_gate, w_up: (F, d), of x's dtype (halves of one (2F, d) tensor are read in place).
        activation: "silu", "gelu" or "gelu_tanh" (gelu by its tanh formula).

    Returns:
        (..., F) of x's dtype.

    Both products, the activation and all sums are fp32, rounded once. The backward pass forms
    both products again instead of keeping them; the gradients of the two are rounded to the
    inputs' type (float32: three bf16 terms; up to 64 tokens: two terms) before the products that they go into.
    """
    fn = "gated_linear"
    usual = _usual(x, w_gate, w_up)
    if not usual:
        _checked(fn, x, w_gate, w_up)
    _check.no_tangents(fn, (x, w_gate, w_up))
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"{fn}: activation must be one of {', '.join(_ACTIVATIONS)} (got {activation!r})")
    if not usual:
        for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up)):
            _check.on_gpu(name, t)
        _check.same_device(x=x, w_gate=w_gate, w_up=w_up)
    flat = x.dim() == 2
    rows = _check.aligned(x if flat else x.reshape(x.numel() // x.shape[-1], x.shape[-1]))
    wg, wu = _check.aligned(w_gate), _check.aligned(w_up)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        h = _GatedLinear.apply(rows, wg, wu, act)
    else:
        h = _forward(rows, wg, wu, act)
    return h if flat else h.view(*x.shape[:-1], w_gate.shape[0])
