"""Attention over packed texts, with gradients: an encoder's layer over a batch without its padding.

Texts stand one behind another, as :func:`flash_maxsim_multi_doc` has its documents, and a
token sees its own text alone. No reference counterpart (the reference does not encode or
train).
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _check, _lib

WIDTHS = (32, 64, 96, 128)


class _Attention(ctypes.Structure):
    """tms_attention"""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v")]
                + [(n, ctypes.c_int64) for n in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head")]
                + [(n, ctypes.c_void_p) for n in ("offsets", "prefix", "slopes")]
                + [(n, ctypes.c_int64) for n in ("texts", "tokens", "heads", "kv_heads", "width")]
                + [("scale", ctypes.c_double), ("cap", ctypes.c_double), ("dtype", ctypes.c_int64)])


def _describe(q, k, v, offsets, prefix, slopes, scale, cap) -> _Attention:
    T, H, D = q.shape
    return _Attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:2], *k.stride()[:2], *v.stride()[:2],
                      offsets.data_ptr(), _lib.ptr(prefix), _lib.ptr(slopes), offsets.numel() - 1, T, H, k.shape[1], D, scale, cap,
                      _lib.dtype_code(q.dtype))


def _forward(q, k, v, offsets, prefix, slopes, scale, cap, train):
    lib = _lib.load()
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    low = torch.empty_like(out) if train and q.dtype != torch.float32 else None
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device) if train else None
    given = _describe(q, k, v, offsets, prefix, slopes, scale, cap)
    status = _lib.launch(q.device, lib.tms_packed_attention, ctypes.addressof(given), out.data_ptr(), _lib.ptr(low), _lib.ptr(lse))
    if status:
        _lib.check(status)
    return out, low, lse


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, prefix, slopes, scale, cap):
        out, low, lse = _forward(q, k, v, offsets, prefix, slopes, scale, cap, True)
        ctx.save_for_backward(q, k, v, offsets, prefix, slopes, out, low, lse)
        ctx.args = scale, cap
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, offsets, prefix, slopes, out, low, lse = ctx.saved_tensors
        lib = _lib.load()
        grad = _check.aligned(grad)
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) if need else None
                      for x, need in zip((q, k, v), ctx.needs_input_grad))
        nbytes = lib.tms_attention_workspace_size(q.shape[0], q.shape[1])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        given = _describe(q, k, v, offsets, prefix, slopes, *ctx.args)
        status = _lib.launch(q.device, lib.tms_packed_attention_grad, ctypes.addressof(given), out.data_ptr(), _lib.ptr(low),
                             lse.data_ptr(), grad.data_ptr(), _lib.ptr(ws), nbytes, _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv))
        if status:
            _lib.check(status)
        return dq, dk, dv, None, None, None, None, None


def _rows(t: torch.Tensor) -> torch.Tensor:
    """As it is where the kernels read it so (whole rows of a head, at 16-byte steps), else a copy."""
    step = 16 // t.element_size()
    if t.stride(2) == 1 and t.stride(0) % step == 0 and t.stride(1) % step == 0 and t.data_ptr() % 16 == 0:
        return t
    return _check.aligned(t)


def _integers(fn: str, name: str, t: torch.Tensor) -> None:
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise TypeError(f"{fn}: {name} must be an integer tensor (got {t.dtype})")


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, *, prefix=None,
                     scale: float | None = None, cap: float | None = None, slopes: torch.Tensor | None = None) -> torch.Tensor:
    """Softmax attention of packed texts, each within itself; differentiable in q, k and v.

    Args:
        q: (T, H, D) queries of all texts' tokens, float16, bfloat16 or float32; D 32, 64, 96 or
            128. A view of a wider projection is read in place.
        k, v: (T, KV, D) of q's dtype, H a multiple of KV: query head h reads head h // (H // KV).
        offsets: (B + 1,) ascending integers within [0, T]: text b is tokens offsets[b] up to
            offsets[b + 1]. Empty texts are allowed. On the CPU they are checked, and copied; on
            the GPU they are taken as they are, without a wait (where they descend, some rows
            come out undefined).
        prefix: None (a token attends to its whole text), or one integer a text, (B,) or a number
            for all: its first ``prefix`` tokens are seen by all of it, the others by themselves and
            those behind them. 0: causal.
        scale: multiplies the products of q and k (positive; default ``1 / sqrt(D)``).
        cap: scores become ``cap * tanh(score / cap)`` (positive; None: as they are).
        slopes: (H,) float32: a score is lessened by ``slope * |i - j|`` for tokens i and j
            (after the cap). They have no gradient.

    Returns:
        (T, H, D) of q's dtype. Rows of no text are zero (as their gradients are); what stands
        there, and in other texts, is not seen, NaN included.

    Scores, softmax and sums are fp32; probabilities and their gradients are rounded to the
    inputs' type between two products. Every sum has one order.
    """
    fn = "packed_attention"
    for name, t in (("q", q), ("k", k), ("v", v), ("offsets", offsets)):
        _check.tensor(name, t)
    _check.no_tangents(fn, (q, k, v))
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"{fn}: q must be (T, H, D), k and v (T, KV, D), got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    T, H, D = q.shape
    if k.shape[1] == 0 or H == 0 or H % k.shape[1]:
        raise ValueError(f"{fn}: {H} query heads cannot share {k.shape[1]} heads of keys")
    if offsets.dim() != 1 or offsets.numel() == 0:
        raise ValueError(f"{fn}: offsets must be (B + 1,), got {tuple(offsets.shape)}")
    _integers(fn, "offsets", offsets)
    B = offsets.numel() - 1
    _check.embedding_dtype("q", q)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{fn}: q is {q.dtype}, k is {k.dtype}, v is {v.dtype}")
    if D not in WIDTHS:
        raise NotImplementedError(f"{fn}: heads of {', '.join(map(str, WIDTHS))} elements (got {D})")
    scale = 1 / math.sqrt(D) if scale is None else float(scale)
    if not 0 < scale < 1e30:
        raise ValueError(f"{fn}: scale must be positive and finite (got {scale})")
    if cap is not None and not 0 < (cap := float(cap)) < 1e30:
        raise ValueError(f"{fn}: cap must be positive and finite (got {cap})")
    if isinstance(prefix, torch.Tensor):
        _integers(fn, "prefix", prefix)
        if tuple(prefix.shape) != (B,):
            raise ValueError(f"{fn}: prefix must be ({B},), one a text, got {tuple(prefix.shape)}")
    elif prefix is not None and (isinstance(prefix, bool) or not isinstance(prefix, int)):
        raise TypeError(f"{fn}: prefix must be an integer or a tensor of them (got {type(prefix).__name__})")
    if slopes is not None:
        _check.tensor("slopes", slopes)
        if tuple(slopes.shape) != (H,) or slopes.dtype != torch.float32:
            raise ValueError(f"{fn}: slopes must be ({H},) float32, got {tuple(slopes.shape)} {slopes.dtype}")
        if slopes.requires_grad:
            raise NotImplementedError(f"{fn}: a gradient of the slopes")
    if offsets.device.type == "cpu":
        if bool((offsets[1:] < offsets[:-1]).any()) or int(offsets[0]) < 0 or int(offsets[-1]) > T:
            raise ValueError(f"{fn}: offsets must ascend within [0, {T}]")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check.on_gpu(name, t)
    given = {"q": q, "k": k, "v": v}
    if slopes is not None:
        given["slopes"] = slopes
    if isinstance(prefix, torch.Tensor) and prefix.device.type != "cpu":
        given["prefix"] = prefix
    if offsets.device.type != "cpu":
        given["offsets"] = offsets
    dev = _check.same_device(**given)
    offsets = offsets.to(dev, torch.int64).contiguous()
    if isinstance(prefix, torch.Tensor):
        prefix = prefix.to(dev, torch.int64).contiguous()
    elif prefix is not None:
        prefix = torch.full((B,), prefix, dtype=torch.int64, device=dev)
    slopes = None if slopes is None else slopes.contiguous()
    q, k, v = _rows(q), _rows(k), _rows(v)
    args = (q, k, v, offsets, prefix, slopes, scale, cap or 0.0)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttention.apply(*args)
    return _forward(*args, False)[0]
