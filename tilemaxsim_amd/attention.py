"""Attention over packed texts, with gradients: an encoder's layer over a batch without its padding.

Texts stand one behind another, as :func:`flash_maxsim_multi_doc` has its documents, and a
token sees its own text alone. No reference counterpart (the reference does not encode or
train).
"""
from __future__ import annotations

import math
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _check, _lib

WIDTHS = (32, 64, 96, 128)
MOST_STRIDE = 1 << 22  # elements between tokens that the kernels read in place


_pack = struct.Struct("@3P6q3P5q2dq").pack  # tms_attention


def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    """Elements between tokens, heads and elements; 0 for a single token or head, whose stride means nothing."""
    (tokens, heads, _), (token, head, one) = t.shape, t.stride()
    return token if tokens > 1 else 0, head if heads > 1 else 0, one


def _describe(q, k, v, offsets, prefix, slopes, scale, cap) -> bytes:
    T, H, D = q.shape
    qt, qh, _ = _strides(q)
    kt, kh, _ = _strides(k)
    vt, vh, _ = _strides(v)
    return _pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), qt, qh, kt, kh, vt, vh, offsets.data_ptr(),
                 0 if prefix is None else prefix.data_ptr(), 0 if slopes is None else slopes.data_ptr(), offsets.shape[0] - 1, T, H,
                 k.shape[1], D, scale, cap, _lib.DTYPE_CODES[q.dtype])


def _forward(q, k, v, offsets, prefix, slopes, scale, cap, train):
    lib = _lib.load()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    low = torch.empty_like(out) if train and q.dtype != torch.float32 else None
    stats = None
    if train or slopes is not None:
        stats = torch.empty(lib.tms_attention_stats(q.shape[0], q.shape[1], k.shape[1]), dtype=torch.float32, device=q.device)
    given = _describe(q, k, v, offsets, prefix, slopes, scale, cap)
    status = _lib.launch(q.device, lib.tms_packed_attention, given, out.data_ptr(), _lib.ptr(low), _lib.ptr(stats))
    if status:
        _lib.check(status)
    return out, low, stats


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, prefix, slopes, scale, cap):
        out, low, stats = _forward(q, k, v, offsets, prefix, slopes, scale, cap, True)
        ctx.save_for_backward(q, k, v, offsets, prefix, slopes, out, low, stats)
        ctx.args = scale, cap
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, offsets, prefix, slopes, out, low, stats = ctx.saved_tensors
        lib = _lib.load()
        grad = _check.aligned(grad)
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) if need else None
                      for x, need in zip((q, k, v), ctx.needs_input_grad))
        nbytes = lib.tms_attention_workspace_size(offsets.shape[0] - 1, *q.shape[:2], *k.shape[1:])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        given = _describe(q, k, v, offsets, prefix, slopes, *ctx.args)
        status = _lib.launch(q.device, lib.tms_packed_attention_grad, given, out.data_ptr(), _lib.ptr(low),
                             stats.data_ptr(), grad.data_ptr(), _lib.ptr(ws), nbytes, _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv))
        if status:
            _lib.check(status)
        return dq, dk, dv, None, None, None, None, None


def _rows(t: torch.Tensor) -> torch.Tensor:
    """As it is where the kernels read it so (whole rows of a head, at 16-byte steps), else a copy."""
    step = 16 // t.element_size()
    token, head, one = _strides(t)
    if one == 1 and token % step == 0 and head % step == 0 and token <= MOST_STRIDE and t.data_ptr() % 16 == 0:
        return t
    return _check.aligned(t)


def _integers(fn: str, name: str, t: torch.Tensor) -> None:
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise TypeError(f"{fn}: {name} must be an integer tensor (got {t.dtype})")


def _usual(q, k, v, offsets) -> bool:
    """Whether the tensors are what a model has in hand, one dtype on one GPU with int64 offsets there,
    and need none of the checks below (which cost a small call as much as its kernel)."""
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor) and isinstance(offsets, torch.Tensor)):
        return False
    if not (q.is_cuda and q.dtype is k.dtype and q.dtype is v.dtype and q.dtype in _lib.DTYPE_CODES and offsets.dtype is torch.int64
            and q.dim() == 3 and k.dim() == 3 and offsets.dim() == 1):
        return False
    (T, H, D), shape, dev = q.shape, k.shape, q.get_device()
    return (shape == v.shape and shape[0] == T and shape[2] == D and D in WIDTHS and H > 0 and shape[1] > 0 and H % shape[1] == 0
            and offsets.shape[0] > 0 and k.get_device() == dev and v.get_device() == dev and offsets.get_device() == dev)


def _checked(fn: str, q, k, v, offsets) -> None:
    for name, t in (("q", q), ("k", k), ("v", v), ("offsets", offsets)):
        _check.tensor(name, t)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"{fn}: q must be (T, H, D), k and v (T, KV, D), got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    T, H, D = q.shape
    if k.shape[1] == 0 or H == 0 or H % k.shape[1]:
        raise ValueError(f"{fn}: {H} query heads cannot share {k.shape[1]} heads of keys")
    if offsets.dim() != 1 or offsets.numel() == 0:
        raise ValueError(f"{fn}: offsets must be (B + 1,), got {tuple(offsets.shape)}")
    _integers(fn, "offsets", offsets)
    _check.embedding_dtype("q", q)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{fn}: q is {q.dtype}, k is {k.dtype}, v is {v.dtype}")
    if D not in WIDTHS:
        raise NotImplementedError(f"{fn}: heads of {', '.join(map(str, WIDTHS))} elements (got {D})")
    if offsets.device.type == "cpu" and (bool((offsets[1:] < offsets[:-1]).any()) or int(offsets[0]) < 0 or int(offsets[-1]) > T):
        raise ValueError(f"{fn}: offsets must ascend within [0, {T}]")


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
        scale: multiplies the products of q and k (1e-15 to 1e15; default ``1 / sqrt(D)``).
        cap: scores become ``cap * tanh(score / cap)`` (1e-15 to 1e15; None: as they are).
        slopes: (H,) float32: a score is lessened by ``slope * |i - j|`` for tokens i and j
            (after the cap). They have no gradient.

    Returns:
        (T, H, D) of q's dtype. Rows of no text are zero (as their gradients are); what stands
        there, in other texts and behind a prefix mask is not seen, NaN included.

    Scores, softmax and sums are fp32; probabilities and their gradients are rounded to the
    inputs' type between two products (backward, where texts are short, to two terms of it). Every sum has one order.
    """
    fn = "packed_attention"
    usual = _usual(q, k, v, offsets)
    if not usual:
        _checked(fn, q, k, v, offsets)
    _check.no_tangents(fn, (q, k, v))
    H, B = q.shape[1], offsets.shape[0] - 1
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    if not 1e-15 <= scale <= 1e15:
        raise ValueError(f"{fn}: scale must be from 1e-15 to 1e15 (got {scale})")
    if cap is not None and not 1e-15 <= (cap := float(cap)) <= 1e15:
        raise ValueError(f"{fn}: cap must be from 1e-15 to 1e15 (got {cap})")
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
        _check.no_tangents(fn, (slopes,))
    if not usual:
        for name, t in (("q", q), ("k", k), ("v", v)):
            _check.on_gpu(name, t)
        _check.same_device(q=q, k=k, v=v)
    dev = q.device
    for name, t in (("slopes", slopes), ("prefix", prefix), ("offsets", offsets)):  # the latter two may come from the host
        if isinstance(t, torch.Tensor) and t.device != dev and (t.is_cuda or name == "slopes"):
            raise ValueError(f"{fn}: {name} is on {t.device}, q on {dev}")
    if not usual or not offsets.is_contiguous():
        offsets = offsets.to(dev, torch.int64).contiguous()
    if isinstance(prefix, torch.Tensor):
        prefix = prefix.to(dev, torch.int64).contiguous()
    elif prefix is not None:
        prefix = torch.full((B,), prefix, dtype=torch.int64, device=dev)
    if slopes is not None:
        slopes = slopes.contiguous()
    q, k, v = _rows(q), _rows(k), _rows(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttention.apply(q, k, v, offsets, prefix, slopes, scale, cap or 0.0)
    return _forward(q, k, v, offsets, prefix, slopes, scale, cap or 0.0, False)[0]
