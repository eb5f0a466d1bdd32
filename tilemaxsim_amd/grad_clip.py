"""The global gradient norm, and clipping to it, over any number of tensors in a few launches.

The norm stays on the GPU: nothing waits for it, and a training step that clips can be
captured into a HIP graph. No reference counterpart (the reference does not train).
"""
from __future__ import annotations

import ctypes
import math
import operator
from array import array

import torch

from . import _check, _lib, _overlap

_requires_grad = operator.attrgetter("requires_grad")
_NORMS = {2.0: _lib.TMS_NORM_2, math.inf: _lib.TMS_NORM_INF}


def _norm_type(fn: str, p) -> int:
    code = _NORMS.get(float(p))
    if code is None:
        raise NotImplementedError(f"{fn}: norm_type must be 2 or inf (got {p})")
    return code


def _not_parameters(fn: str, ts: list) -> None:
    if any(t.is_leaf and t.requires_grad for t in ts):
        raise ValueError(f"{fn}: got parameters (leaves that require a gradient); pass their gradients, [p.grad for p in parameters]")


def _no_graph(fn: str, ts: list) -> None:
    if torch.is_grad_enabled():
        raise RuntimeError(f"{fn}: the norm is not differentiable, and a tensor requires a gradient; detach the tensors, or call it under torch.no_grad()")


def _list(fn: str, tensors, of_a_graph=None) -> tuple[list, list]:
    """The tensors, and their dtypes; where any requires a gradient, `of_a_graph` may refuse them."""
    ts = [tensors] if isinstance(tensors, torch.Tensor) else [t for t in tensors if t is not None]
    # a model's hundreds of tensors are few types, dtypes and devices: only a mixture is looked at singly
    if not all(issubclass(k, torch.Tensor) for k in set(map(type, ts))):
        bad = next(t for t in ts if not isinstance(t, torch.Tensor))
        raise TypeError(f"{fn}: expected tensors, got {type(bad).__name__}")
    _check.no_tangents(fn, ts)
    kinds = [t.dtype for t in ts]
    for kind in set(kinds):
        if kind not in _lib.DTYPE_CODES:
            raise TypeError(f"{fn}: gradients must be float16, bfloat16 or float32 (got {kind})")
    if of_a_graph is not None and True in map(_requires_grad, ts):
        of_a_graph(fn, ts)
    return ts, kinds


_contiguous = torch.Tensor.is_contiguous


def _on_one_gpu(fn: str, ts: list) -> None:
    on = {t.get_device() for t in ts}  # -1: not on a GPU
    if len(on) > 1 or -1 in on:
        for t in ts:
            if not t.is_cuda:
                raise ValueError(f"{fn}: gradients must be on a ROCm GPU device (got {t.device}); tilemaxsim_amd has no CPU path")
            if t.device != ts[0].device:
                raise ValueError(f"{fn}: all gradients must be on one device; got {t.device} and {ts[0].device}")


def _codes(kinds: list) -> list:
    if kinds.count(kinds[0]) == len(kinds):
        return [_lib.DTYPE_CODES[kinds[0]]] * len(kinds)
    return [_lib.DTYPE_CODES[k] for k in kinds]


def _table(src: list, src_kinds: list, dst: list, dst_kinds: list) -> array:
    """tms_grad_tensor entries: two addresses, the size, and both dtypes in one word."""
    words = array("q", bytes(32 * len(src)))
    from_ = array("q", [t.data_ptr() for t in src])
    codes = _codes(src_kinds)
    words[0::4] = from_
    words[1::4] = from_ if dst is src else array("q", [t.data_ptr() for t in dst])
    words[2::4] = array("q", [t.numel() for t in src])
    words[3::4] = array("q", [s | d << 32 for s, d in zip(codes, codes if dst is src else _codes(dst_kinds))])
    return words


def _same(t: torch.Tensor, o: torch.Tensor) -> bool:
    """Whether a gradient and its tensor in `out` are the same elements."""
    return t is o or (t.data_ptr() == o.data_ptr() and t.dtype == o.dtype
                      and all(n < 2 or a == b for n, a, b in zip(t.shape, t.stride(), o.stride())))


def _workspace(lib, count: int, dev: torch.device) -> torch.Tensor:
    return torch.empty(lib.tms_grad_workspace_size(count) // 8, dtype=torch.float64, device=dev)


def grad_norm(tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all gradients taken as one vector: a float32 scalar on their device.

    Args:
        tensors: gradients (float16, bfloat16 or float32, any mix, one device); None entries
            are passed over, as parameters without a gradient leave them. The norm has no
            gradient of its own: with gradients enabled, tensors that require one are
            refused (RuntimeError).
        norm_type: 2.0, or ``inf`` for the largest absolute value.
    """
    code = _norm_type("grad_norm", norm_type)
    ts, kinds = _list("grad_norm", tensors, _no_graph)
    _on_one_gpu("grad_norm", ts)
    ts = [t if t.is_contiguous() else t.contiguous() for t in ts]
    if not ts:
        return torch.zeros(())
    dev = ts[0].device
    lib = _lib.load()
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = _workspace(lib, len(ts), dev)
    table = _table(ts, kinds, ts, kinds)
    status = _lib.launch(dev, lib.tms_grad_norm, table.buffer_info()[0], len(ts), code, ws.data_ptr(), 8 * ws.numel(),
                         norm.data_ptr())
    if status:
        _lib.check(status)
    return norm


@torch.no_grad()
def clip_grad_norm_(tensors, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    out=None) -> torch.Tensor:
    """Scale all gradients by ``min(1, max_norm / (norm + 1e-6))``, their norm taken together.

    Args:
        tensors: as for :func:`grad_norm`; changed in place, unless ``out`` is given. The
            gradients, not the parameters (a leaf that requires a gradient is refused), and
            no two that share memory: a tied weight's gradient is listed once (ValueError
            otherwise).
        max_norm: the norm to clip to (at least 0).
        norm_type: 2.0 or ``inf``.
        error_if_nonfinite: wait for the norm, and raise RuntimeError on a NaN or infinite
            one, before anything is scaled. Without it such a norm goes into the factor
            (an infinite one gives 0, NaN stays NaN), and nothing waits.
        out: tensors of the same sizes, one for each of ``tensors``, that take the scaled
            gradients (in their own dtype: bf16 gradients into an optimizer's fp32 ones). None
            may share memory with another one or with a gradient other than its own.

    Returns:
        The norm before clipping, a float32 scalar on the gradients' device.
    """
    fn = "clip_grad_norm_"
    code = _norm_type(fn, norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"{fn}: max_norm must be at least 0 (got {max_norm})")
    if out is None:
        ts, kinds = to, into = _list(fn, tensors, _not_parameters)
        _on_one_gpu(fn, ts)
    else:
        pairs_in = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        pairs_out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(pairs_in) != len(pairs_out):
            raise ValueError(f"{fn}: {len(pairs_in)} gradients and {len(pairs_out)} tensors in out")
        kept = [(t, o) for t, o in zip(pairs_in, pairs_out) if t is not None]
        ts, kinds = _list(fn, [t for t, _ in kept], _not_parameters)
        to, into = _list(fn, [o for _, o in kept], _not_parameters)
        if len(to) != len(ts):
            raise ValueError(f"{fn}: out has None in the place of a gradient's tensor")
        for t, o in zip(ts, to):
            if t.shape != o.shape:
                raise ValueError(f"{fn}: a gradient is {tuple(t.shape)}, its tensor in out {tuple(o.shape)}")
        _on_one_gpu(fn, ts)
        _on_one_gpu(fn, to)
        if to and to[0].device != ts[0].device:
            raise ValueError(f"{fn}: gradients are on {ts[0].device}, out is on {to[0].device}")
    if not ts:
        return torch.zeros(())
    if error_if_nonfinite and not bool(torch.isfinite(norm := grad_norm(ts, norm_type))):
        raise RuntimeError(f"{fn}: the norm of the gradients is {norm.item()}; they are left as they are")
    dev = ts[0].device
    lib = _lib.load()
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = _workspace(lib, len(ts), dev)
    src = ts if all(map(_contiguous, ts)) else [t if t.is_contiguous() else t.contiguous() for t in ts]
    if to is ts:
        dst = src
    else:
        dst = to if all(map(_contiguous, to)) else [o if o.is_contiguous() else torch.empty_like(o, memory_format=torch.contiguous_format) for o in to]
    copies = [] if dst is to else [(o, d) for o, d in zip(to, dst) if o is not d]  # strided tensors' own elements
    if copies or src is not ts:  # contiguous ones the library looks over
        _overlap.apart(fn, to, [t for t, o in zip(ts, to) if not _same(t, o)])
    table = _table(src, kinds, dst, into)
    limit = ctypes.c_double(max_norm)
    status = _lib.launch(dev, lib.tms_grad_clip, table.buffer_info()[0], len(src), code, ctypes.addressof(limit),
                         ws.data_ptr(), 8 * ws.numel(), norm.data_ptr())
    if status:
        _lib.check(status)
    for o, d in copies:
        o.copy_(d)
    torch.autograd.graph.increment_version([o for o in to if not o.is_inference()])
    return norm
