"""An AdamW step over any number of tensors in a few launches, with states of 32 or 8 bits.

Steps are counted on the GPU and the norm that clips is read there: nothing waits, and a
training step that ends in it can be captured into a HIP graph. No reference counterpart (the
reference does not train).
"""
from __future__ import annotations

import math
import struct
from array import array

import torch

from . import _check, _lib, _overlap

BLOCK = _lib.TMS_ADAMW_BLOCK


_pack = struct.Struct("@8P3q6d").pack  # tms_adamw
_pointer, _contiguous = torch.Tensor.data_ptr, torch.Tensor.is_contiguous


class AdamWState:
    """What :func:`adamw_` keeps between steps: the running means of the gradients and of their
    squares, and each tensor's count of steps.

    Args:
        params: the parameters, in the order in which ``adamw_`` gets them; on one GPU.
        bits: 32 (floats), or 8: a byte each, in blocks of 128 elements that share an exponent (a
            byte more a block).

    Attributes:
        m, v: the states of all tensors, flat: tensor i's begin at ``places[i]``, a multiple of 128, in
            the order of its elements. float32, or uint8 codes.
        m_exp, v_exp: with 8 bits the blocks' exponents, uint8; else None.
        steps: int64, one a tensor, on the GPU.
    """

    def __init__(self, params, bits: int = 32):
        fn = "AdamWState"
        ts = [params] if isinstance(params, torch.Tensor) else list(params)
        if bits not in (8, 32):
            raise NotImplementedError(f"{fn}: states of 8 or 32 bits (got {bits})")
        if not ts:
            raise ValueError(f"{fn}: no parameters")
        for t in ts:
            _check.tensor("a parameter", t)
            _check.embedding_dtype("a parameter", t)
        for t in ts:
            _check.on_gpu("a parameter", t)
            if t.device != ts[0].device:
                raise ValueError(f"{fn}: all parameters must be on one device; got {t.device} and {ts[0].device}")
        self.bits = bits
        self.shapes = [tuple(t.shape) for t in ts]
        self.sizes = [math.prod(s) for s in self.shapes]
        self.places, at = [], 0
        for n in self.sizes:
            self.places.append(at)
            at += -(-n // BLOCK) * BLOCK
        self.size = at
        dev, kind = ts[0].device, torch.float32 if bits == 32 else torch.uint8
        self.m, self.v = (torch.zeros(at, dtype=kind, device=dev) for _ in range(2))
        self.m_exp, self.v_exp = (torch.zeros(at // BLOCK, dtype=torch.uint8, device=dev) if bits == 8 else None for _ in range(2))
        self.steps = torch.zeros(len(ts), dtype=torch.int64, device=dev)

    def _tensors(self) -> dict:
        named = {"steps": self.steps, "m": self.m, "v": self.v}
        return named if self.bits == 32 else {**named, "m_exp": self.m_exp, "v_exp": self.v_exp}

    def state_dict(self) -> dict:
        """The state's tensors by name (not copies)."""
        return self._tensors()

    def load_state_dict(self, tensors: dict) -> None:
        """Takes over (as copies) what ``state_dict`` of a state of the same parameters and bits gave."""
        mine = self._tensors()
        if set(tensors) != set(mine):
            raise ValueError(f"AdamWState: expected {', '.join(mine)}, got {', '.join(map(str, tensors))}")
        for name, t in mine.items():
            _check.tensor(name, tensors[name])
            if tensors[name].shape != t.shape or tensors[name].dtype != t.dtype:
                raise ValueError(f"AdamWState: {name} must be {tuple(t.shape)} {t.dtype}, got {tuple(tensors[name].shape)} {tensors[name].dtype}")
        for name, t in mine.items():
            t.copy_(tensors[name])

    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The running means of gradients and squares as float32, in the states' places: the
        states themselves with 32 bits, the numbers that they stand for with 8."""
        if self.bits == 32:
            return self.m, self.v
        mean, square = (torch.empty(self.size, dtype=torch.float32, device=self.m.device) for _ in range(2))
        status = _lib.launch(self.m.device, _lib.load().tms_adamw_moments, self.m.data_ptr(), self.m_exp.data_ptr(), self.v.data_ptr(),
                             self.v_exp.data_ptr(), self.size, mean.data_ptr(), square.data_ptr())
        if status:
            _lib.check(status)
        return mean, square

    def views(self, flat: torch.Tensor) -> list:
        """A flat tensor of the states' places (``moments()``, or ``m``) as one view a parameter, of its shape."""
        return [flat[a:a + n].view(s) for a, n, s in zip(self.places, self.sizes, self.shapes)]


def _scalar(fn: str, name: str, t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    if t.numel() != 1 or t.dtype != torch.float32:
        raise ValueError(f"{fn}: {name} must be one float32 number, got {tuple(t.shape)} {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{fn}: {name} is on {t.device}, the parameters are on {dev}")
    return t.detach()


def _kinds(fn: str, name: str, ts: list, dev: torch.device) -> list:
    """The tensors' C dtype codes; they have to be floating-point tensors on `dev`."""
    if not all(issubclass(k, torch.Tensor) for k in set(map(type, ts))):
        bad = next(t for t in ts if not isinstance(t, torch.Tensor))
        raise TypeError(f"{fn}: {name} must be tensors, got {type(bad).__name__}")
    try:
        kinds = [_lib.DTYPE_CODES[t.dtype] for t in ts]
    except KeyError as e:
        raise TypeError(f"{fn}: {name} must be float16, bfloat16 or float32 (got {e.args[0]})") from None
    if set(map(torch.Tensor.get_device, ts)) - {dev.index}:
        bad = next(t for t in ts if t.device != dev)
        raise ValueError(f"{fn}: {name} must be on {dev}, where the states are (got {bad.device})")
    return kinds


def _shapes_match(fn: str, name: str, ts: list, shapes: list) -> None:
    if [t.shape for t in ts] != shapes:  # torch.Size is a tuple
        i = next(i for i, (t, s) in enumerate(zip(ts, shapes)) if tuple(t.shape) != s)
        raise ValueError(f"{fn}: {name}[{i}] is {tuple(ts[i].shape)}, the states are for {shapes[i]}")


@torch.no_grad()
def adamw_(params, grads, state: AdamWState, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, *,
           norm: torch.Tensor | None = None, max_norm: float | None = None, copies=None) -> None:
    """One AdamW step, in place: ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``,
    ``p = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)``, all in float32.

    Args:
        params: float32, float16 or bfloat16 (rounded to their type after the step: a small step may not
            move them; float32 ones with ``copies`` do not have that). No two may share memory, nor elements of one.
        grads: one for each parameter, of its shape, in any of those types; None: the parameter is left
            as it is, and so are its states and its count.
        state: an :class:`AdamWState` of these parameters; its counts are raised by this call.
        lr: a number, or a float32 tensor of one on the parameters' GPU, which is read there (a captured
            step then follows it from replay to replay).
        norm, max_norm: a norm of the gradients, as :func:`grad_norm` returns it, and what to clip it
            to: gradients count ``min(1, max_norm / (norm + 1e-6))`` times, as :func:`clip_grad_norm_`
            would have scaled them. They are not changed.
        copies: tensors of the parameters' shapes that take the new parameters in their own dtype (the
            16-bit weights that the next pass reads), or None in the place of one.

    NaN or infinite gradients (or norms) go into the parameters and states as the formulas say; in 8 bits a
    state that is not finite is kept as NaN.
    """
    fn = "adamw_"
    ps = [params] if isinstance(params, torch.Tensor) else list(params)
    gs = [grads] if grads is None or isinstance(grads, torch.Tensor) else list(grads)
    cs = None if copies is None else [copies] if isinstance(copies, torch.Tensor) else list(copies)
    if not isinstance(state, AdamWState):
        raise TypeError(f"{fn}: state must be an AdamWState, got {type(state).__name__}")
    if len(ps) != len(state.shapes) or len(gs) != len(ps) or (cs is not None and len(cs) != len(ps)):
        raise ValueError(f"{fn}: {len(ps)} parameters, {len(gs)} gradients" + ("" if cs is None else f", {len(cs)} copies")
                         + f" and states for {len(state.shapes)}")
    beta1, beta2 = map(float, betas)
    eps, weight_decay = float(eps), float(weight_decay)
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1):
        raise ValueError(f"{fn}: betas must be in [0, 1) (got {betas})")
    if not (0 <= eps < 1e30 and 0 <= weight_decay < 1e30):
        raise ValueError(f"{fn}: eps and weight_decay must be at least 0 and finite (got {eps} and {weight_decay})")
    if not isinstance(lr, torch.Tensor) and not 0 <= (lr := float(lr)) < 1e30:
        raise ValueError(f"{fn}: lr must be at least 0 and finite (got {lr})")
    if (norm is None) != (max_norm is None):
        raise ValueError(f"{fn}: norm and max_norm go together")
    if norm is not None:
        _check.tensor("norm", norm)
        max_norm = float(max_norm)
        if not max_norm >= 0:
            raise ValueError(f"{fn}: max_norm must be at least 0 (got {max_norm})")
    indexes, places, sizes, shapes = range(len(ps)), state.places, state.sizes, state.shapes
    if any(g is None for g in gs):
        indexes = [i for i, g in enumerate(gs) if g is not None]
        ps, gs, places, sizes, shapes = ([x[i] for i in indexes] for x in (ps, gs, places, sizes, shapes))
        cs = None if cs is None else [cs[i] for i in indexes]
    dev = state.m.device
    p_kinds, g_kinds = _kinds(fn, "parameters", ps, dev), _kinds(fn, "gradients", gs, dev)
    _check.no_tangents(fn, [*ps, *gs])
    _shapes_match(fn, "parameters", ps, shapes)
    _shapes_match(fn, "gradients", gs, shapes)
    given = range(0)  # places in the list of what has a copy
    if cs is None:
        cs = []
    else:
        given = range(len(cs))
        if any(c is None for c in cs):
            given = [i for i in given if cs[i] is not None]
            cs = [cs[i] for i in given]
            _shapes_match(fn, "copies", cs, [shapes[i] for i in given])
        else:
            _shapes_match(fn, "copies", cs, shapes)
    c_kinds = _kinds(fn, "copies", cs, dev)
    if not ps:
        return
    if isinstance(lr, torch.Tensor):
        lr = _scalar(fn, "lr", lr, dev)
    if norm is not None:
        norm = _scalar(fn, "norm", norm, dev)

    def whole(ts):  # strided tensors are written through copies of their own
        return ts if all(map(_contiguous, ts)) else [t if t.is_contiguous() else t.contiguous() for t in ts]

    p_to, c_to, g_from = whole(ps), whole(cs), whole(gs)
    back = [] if p_to is ps and c_to is cs else [(t, d) for t, d in zip([*ps, *cs], [*p_to, *c_to]) if t is not d]
    if back or g_from is not gs:
        _overlap.apart(fn, [*ps, *cs], gs)  # the library sees the copies
    n = len(ps)
    copied, kinds = [0] * n, g_kinds
    if len(given) == n:
        copied, kinds = map(_pointer, c_to), [g | c << 32 for g, c in zip(g_kinds, c_kinds)]
    else:
        kinds = list(g_kinds)
        for i, c, k in zip(given, c_to, c_kinds):
            copied[i] = c.data_ptr()
            kinds[i] |= k << 32
    words = array("q", bytes(56 * n))  # tms_adamw_tensor entries
    words[0::7] = array("q", map(_pointer, p_to))
    words[1::7] = array("q", map(_pointer, g_from))
    words[2::7] = array("q", copied)
    words[3::7] = array("q", sizes)
    words[4::7] = array("q", places)
    words[5::7] = array("q", [i | k << 32 for i, k in zip(indexes, p_kinds)])
    words[6::7] = array("q", kinds)
    factors = torch.empty(4 * len(state.shapes), dtype=torch.float32, device=dev)
    host_lr = 0.0 if isinstance(lr, torch.Tensor) else lr
    described = _pack(state.m.data_ptr(), state.v.data_ptr(), _lib.ptr(state.m_exp) or 0, _lib.ptr(state.v_exp) or 0,
                      state.steps.data_ptr(), factors.data_ptr(), _lib.ptr(norm) or 0, lr.data_ptr() if isinstance(lr, torch.Tensor) else 0,
                      state.size, len(state.shapes), state.bits, host_lr, beta1, beta2, eps, weight_decay, max_norm or 0.0)
    status = _lib.launch(dev, _lib.load().tms_adamw_step, words.buffer_info()[0], n, described)
    if status:
        _lib.check(status)
    for t, d in back:
        t.copy_(d)
    changed = [*ps, *cs]
    try:
        torch.autograd.graph.increment_version(changed)
    except RuntimeError:  # inference tensors count no versions
        torch.autograd.graph.increment_version([t for t in changed if not t.is_inference()])
