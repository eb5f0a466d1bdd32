"""MaxSim of query and document batches with gradients: what a late-interaction encoder is
trained through.

``maxsim_pairs(Qs, D)`` scores every query against every document (in-batch negatives), or
each query against documents of its own (distillation, hard negatives), and is
differentiable in both. The similarities are never in memory: the forward kernel keeps the
position of each maximum (2 bytes), and the backward kernels gather and add the token
embeddings that won. No reference counterpart (the reference scores only; its callers'
``pytorch_maxsim_score``, ``src/e2e_retrieval_quality.py:105-110``, is the same sum).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _check, _lib

MAX_DOC_TOKENS = 65535


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, and at an address the kernels' 16-byte loads take."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _documents(Q, D):
    """The documents of all queries and of each one's own (0: every query with every document),
    as the library counts them; and the scores' columns."""
    if D.dim() == 3:
        return D.shape[0], 0, D.shape[0]
    return Q.shape[0] * D.shape[1], D.shape[1], D.shape[1]


def _forward(Q, D, qmask, dmask, keep):
    nQ, Nq, d = Q.shape
    Nd = D.shape[-2]
    B, nway, columns = _documents(Q, D)
    lib = _lib.load()
    code = _lib.dtype_code(D.dtype)
    scores = torch.empty(nQ, columns, dtype=torch.float32, device=D.device)
    positions = None
    if keep:
        positions = torch.empty(lib.tms_pairs_positions(nQ, Nq, B, nway), dtype=torch.int16, device=D.device)
    if scores.numel():
        nbytes = lib.tms_pairs_workspace_size(nQ, Nq, d, B, Nd, code)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=D.device) if nbytes else None
        status = _lib.launch(D.device, lib.tms_maxsim_pairs, Q.data_ptr(), nQ, Nq, d, D.data_ptr(), B, Nd, nway,
                             _lib.ptr(qmask), _lib.ptr(dmask), code, _lib.ptr(ws), nbytes, scores.data_ptr(),
                             _lib.ptr(positions))
        if status:
            _lib.check(status)
    return scores, positions


class _Pairs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, Q, D, qmask, dmask):
        scores, positions = _forward(Q, D, qmask, dmask, True)
        ctx.save_for_backward(Q, D, positions)
        return scores

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        Q, D, positions = ctx.saved_tensors
        nQ, Nq, d = Q.shape
        Nd = D.shape[-2]
        B, nway, _ = _documents(Q, D)
        lib = _lib.load()
        grad = grad.contiguous()
        dQ = torch.empty_like(Q) if ctx.needs_input_grad[0] else None
        dD = torch.empty_like(D) if ctx.needs_input_grad[1] else None
        nbytes = lib.tms_pairs_grad_workspace_size(nQ, Nq, d, B, Nd, nway)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=D.device) if nbytes else None
        status = _lib.launch(D.device, lib.tms_maxsim_pairs_grad, Q.data_ptr(), nQ, Nq, d, D.data_ptr(), B, Nd, nway,
                             positions.data_ptr(), grad.data_ptr(), _lib.dtype_code(D.dtype), _lib.ptr(ws), nbytes,
                             _lib.ptr(dQ), _lib.ptr(dD))
        if status:
            _lib.check(status)
        return dQ, dD, None, None


def _mask(name: str, mask, shape):
    if mask is None:
        return None
    _check.tensor(name, mask)
    if tuple(mask.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(mask.shape)}")
    if mask.dtype not in (torch.bool, torch.uint8, torch.int8):
        if mask.is_floating_point() or mask.is_complex():
            raise TypeError(f"{name} must be a boolean or integer tensor (got {mask.dtype})")
        mask = mask != 0
    return mask.contiguous()


def maxsim_pairs(Qs: torch.Tensor, D: torch.Tensor, D_mask: torch.Tensor | None = None,
                 Q_mask: torch.Tensor | None = None) -> torch.Tensor:
    """MaxSim scores of a batch of queries and a batch of documents, differentiable in both.

    ``scores[q, b] = sum_i max_j Qs[q, i] . D[b, j]`` over the real tokens i and j, in fp32.

    Args:
        Qs: (nQ, Nq, d) query token embeddings, float16, bfloat16 or float32.
        D: (B, Nd, d) documents, which every query is scored against; or (nQ, nway, Nd, d),
            query q's own documents D[q]. Same dtype and device as Qs; any d; Nd <= 65535.
        D_mask: (B, Nd) or (nQ, nway, Nd), bool or integer, non-zero for a real token. What
            stands at the masked tokens (NaN included) is never seen.
        Q_mask: (nQ, Nq), likewise: a masked query token adds nothing.

    Returns:
        (nQ, B) or (nQ, nway) float32 scores. A document without a real token scores -inf
        and takes and gives no gradient. NaN at a real token makes its scores NaN.

    A maximum's gradient goes to one token, the first of equal ones. Gradients are summed in
    fp32, in one order whatever the timing, and rounded once to the inputs' dtype.
    """
    _check.tensor("Qs", Qs)
    _check.tensor("D", D)
    _check.no_tangents("maxsim_pairs", (Qs, D))
    if Qs.dim() != 3 or D.dim() not in (3, 4):
        raise ValueError("maxsim_pairs: Qs must be (nQ, Nq, d), and D (B, Nd, d) or (nQ, nway, Nd, d), got "
                         f"{tuple(Qs.shape)} and {tuple(D.shape)}")
    if Qs.shape[-1] != D.shape[-1]:
        raise ValueError(f"maxsim_pairs: Qs width {Qs.shape[-1]} != D width {D.shape[-1]}")
    if D.dim() == 4 and D.shape[0] != Qs.shape[0]:
        raise ValueError(f"maxsim_pairs: D has documents for {D.shape[0]} queries, Qs has {Qs.shape[0]}")
    _check.embedding_dtype("D", D)
    if Qs.dtype != D.dtype:
        raise TypeError(f"maxsim_pairs: Qs is {Qs.dtype}, D is {D.dtype}")
    qmask = _mask("Q_mask", Q_mask, Qs.shape[:2])
    dmask = _mask("D_mask", D_mask, D.shape[:-1])
    if D.shape[-2] > MAX_DOC_TOKENS:
        raise NotImplementedError(f"maxsim_pairs: documents of more than {MAX_DOC_TOKENS} tokens (got {D.shape[-2]})")
    _check.on_gpu("Qs", Qs)
    _check.on_gpu("D", D)
    given = {"Qs": Qs, "D": D}
    if qmask is not None:
        given["Q_mask"] = qmask
    if dmask is not None:
        given["D_mask"] = dmask
    _check.same_device(**given)
    Qs, D = _aligned(Qs), _aligned(D)
    if torch.is_grad_enabled() and (Qs.requires_grad or D.requires_grad):
        return _Pairs.apply(Qs, D, qmask, dmask)
    return _forward(Qs, D, qmask, dmask, False)[0]
