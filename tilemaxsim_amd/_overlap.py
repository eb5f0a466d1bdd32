"""Which strided tensors share memory, exactly. The library looks over contiguous ranges itself; strided tensors
that a call writes go through contiguous copies, which share nothing, so their own memory is looked over here.

Two elements i and j of one address are a solution of sum s_k i_k - sum t_l j_l = distance with 0 <= i_k < n_k, 0 <= j_l < m_l:
with m_l - 1 - j_l in the place of j_l all coefficients are positive. The largest stride's multiples that the
others can make up for are few where rows do not overlap, so a search that takes the strides in turn, with the greatest
common divisor and the reach of those left, ends soon.
"""
from __future__ import annotations

import math

import torch

_MOST = 20_000  # steps of a search; more are taken for an overlap


def _solvable(dims, target: int) -> bool:
    """Whether sum s x = target has a solution with 0 <= x <= most for each (s, most) of dims."""
    by_stride: dict = {}
    for s, most in dims:
        if s and most:
            by_stride[s] = by_stride.get(s, 0) + most
    dims = sorted(by_stride.items(), reverse=True)
    reach, gcd = [0], [0]
    for s, most in reversed(dims):
        reach.append(reach[-1] + s * most)
        gcd.append(math.gcd(gcd[-1], s))
    reach.reverse()
    gcd.reverse()
    left = _MOST

    def go(k: int, rest: int) -> bool:
        nonlocal left
        left -= 1
        if rest == 0 or left < 0:
            return True
        if rest < 0 or rest > reach[k] or rest % gcd[k]:
            return False
        s, most = dims[k]
        high, low = min(most, rest // s), max(0, -(-(rest - reach[k + 1]) // s))
        return any(go(k + 1, rest - s * x) for x in range(low, high + 1))

    return go(0, target)


def _dims(t: torch.Tensor) -> list:
    size = t.element_size()
    return [(s * size, n - 1) for s, n in zip(t.stride(), t.shape) if n > 1]


def _folds(t: torch.Tensor) -> bool:
    """Whether two elements of t are at one address."""
    dims = sorted(_dims(t))
    below = t.element_size()
    for s, most in dims:
        if s < below:
            break
        below = s * most + below
    else:
        return False
    # the first stride in which they differ by 1 + x, the ones after it by -most .. most
    for k, (s, most) in enumerate(dims):
        rest = dims[k + 1:]
        if s == 0 or _solvable([(s, most - 1), *((r, 2 * m) for r, m in rest)], sum(r * m for r, m in rest) - s):
            return True
    return False


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether any byte of a is one of b's."""
    theirs = _dims(b)
    inner = [(1, a.element_size() - 1), (1, b.element_size() - 1)]
    target = b.data_ptr() - a.data_ptr() + sum(s * most for s, most in theirs) + b.element_size() - 1
    return _solvable([*_dims(a), *theirs, *inner], target)


def _apart(fn: str, order: list, begins: list, ends: list, pair) -> None:
    """Goes over spans in order of their begins, and asks pair(i, j) of those that overlap."""
    near: list = []  # those that reach the next one's begin
    for i in order:
        if near:
            at = begins[i]
            near = [j for j in near if ends[j] > at]
            if any(pair(i, j) for j in near):
                raise ValueError(f"{fn}: two of the tensors overlap")
        near.append(i)


def apart(fn: str, written: list, read: list) -> None:
    """Refuses tensors of which a written one shares memory with another one, or with itself."""
    ts, writes = [*written, *read], len(written)
    begins = list(map(torch.Tensor.data_ptr, ts))
    sizes = list(map(torch.Tensor.numel, ts))
    ends = [at + n * size for at, n, size in zip(begins, sizes, map(torch.Tensor.element_size, ts))]
    strided = {i for i, whole in enumerate(map(torch.Tensor.is_contiguous, ts)) if not whole and sizes[i]}
    for i in strided:
        if i < writes and _folds(ts[i]):
            raise ValueError(f"{fn}: two elements of a tensor overlap")
        ends[i] = begins[i] + ts[i].element_size() + sum(s * most for s, most in _dims(ts[i]))

    def pair(i: int, j: int) -> bool:
        if i >= writes and j >= writes:
            return False
        if i not in strided and j not in strided:
            return begins[i] < ends[j] and begins[j] < ends[i]
        return _meet(ts[i], ts[j])

    order = sorted((i for i, n in enumerate(sizes) if n), key=begins.__getitem__)
    first = 0
    while first < len(order):  # tensors whose spans hang together
        last, reach = first + 1, ends[order[first]]
        while last < len(order) and begins[order[last]] < reach:
            reach = max(reach, ends[order[last]])
            last += 1
        group, first = order[first:last], last
        rows = _rows(group, ts, begins) if len(group) > 2 and not strided.isdisjoint(group) else None
        _apart(fn, *(rows or (group, begins, ends)), pair)


def _rows(group: list, ts: list, begins: list):
    """Views of some columns of one matrix as spans within its rows (many of them would be compared pair by pair
    otherwise): the order, begins and ends; None if they are no such views."""
    pitch, at, to = None, {}, {}
    for i in group:
        dims = _dims(ts[i])
        if not dims:
            return None
        s = max(s for s, _ in dims)
        inner = ts[i].element_size() + sum(r * most for r, most in dims) - s * max(most for r, most in dims if r == s)
        at[i] = (begins[i] - begins[group[0]]) % (pitch or s or 1)
        to[i] = at[i] + inner
        if s != (pitch or s) or not s or to[i] > s:
            return None
        pitch = s
    return sorted(group, key=at.__getitem__), at, to
