"""``linear_cross_entropy`` over several pieces of the vocabulary: the second piece on adds to dH's
sums, finds targets past its first row, and ends short. The bounds are those of the other sizes."""
import ctypes

import pytest
import torch
from test_gpu_cross_entropy import check, data
from test_training_host import plan  # noqa: F401 (a fixture: the rules that pick the pieces)

# N, V, d, dtype, pieces at least
SIZES = [(9000, 60000, 16, "bf16", 2), (9000, 60000, 16, "fp16", 2), (20000, 70001, 8, "bf16", 3), (9000, 33000, 16, "fp32", 2),
         (6001, 100_003, 8, "fp32", 3)]


def pieces_of(plan, N, V, d, dtype):  # noqa: F811
    out = (ctypes.c_int64 * 7)()
    plan.lce_plan_of(N, V, d, 3 if dtype == "fp32" else 1, out)
    return out[2], -(-V // out[2])


@pytest.mark.parametrize("N,V,d,dtype,least", SIZES)
def test_sizes_have_several_pieces(plan, N, V, d, dtype, least):  # noqa: F811
    piece, pieces = pieces_of(plan, N, V, d, dtype)
    assert pieces >= least and V % piece  # the last one is short


@pytest.mark.gpu
@pytest.mark.parametrize("N,V,d,dtype,least", SIZES)
def test_pieces(cuda, plan, N, V, d, dtype, least):  # noqa: F811
    piece, pieces = pieces_of(plan, N, V, d, dtype)
    assert pieces >= least
    given = H, W, t = data(N, V, d, dtype, N + V)
    for i in range(pieces):  # a target at each piece's ends
        t[2 * i], t[2 * i + 1] = i * piece, min((i + 1) * piece, V) - 1
    check(N, V, d, dtype, given=given)
