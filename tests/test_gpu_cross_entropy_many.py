"""``linear_cross_entropy`` of so many rows and classes that the tiles of their product, with a
workgroup of 512 threads each, pass the 2^32 threads of one axis of a launch."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_million_rows_and_classes(cuda):
    """64 different rows over and over, on a grid on which logits are exact, so that the loss's
    own rounding is left: |x| of at most 4, 2^-20 for the exponentials and a row's sum, and the
    join of 8000 blocks 2^-18."""
    import tilemaxsim_amd as tms
    N, V, d = (1 << 20) + 77, (1 << 20) + 300, 8
    assert -(-N // 256) * -(-V // 256) * 512 > 1 << 32
    rng = np.random.default_rng(4)
    base = torch.from_numpy(rng.integers(-4, 5, (64, d)) / 8.0).cuda()
    W = torch.from_numpy(rng.integers(-8, 9, (V, d)) / 8.0).cuda()
    t = torch.from_numpy(rng.integers(0, V, N)).cuda()
    t[0], t[-1], t[-2] = V - 1, 0, V - 1
    row = torch.arange(N, device="cuda") % 64
    print(f"ce N={N} V={V} d={d}", flush=True)
    loss = tms.linear_cross_entropy(base[row].bfloat16(), W.bfloat16(), t, reduction="none")
    x = base @ W.t()  # (64, V), float64
    want = torch.logsumexp(x, 1)[row] - x[row, t]
    assert float(((loss.double() - want).abs() / want).max()) <= 2.0 ** -17
