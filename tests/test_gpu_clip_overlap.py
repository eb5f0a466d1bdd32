"""Gradients that share memory are refused by ``clip_grad_norm_``, with nothing changed: two entries
of one tensor would be scaled once or twice, by timing."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_one_tensor_twice(cuda):
    import tilemaxsim_amd as tms
    flat = torch.randn(70_000, device="cuda")
    keep = flat.clone()
    wide = torch.randn(40, 60, device="cuda")
    cases = [[flat, flat], [flat[:1000], flat[999:3000]], [flat[5:], flat[:6]], [flat[::2], flat[::2]], [wide, wide.t()],
             [flat.view(torch.bfloat16)[:10], flat[4:8]]]
    for ts in cases:
        with pytest.raises(ValueError, match="overlap"):
            tms.clip_grad_norm_(ts, 1e-3)
        assert torch.equal(flat, keep)
    a, b = torch.randn(100, device="cuda"), torch.randn(100, device="cuda")
    before = a.clone(), b.clone()
    for ts, out in (([a, b], [flat[:100], flat[50:150]]), ([a, b], [b, flat[:100]]), ([a, a], [b, b]), ([flat[:100]], [flat[1:101]])):
        with pytest.raises(ValueError, match="overlap"):
            tms.clip_grad_norm_(ts, 1e-3, out=out)
        assert torch.equal(flat, keep) and torch.equal(a, before[0]) and torch.equal(b, before[1])


def test_neighbours_and_one_gradient_into_two(cuda):
    import tilemaxsim_amd as tms
    flat = torch.ones(3000, device="cuda")
    tms.clip_grad_norm_([flat[2000:], flat[:1000], flat[1000:2000]], 1.0)
    assert bool((flat == flat[0]).all()) and 0 < float(flat[0]) < 1
    g, out = torch.ones(4, device="cuda"), torch.zeros(8, device="cuda")
    tms.clip_grad_norm_([g, g], 1.0, out=[out[:4], out[4:]])
    assert bool((g == 1).all()) and torch.equal(out[:4], out[4:]) and float(out[0]) > 0
    wide = torch.ones(10, 20, device="cuda")
    tms.clip_grad_norm_([wide[:, ::2], wide[:, 1::2]], 1.0)  # one inside the other, no element in both
    assert bool((wide == wide[0, 0]).all()) and float(wide[0, 0]) < 1
