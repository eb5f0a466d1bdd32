"""CPU tests: calls of the training operators that would give a wrong result are refused, before
any HIP call."""
import ctypes

import pytest
import torch
from test_training_host import F16, F32, Grad, call, numbers

KB = 1 << 10


def clip(*entries):
    """What the call says of these tensors; without a workspace, so that one it takes ends there."""
    table, most = (Grad * len(entries))(*entries), numbers(1.0)[0]
    return call("tms_grad_clip", ctypes.addressof(table), len(entries), 2, ctypes.addressof(most), None, 0, 16, None)


IN_PLACE = Grad(4096 * KB, 4096 * KB, 256, F32, F32)  # 1 KB


@pytest.mark.parametrize("entries", [
    (IN_PLACE, IN_PLACE),  # one tensor twice, as tied weights are gathered module by module
    (IN_PLACE, Grad(64, 64, 4, F16, F16), Grad(4097 * KB - 4, 4097 * KB - 4, 1, F32, F32)),  # its last element alone
    (IN_PLACE, Grad(4096 * KB - 8, 4096 * KB - 8, 5, F16, F16)),  # and its first one, of another dtype
    (Grad(64 * KB, 128 * KB, 256, F32, F32), Grad(192 * KB, 128 * KB, 256, F32, F32)),  # two gradients into one tensor
    (Grad(64 * KB, 128 * KB, 256, F32, F32), Grad(128 * KB + 512, 256 * KB, 4, F32, F32)),  # into another one's gradient
    (Grad(128 * KB + 512, 256 * KB, 4, F32, F32), Grad(64 * KB, 128 * KB, 256, F32, F32)),
    (Grad(64 * KB, 64 * KB + 4, 256, F32, F32),),  # into itself, one element on
    (Grad(64 * KB, 64 * KB, 256, F32, F16),),  # into itself in another dtype
    tuple(Grad(k * KB, k * KB, 4, F32, F32) for k in (9, 2, 7, 5, 2, 8)),  # in no order
    tuple(Grad((500 - k) * KB, (500 - k) * KB, 256, F32, F32) for k in range(300)) + (Grad(300 * KB, 300 * KB, 1, F32, F32),)])
def test_overlapping_tensors_are_not_clipped(entries):
    rc, msg = clip(*entries)
    assert rc == 1 and "overlap" in msg and "tms_grad_clip" in msg


@pytest.mark.parametrize("entries", [
    (IN_PLACE, Grad(4097 * KB, 4097 * KB, 256, F32, F32), Grad(4095 * KB, 4095 * KB, 256, F32, F32)),  # end to end
    (IN_PLACE, Grad(4096 * KB, 4096 * KB, 0, F32, F32)),  # an empty one takes no place
    (Grad(64 * KB, 128 * KB, 256, F32, F32), Grad(64 * KB, 192 * KB, 256, F32, F32)),  # one gradient into two tensors
    (Grad(64 * KB, 128 * KB, 256, F16, F32), Grad(64 * KB + 512, 129 * KB, 256, F16, F32))])
def test_neighbours_and_shared_sources_are_taken(entries):
    rc, msg = clip(*entries)
    assert rc == 1 and "workspace" in msg


def test_parameters_are_not_gradients():
    """``clip_grad_norm_(model.parameters(), 1.0)`` would scale the parameters."""
    import tilemaxsim_amd as tms
    model = torch.nn.Linear(3, 2)
    before = [p.detach().clone() for p in model.parameters()]
    for given in (model.parameters(), list(model.parameters()), model.weight):
        with pytest.raises(ValueError, match="their gradients"):
            tms.clip_grad_norm_(given, 1.0)
    g = [torch.ones(2, 3), torch.ones(2)]
    with pytest.raises(ValueError, match="their gradients"):
        tms.clip_grad_norm_(model.parameters(), 1.0, out=g)
    with pytest.raises(ValueError, match="their gradients"):
        tms.clip_grad_norm_(g, 1.0, out=list(model.parameters()))
    assert all(torch.equal(p, b) for p, b in zip(model.parameters(), before))
    # gradients that are a graph's (create_graph) are clipped, as any
    x = torch.ones(3, requires_grad=True)
    grad, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    with pytest.raises(ValueError, match="no CPU path"):
        tms.clip_grad_norm_([grad], 1.0)


def test_a_norm_without_a_graph_is_not_taken_for_one():
    """A gradient penalty through ``grad_norm`` would train nothing."""
    import tilemaxsim_amd as tms
    x = torch.ones(3, requires_grad=True)
    grad, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    for t in (x, grad):
        with pytest.raises(RuntimeError, match="not differentiable"):
            tms.grad_norm([torch.ones(2), t])
        with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
            tms.grad_norm([t])
        with pytest.raises(ValueError, match="no CPU path"):
            tms.grad_norm([t.detach()])


def test_forward_mode_is_refused():
    """A dual tensor's tangent would be lost."""
    import tilemaxsim_amd as tms
    from torch.autograd import forward_ad
    Q, D, H, W, t = torch.ones(2, 4, 32), torch.ones(3, 5, 32), torch.ones(3, 8), torch.ones(10, 8), torch.tensor([0, 1, 2])
    with forward_ad.dual_level():
        def dual(x):
            return forward_ad.make_dual(x, torch.ones_like(x))
        calls = [lambda: tms.maxsim_pairs(dual(Q), D), lambda: tms.maxsim_pairs(Q, dual(D)), lambda: tms.linear_cross_entropy(dual(H), W, t),
                 lambda: tms.linear_cross_entropy(H, dual(W), t), lambda: tms.grad_norm([H, dual(W)]),
                 lambda: tms.clip_grad_norm_([dual(H)], 1.0)]
        for f in calls:
            with pytest.raises(NotImplementedError, match="forward mode"):
                f()
        with pytest.raises(ValueError, match="no CPU path"):
            tms.maxsim_pairs(Q, D)
    # the same through torch.func, whose tensors are dual ones inside
    for f, x in ((lambda q: tms.maxsim_pairs(q, D), Q), (lambda w: tms.linear_cross_entropy(H, w, t), W)):
        with pytest.raises(NotImplementedError, match="forward mode"):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
