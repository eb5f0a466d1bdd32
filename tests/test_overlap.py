"""CPU tests: which tensors share memory, exactly, where they are strided; and that the optimizer's step and clipping refuse those
before anything is launched."""
import itertools
import random

import pytest
import torch


def places(t):
    """The bytes of a tensor's elements, one by one."""
    at = [t.data_ptr()]
    for n, s in zip(t.shape, t.stride()):
        at = [a + i * s * t.element_size() for a in at for i in range(n)]
    return [a + b for a in at for b in range(t.element_size())]


def refused(written, read=()):
    from tilemaxsim_amd import _overlap
    try:
        _overlap.apart("fn", list(written), list(read))
    except ValueError as e:
        assert "fn" in str(e) and "overlap" in str(e)
        return True
    return False


def test_against_every_place():
    """Random strided views of one buffer, of several element sizes: refused where two places are one, and only there."""
    rng = random.Random(0)
    flat = torch.zeros(8192, dtype=torch.uint8)
    outcomes = []
    for _ in range(3000):
        views = []
        for _ in range(rng.choice((1, 2, 2, 3, 4))):
            dt = rng.choice((torch.float32, torch.bfloat16, torch.float32))
            dims = rng.randint(1, 3)
            shape = [rng.choice((1, 2, 3, 5, 8)) for _ in range(dims)]
            stride = [rng.choice((0, 1, 2, 3, 4, 6, 8, 15, 16, 40)) if rng.random() < 0.6 else rng.choice((1, 8, 64)) for _ in range(dims)]
            size = torch.empty(0, dtype=dt).element_size()
            views.append(flat.view(dt).as_strided(shape, stride, rng.randrange(0, 400) * 2 // size))
        cut = rng.randint(1, len(views))
        written, read = views[:cut], views[cut:]
        taken = [p for t in written for p in places(t)]
        want = len(set(taken)) != len(taken) or any(set(taken) & set(places(t)) for t in read)
        assert refused(written, read) == want, [(t.shape, t.stride(), t.storage_offset(), t.dtype) for t in views]
        outcomes.append(want)
    assert 300 < sum(outcomes) < 2700


def test_views_of_one_buffer():
    w = torch.zeros(30, 80)
    assert not refused([w[:, :40], w[:, 40:]]) and not refused([w[:, ::2], w[:, 1::2]]) and not refused([w.t()]) and not refused([w[:10], w[10:].t()])
    assert not refused([w[:, i] for i in range(80)]) and not refused([w[:, :40]], [w[:, 40:]]) and not refused([], [w, w.t()])
    assert refused([w[:, :50], w[:, 40:]]) and refused([w[:, 0:4], w[:, 2:6]]) and refused([w.t(), w[5:6]]) and refused([w[::2, 3]], [w[4]])
    assert refused([w.view(-1).as_strided((30, 80), (40, 1))]) and refused([w[:1].expand(4, 80)]) and refused([w, w])
    assert not refused([w[:0], w[:, :0], w]) and not refused([w[0, 0], w[0, 1:]]) and refused([w[0, 1], w[0, 1:]])
    wide = torch.empty(1 << 16, 64)  # no list of places: strides are compared
    assert not refused([wide[:, :32], wide[:, 32:]]) and refused([wide[:, :33], wide[:, 32:]])


def test_many_columns_of_one_matrix():
    """Hundreds of views side by side are told from each other in a moment; one that reaches into its neighbour is found."""
    import time
    w = torch.zeros(50, 4096)
    columns = [w[:, 8 * i:8 * i + 8] for i in range(512)]
    began = time.perf_counter()
    assert not refused(columns) and not refused(columns[::2], columns[1::2])
    assert time.perf_counter() - began < 1.0  # pair by pair: some 131,000 comparisons of 10 us
    assert refused([*columns[:100], w[:, 799:808], *columns[101:]]) and refused(columns[:9], [w[3:4, 5:9], w[:, 4000]])
    assert not refused([*columns[:100], *columns[101:]], [w[:, 800:804], w[2, 804:806]])
    halves = [w[::2, :64], w[1::2, :64], w[::2, 64:], w[1::2, 64:]]  # rows in turn: another pitch than the matrix's
    assert not refused(halves) and refused([*halves, w[3:4, 10:20]])
    assert refused([w.as_strided((49, 10), (4096, 1), 4090), w[:, :8], w[:, 8:16]])  # behind a row's end, into the next one
    flat = torch.zeros(100)
    assert not refused([flat[::2], flat[1:50:2], flat[51:60:2], flat[61:62], flat[63:64]]) and refused([flat[::2], flat[1:50:2], flat[50:51]])


def test_what_takes_too_long_to_tell_is_refused():
    """Strides made so that their sums are hard to compare: refused, in a moment."""
    shape = [2] * 24
    flat = torch.zeros(1)
    a = torch.as_strided(flat, [1] * 24, [1] * 24).expand([1] * 24)
    assert not refused([a])
    rng = random.Random(1)
    sizes = sorted(rng.sample(range(1 << 18, 1 << 19), 24))
    big = torch.empty(sum(sizes) + 1)
    assert refused([big.as_strided(shape, sizes)])


def step_of(params, grads, copies=None, monkeypatch=None):
    import tilemaxsim_amd as tms
    from test_encoder_host import fake_state
    from tilemaxsim_amd import adamw as module
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: None)
    monkeypatch.setattr(module._lib, "launch", lambda *a: pytest.fail("launched"))
    tms.adamw_(params, grads, fake_state([p.shape for p in params]), copies=copies)


def test_adamw_refuses_strided_tensors_that_overlap(monkeypatch):
    w = torch.zeros(30, 80)
    ones = torch.ones(30, 80)
    cases = [([w[:, :50], w[:, 40:]], [ones[:, :50], ones[:, :40]], None), ([w.t()[:, :3], w[2]], [ones.t()[:, :3], ones[2]], None),
             ([ones[:, :40]], [w[:, :40]], [ones[:, 30:70]]), ([w[:, :40]], [w[:, 20:60]], None), ([w[:, :40]], [w[5].view(2, 40).expand(15, 2, 40).reshape(30, 40)], [w[:, 39:79]]),
             ([w.view(-1).as_strided((30, 40), (30, 1))], [ones[:, :40]], None), ([w[:, 0]], [w.view(-1)[75:105]], None),
             ([w[5:7].view(160)], [w.view(-1)[300:620:2]], None)]
    for params, grads, copies in cases:
        with pytest.raises(ValueError, match="overlap"):
            step_of(params, grads, copies, monkeypatch)


def test_clipping_refuses_strided_tensors_that_overlap(monkeypatch):
    """Gradients scaled in place, and scaled into others: a gradient's own tensor may be the gradient itself, as a whole."""
    import tilemaxsim_amd as tms
    from tilemaxsim_amd import grad_clip as module
    monkeypatch.setattr(module, "_on_one_gpu", lambda *a: None)

    class Launched(Exception):
        pass

    def launch(*a):
        raise Launched

    monkeypatch.setattr(module._lib, "launch", launch)
    w, x = torch.zeros(30, 80), torch.zeros(30, 80)
    for grads, out in (([w[:, :50], w[:, 40:]], None), ([w.t()[:, :3], w[2]], None), ([w[:1].expand(30, 80)], None), ([x[:, :40]], [w.view(-1).as_strided((30, 40), (30, 1))]),
                       ([w[:, :40]], [w[:, 1:41]]), ([w[5:7].view(160)], [w.view(-1)[300:620:2]]), ([w.view(-1)[300:620:2]], [w[5:7].view(160)]),
                       ([w[:, :40], x[:, :40]], [w[:, 40:], w[:, :40]]), ([w[:30, :30]], [w[:30, :30].t()])):
        with pytest.raises(ValueError, match="overlap"):
            tms.clip_grad_norm_(grads, 1.0, out=out)
    for grads, out in (([w[:, :50], w[:, 50:]], None), ([w[:, ::2], w[:, 1::2]], None), ([w[:, :40]], [w[:, :40]]), ([w[:, :40]], [w[:, 40:]]),
                       ([w[:1].expand(30, 80)], [x]), ([w[3:4], w[5].view(40, 2)[:, 0]], [w[3].as_strided((1, 80), (7, 1)), x[:20, 0:4:2].reshape(40)]), ([w[:, :40], w[:, :40]], [x[:, :40], x[:, 40:]])):
        with pytest.raises(Launched):
            tms.clip_grad_norm_(grads, 1.0, out=out)
