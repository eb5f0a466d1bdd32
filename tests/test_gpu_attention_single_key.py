"""Rows of attention that see one key: P is 1 whatever the score, so queries have no gradient there, and keys none from them.

The output is P v / P, where P is 1 + d, |d| at most 2^-22 of the score (below 2^-14 here). In 16 bits P rounds to 1 on its way to
the product, and the quotient is off by d and half a step: below two steps of fp16. In fp32: three roundings, below two steps."""
import math

import pytest
import torch

from test_gpu_attention import DT, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("H,KV", [(1, 1), (4, 2), (12, 1)])
@pytest.mark.parametrize("how", [{}, dict(prefix=0), dict(prefix=5, cap=3.0), dict(slopes=0.5), dict(cap=200.0, slopes=-2.0)], ids=str)
def test_texts_of_one_token(cuda, H, KV, D, how, dt):
    import tilemaxsim_amd as tms
    ts, offsets, G = make([1] * 70 + [0, 1], H, KV, D, dt, seed=H, scale=4.0, behind=2)
    how = {**how, **({"slopes": torch.full((H,), how["slopes"], device="cuda")} if "slopes" in how else {})}
    out = tms.packed_attention(*ts, offsets, **how)
    dq, dk, dv = torch.autograd.grad(out, ts, G)
    v = ts[2][:71].repeat_interleave(H // KV, 1).double()
    assert bool(((out[:71].double() - v).abs() <= 2 * torch.finfo(dt).eps * v.abs()).all()) and not out[71:].any()
    assert not dq.any() and not dk.any()
    want = G.double().unflatten(1, (KV, H // KV)).sum(2)
    want[71:] = 0
    # a sum of H / KV addends in fp32, P of 1 + d each, rounded once
    off = torch.finfo(dt).eps / 2 * want.abs() + (2.0 ** -14 + H // KV * 2.0 ** -23) * G.double().abs().unflatten(1, (KV, H // KV)).sum(2)
    assert bool(((dv.double() - want).abs() <= off).all())
    with torch.no_grad():
        g = G.clone()
        g[3, 0, 1] = math.nan
    dq, dk, dv = torch.autograd.grad(tms.packed_attention(*ts, offsets, **how), ts, g)  # not hidden by a factor of 0
    assert bool(torch.isnan(dq[3, 0]).all()) and bool(torch.isnan(dk[3, 0]).all()) and not dq[:3].any() and not dk[4:].any()


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[40, 1, 90], [700, 1300], [2500]])
def test_first_rows_of_causal_texts(cuda, lens, D, dt):
    import tilemaxsim_amd as tms
    H = 24 if sum(lens) > 1000 else 2
    ts, offsets, G = make(lens, H, H, D, dt, seed=D, scale=3.0)
    for prefix in (0, 1):
        out = tms.packed_attention(*ts, offsets, prefix=prefix)
        dq, _, _ = torch.autograd.grad(out, ts, G)
        first = offsets[:-1].cuda()
        v = ts[2][first].double()
        assert not dq[first].any() and bool(((out[first].double() - v).abs() <= 2 * torch.finfo(dt).eps * v.abs()).all())
        last = (offsets[1:] - 1)[torch.tensor(lens) > 1].cuda()
        assert bool(dq[last].any())
