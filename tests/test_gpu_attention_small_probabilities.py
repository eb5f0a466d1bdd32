"""Attention rows with one key far above many others: each of those has a probability next to nothing, and
all of them together a part of the row.

Row i's score is a[i] for every key but the first, which has a[i] + gap[i]: exact in the products (one
element of q and k each, powers of two and halves). The bound: 2 u for P, rounded the same way in all keys, and in
fp16 as much again where 2^15 P is below its normal numbers, 2^-25 of 2^15 at worst (2^-40); exponentials of 2^-22 and what
an exponent of 40 loses, 2^-17, together 2^-16 of P; the normaliser's sum, of which a quarter of the keys adds to the
first key's 1 and may be lost there, T / 4 2^-24, and sums of a tile's products, T / 32 2^-24: together T 2^-25; and half a
step of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("T,H,D", [(300, 2, 32), (300, 1, 64), (700, 1, 96), (700, 2, 128), (66_000, 1, 32), (131_072, 1, 32)])
def test_they_add_up(cuda, T, H, D, dt):
    import tilemaxsim_amd as tms
    print(T, H, D, dt, flush=True)
    gaps = torch.arange(20, 38, device="cuda") / 2.0  # e^-10 to e^-18.5: 2^-14.4 to 2^-26.7
    gap = gaps[torch.arange(T, device="cuda") % len(gaps)]
    q, k, v = (torch.zeros(T, H, D, device="cuda", dtype=dt) for _ in range(3))
    q[:, :, 5] = gap[:, None].to(dt)
    k[0, :, 5] = 1.0
    g = torch.Generator(device="cuda").manual_seed(T)
    v[1:] = (torch.rand(T - 1, H, D, generator=g, device="cuda") + 0.5).to(dt)
    offsets = torch.tensor([0, T])
    got = tms.packed_attention(q, k, v, offsets, scale=1.0).double()
    others = v[1:].double().sum(0)
    each = torch.exp(-gap.double())  # beside the first key's 1
    want = each[:, None, None] * others / (1 + (T - 1) * each)[:, None, None]
    u = U[dt]
    off = (2 * u if dt != torch.float32 else 0) + 2.0 ** -16 + T * 2.0 ** -25
    low = 2.0 ** -40 * others if dt == torch.float16 else 0
    bound = off * want + low + u * want + (2.0 ** -25 if dt == torch.float16 else 0)
    over = ((got - want).abs() / bound).amax((1, 2))
    assert float(over.max()) <= 1.0, f"{float(over.max()):.3g} times its bound off, {float((1 - got / want).abs().max()):.3g} of itself"
