"""``linear_cross_entropy``'s gradient of the hidden states where the vocabulary's rows have much in
common, which cancels: the softmax less one at the target keeps its 32 bits there.

Hidden states are zero, so the softmax is 1 / V with V a power of two, and every product and
sum is exact in fp32 (weights of 1/8 steps below 128, 2^-13 of them, added below 256). What is
left is the factor's product, 2^-23, and one rounding to the inputs' type."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,V,base,step", [(torch.bfloat16, 1024, 16, 2.0 ** -8), (torch.bfloat16, 4096, 16, 2.0 ** -8),
                                               (torch.float16, 8192, 64, 2.0 ** -11), (torch.float32, 8192, 64, 2.0 ** -24)])
@pytest.mark.parametrize("N,d", [(5, 64), (300, 136), (70, 33)])
def test_what_all_words_share_cancels(cuda, N, d, dtype, V, base, step):
    import tilemaxsim_amd as tms
    g = torch.Generator(device="cuda").manual_seed(V + N)
    W = (base + torch.randint(0, 8, (V, d), generator=g, device="cuda") / 8.0).to(dtype)
    assert float(W.min()) >= base and bool((W.double() * 8 % 1 == 0).all())
    H = torch.zeros(N, d, device="cuda", dtype=dtype, requires_grad=True)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    t[0], t[1] = 0, V - 1
    t[3] = -100
    print(f"ce of a common mean N={N} V={V} d={d} {dtype}", flush=True)
    dH, = torch.autograd.grad(tms.linear_cross_entropy(H, W, t, reduction="sum"), H)
    want = W.double().mean(0) - W.double()[t.clamp(min=0)]
    want[3] = 0
    assert bool(((dH.double() - want).abs() <= (step + 2.0 ** -22) * want.abs()).all()), float((dH.double() - want).abs().max())
