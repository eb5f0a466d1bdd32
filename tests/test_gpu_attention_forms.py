"""Forms of attention that its general tests would not tell from another: two terms in short texts, far keys left out
under a bias, memory beside the tensors, and strides that a single token or head leaves open.

References and bounds are those of test_gpu_attention.py."""
import math

import pytest
import torch

import test_gpu_attention as base
from test_gpu_attention import DT, close, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["plain", "causal", "bias", "cap"])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=str)
def test_two_terms_in_short_texts(cuda, monkeypatch, dt, D, kind):
    """Gradients where every text is one tile of keys: P and dS go into their products as two 16-bit terms, and delta comes
    from P and dP before they are rounded. What is left of u is u^2, for each of the three."""
    import tilemaxsim_amd as tms
    (q, k, v), offsets, G = make([1, 2, 5, 32, 31, 0, 17, 8, 3, 3, 29], 2, 1, D, dt, seed=D)
    how = dict(causal=dict(prefix=0), bias=dict(slopes=torch.tensor([0.3, 0.01], device="cuda")), cap=dict(cap=5.0)).get(kind, {})
    grads = torch.autograd.grad(tms.packed_attention(q, k, v, offsets, **how), (q, k, v), G)
    monkeypatch.setitem(base.U, dt, base.U[dt] ** 2)
    want, off = reference(q, k, v, offsets, G, **how)
    none = torch.zeros_like(want[0])
    close((none, *grads), (none, *want[1:]), (none, *off[1:]), f"two terms {kind} {D} {dt}")


@pytest.mark.parametrize("prefix", [None, 0, 700])
@pytest.mark.parametrize("dt", DT, ids=str)
def test_reach_with_masks(cuda, dt, prefix):
    """Two unequal texts, long enough for far keys to be left out: slopes from steep to flat, masks that end elsewhere."""
    slopes = torch.tensor([2.0, 0.25, 0.06, 0.0], device="cuda")
    qkv, offsets, G = make([3001, 1250], 4, 2, 64, dt, seed=12, behind=3)
    base.check(*qkv, offsets, G, f"reach {prefix} {dt}", slopes=slopes, prefix=prefix)


@pytest.mark.parametrize("prefix", [None, 300])
@pytest.mark.parametrize("dt", DT, ids=str)
def test_reach_of_norms_that_are_not_finite(cuda, dt, prefix):
    """NaN and infinite keys and queries in rows of no text: nothing is left out, in the output and in all gradients."""
    import tilemaxsim_amd as tms
    (q, k, v), offsets, G = make([2100, 30], 2, 1, 64, dt, seed=2, behind=3)
    slopes = torch.tensor([0.05, 0.3], device="cuda")
    want, off = reference(q, k, v, offsets, G, slopes=slopes, prefix=prefix)
    for value in (math.nan, math.inf):
        with torch.no_grad():
            q2, k2 = q.clone(), k.clone()
            q2[2131:], k2[2130:] = value, value
        ts = [q2.requires_grad_(True), k2.requires_grad_(True), v]
        out = tms.packed_attention(*ts, offsets, slopes=slopes, prefix=prefix)
        grads = torch.autograd.grad(out, ts, G)
        close((out.detach(), *grads), want, off, f"norms of {value} {dt}")


@pytest.mark.parametrize("dt", DT, ids=str)
def test_nothing_beside_the_tensors_is_written(cuda, dt):
    """Every output and workspace inside a buffer of sevens, through the C entries: texts in order, and offsets that are not."""
    from tilemaxsim_amd import _lib
    from tilemaxsim_amd.attention import _describe
    lib = _lib.load()
    T, H, KV, D, BAND = 300, 4, 2, 64, 1024

    def banded(n, kind):
        flat = torch.full((n + 2 * BAND,), 7, device="cuda", dtype=kind)
        return flat, flat[BAND:BAND + n]

    def kept(flat):
        return bool((flat[:BAND] == 7).all()) and bool((flat[-BAND:] == 7).all())

    for given in ([0, 130, 130, 290], [0, 200, 100, 300], [-50, 20, 4000], [300, 0], [5, 1 << 40, -(1 << 40), 9]):
        for prefix, slopes in ((None, None), (-7, 0.5), (40, None)):
            print(dt, given, prefix, slopes, flush=True)
            (q, k, v), _, G = make([T], H, KV, D, dt, seed=1)
            o = torch.tensor(given, device="cuda")
            p = None if prefix is None else torch.full((len(given) - 1,), prefix, device="cuda")
            s = None if slopes is None else torch.full((H,), slopes, device="cuda")
            at = _describe(q, k, v, o, p, s, 0.125, 0.0)
            nbytes = lib.tms_attention_workspace_size(len(given) - 1, T, H, KV, D)
            sizes = dict(out=(T * H * D, dt), low=(T * H * D, dt), stats=(lib.tms_attention_stats(T, H, KV), torch.float32), ws=(nbytes, torch.uint8),
                         dq=(T * H * D, dt), dk=(T * KV * D, dt), dv=(T * KV * D, dt))
            bufs = {name: banded(*size) for name, size in sizes.items()}
            ptr = {name: inner.data_ptr() for name, (_, inner) in bufs.items()}
            _lib.check(_lib.launch(q.device, lib.tms_packed_attention, at, ptr["out"], ptr["low"], ptr["stats"]))
            _lib.check(_lib.launch(q.device, lib.tms_packed_attention_grad, at, ptr["out"], ptr["low"], ptr["stats"], G.data_ptr(), ptr["ws"], nbytes,
                                   ptr["dq"], ptr["dk"], ptr["dv"]))
            torch.cuda.synchronize()
            assert all(kept(flat) for flat, _ in bufs.values()), [name for name, (flat, _) in bufs.items() if not kept(flat)]


@pytest.mark.parametrize("dt", DT, ids=str)
@pytest.mark.parametrize("H,KV", [(1, 1), (3, 1), (4, 2)])
def test_one_token_of_any_stride(cuda, H, KV, dt):
    """A single token, and a single head, as views whose other strides the kernels could not read in place: what a call on
    contiguous tensors gives."""
    import tilemaxsim_amd as tms
    for T in (1, 5):
        (q, k, v), offsets, G = make([T], H, KV, 64, dt, seed=T)
        want = tms.packed_attention(q, k, v, offsets)
        grads = torch.autograd.grad(want, (q, k, v), G)
        views = {
            "odd token": lambda t: torch.empty(T, t.shape[1] * 64 + 4, device="cuda", dtype=dt)[:, :t.shape[1] * 64].unflatten(1, (t.shape[1], 64)),
            "odd head": lambda t: torch.empty(T, t.shape[1], 68, device="cuda", dtype=dt)[..., :64],
            "far token": lambda t: torch.empty(1, 1, 64, device="cuda", dtype=dt).as_strided((1, 1, 64), ((1 << 22) + 8, 64, 1)) if T == t.shape[1] == 1 else torch.empty_like(t),
            "far head": lambda t: torch.empty(64 * T, device="cuda", dtype=dt).as_strided((T, 1, 64), (64, (1 << 40) + 3, 1)) if t.shape[1] == 1 else torch.empty_like(t),
        }
        for name, view in views.items():
            with torch.no_grad():
                xs = [view(t).copy_(t).detach().requires_grad_(True) for t in (q, k, v)]
            out = tms.packed_attention(*xs, offsets.cuda())
            assert torch.equal(out, want), (name, T)
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, xs, G), grads)), (name, T)
