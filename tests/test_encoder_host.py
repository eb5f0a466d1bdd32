"""CPU tests of attention, the gated projection and AdamW: what the C ABI and the Python entry points
refuse before any HIP call, workspace sizes, and the rules that pick tiles, parts and splits."""
import ctypes
import itertools
import os
import random
import shutil
import subprocess

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, BF16, F32 = 0, 1, 2
NAN, INF = float("nan"), float("inf")


def call(name, *args):
    from tilemaxsim_amd import _lib
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.tms_last_error().decode()


# ---------------------------------------------------------------- attention

class Attention(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v")]
                + [(n, ctypes.c_int64) for n in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head")]
                + [(n, ctypes.c_void_p) for n in ("offsets", "prefix", "slopes")]
                + [(n, ctypes.c_int64) for n in ("texts", "tokens", "heads", "kv_heads", "width")]
                + [("scale", ctypes.c_double), ("cap", ctypes.c_double), ("dtype", ctypes.c_int64)])


GIVEN = dict(q=256, k=256, v=256, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, offsets=256, prefix=None,
             slopes=None, texts=2, tokens=100, heads=4, kv_heads=2, width=64, scale=0.125, cap=0.0, dtype=BF16)
REFUSED = [
    (dict(texts=-1), 1, "negative"), (dict(tokens=-1), 1, "negative"), (dict(heads=-4), 1, "negative"), (dict(width=-1), 1, "negative"),
    (dict(dtype=3), 2, "dtype"), (dict(width=48), 2, "32, 64, 96 or 128"), (dict(width=256), 2, "256"),
    (dict(heads=0), 1, "share"), (dict(kv_heads=0), 1, "share"), (dict(heads=5), 1, "share"),
    (dict(scale=0.0), 1, "scale"), (dict(scale=-1.0), 1, "scale"), (dict(scale=NAN), 1, "scale"), (dict(scale=INF), 1, "scale"),
    (dict(scale=1e-16), 1, "scale"), (dict(scale=1e16), 1, "scale"), (dict(cap=1e-16), 1, "cap"), (dict(cap=1e16), 1, "cap"),
    (dict(cap=-1.0), 1, "cap"), (dict(cap=NAN), 1, "cap"), (dict(cap=INF), 1, "cap"),
    (dict(tokens=1 << 31), 2, "too many"), (dict(texts=1 << 31), 2, "too many"), (dict(tokens=1 << 29), 2, "too many"),
    (dict(texts=1 << 23), 2, "too many"), (dict(heads=1 << 17, kv_heads=1), 2, "too many"),
    (dict(q=None), 1, "NULL"), (dict(k=None), 1, "NULL"), (dict(v=None), 1, "NULL"), (dict(offsets=None), 1, "NULL"),
    (dict(q=264), 1, "16-byte"), (dict(k=258), 1, "16-byte"), (dict(v=272 + 8), 1, "16-byte"),
    (dict(q_token=252), 1, "strides"), (dict(k_head=4), 1, "strides"), (dict(v_token=1), 1, "strides"),
    (dict(dtype=F32, q_token=258), 1, "strides"),
    (dict(q_token=-256), 2, "apart"), (dict(k_token=(1 << 22) + 8), 2, "apart"), (dict(heads=1 << 16, kv_heads=2, width=128), 2, "apart")]


@pytest.mark.parametrize("change,status,says", REFUSED)
def test_attention_c_abi(change, status, says):
    given = Attention(**{**GIVEN, **change})
    at = ctypes.addressof(given)
    for name, rest in (("tms_packed_attention", (256, None, None, None)),
                       ("tms_packed_attention_grad", (256, 256, 256, 256, 256, 1 << 40, 256, 256, 256, None))):
        rc, msg = call(name, at, *rest)
        assert rc == status and says in msg and name in msg, msg


def test_attention_c_abi_tensors():
    given, other = Attention(**GIVEN), Attention(**{**GIVEN, "dtype": F32})
    at, fp32 = ctypes.addressof(given), ctypes.addressof(other)
    for args, word in (((at, None, None, None, None), "NULL"), ((at, 264, None, None, None), "aligned"), ((at, 256, 8, None, None), "aligned"),
                       ((at, 256, None, 260, None), "aligned"), ((None, 256, None, None, None), "NULL")):
        rc, msg = call("tms_packed_attention", *args)
        assert rc == 1 and word in msg
    good = [256, 256, 256, 256, 256, 1 << 40, 256, 256, 256, None]
    for place, value, word in ((0, None, "NULL"), (1, None, "NULL"), (2, None, "NULL"), (3, None, "NULL"), (4, None, "workspace"),
                               (4, 272, "workspace"), (5, 100, "workspace"), (0, 264, "aligned"), (3, 8, "aligned"), (6, 4, "aligned"), (8, 20, "aligned")):
        rc, msg = call("tms_packed_attention_grad", at, *good[:place], value, *good[place + 1:])
        assert rc == 1 and word in msg, (place, value, msg)
    rc, msg = call("tms_packed_attention_grad", fp32, 256, None, 256, 256, None, 0, 256, None, None, None)
    assert rc == 1 and "workspace" in msg  # fp32 has no low
    for empty in (dict(tokens=0), dict(tokens=0, q=None, k=None, v=None, offsets=None)):
        kept = Attention(**{**GIVEN, **empty})
        none = ctypes.addressof(kept)
        assert call("tms_packed_attention", none, None, None, None, None)[0] == 0
        assert call("tms_packed_attention_grad", none, *[None] * 5, 0, *[None] * 4)[0] == 0
    assert call("tms_packed_attention_grad", at, 256, 256, 256, 256, 256, 1 << 40, None, None, None, None)[0] == 0  # nothing wanted


def test_attention_sizes():
    from tilemaxsim_amd import _lib
    lib = _lib.load()
    assert lib.tms_attention_stats(100, 4, 2) == 400 + 64 * 6 and lib.tms_attention_stats(5, 1, 1) == 8 + 128
    assert lib.tms_attention_stats(0, 4, 2) == 0 and lib.tms_attention_stats(5, -1, 1) == 0
    size = lib.tms_attention_workspace_size
    assert size(2, 100, 4, 4, 64) == 1792  # delta, up to 256 bytes
    assert size(2, 100, 4, 2, 64) == 1792 + 2 * 2 * 100 * 2 * 64 * 4  # two workgroups share a tile's heads
    assert size(2, 0, 4, 2, 64) == 0 and size(-1, 5, 4, 2, 64) == 0


def bf(*shape, **kw):
    return torch.zeros(*shape, dtype=torch.bfloat16, **kw)


Q, K, O = bf(10, 4, 64), bf(10, 2, 64), torch.tensor([0, 4, 10])


@pytest.mark.parametrize("change,error,says", [
    (dict(q=[1]), TypeError, "Tensor"), (dict(offsets=[0, 10]), TypeError, "Tensor"),
    (dict(q=bf(10, 256)), ValueError, "(T, H, D)"), (dict(v=bf(10, 2, 32)), ValueError, "(T, H, D)"), (dict(k=bf(9, 2, 64), v=bf(9, 2, 64)), ValueError, "(T, H, D)"),
    (dict(k=bf(10, 3, 64), v=bf(10, 3, 64)), ValueError, "share"), (dict(k=bf(10, 0, 64), v=bf(10, 0, 64)), ValueError, "share"),
    (dict(q=bf(10, 4, 48), k=bf(10, 2, 48), v=bf(10, 2, 48)), NotImplementedError, "48"),
    (dict(q=Q.double(), k=K.double(), v=K.double()), TypeError, "float16"), (dict(v=K.half()), TypeError, "float16"),
    (dict(offsets=torch.tensor([[0, 10]])), ValueError, "offsets"), (dict(offsets=torch.tensor([], dtype=torch.int64)), ValueError, "offsets"),
    (dict(offsets=torch.tensor([0.0, 10.0])), TypeError, "integer"), (dict(offsets=torch.tensor([False, True])), TypeError, "integer"),
    (dict(offsets=torch.tensor([0, 11])), ValueError, "ascend"), (dict(offsets=torch.tensor([-1, 10])), ValueError, "ascend"),
    (dict(offsets=torch.tensor([0, 6, 4])), ValueError, "ascend"),
    (dict(scale=0.0), ValueError, "scale"), (dict(scale=-1), ValueError, "scale"), (dict(scale=NAN), ValueError, "scale"),
    (dict(cap=0.0), ValueError, "cap"), (dict(cap=-2.0), ValueError, "cap"), (dict(cap=INF), ValueError, "cap"), (dict(cap=1e-16), ValueError, "cap"), (dict(scale=1e16), ValueError, "scale"),
    (dict(prefix=True), TypeError, "prefix"), (dict(prefix=1.5), TypeError, "prefix"), (dict(prefix=torch.tensor([1.0, 2.0])), TypeError, "prefix"),
    (dict(prefix=torch.tensor([1])), ValueError, "prefix"),
    (dict(slopes=torch.zeros(3)), ValueError, "slopes"), (dict(slopes=torch.zeros(4).half()), ValueError, "slopes"),
    (dict(slopes=torch.zeros(4, requires_grad=True)), NotImplementedError, "slopes"), (dict(slopes=[0.0] * 4), TypeError, "slopes"),
    (dict(), ValueError, "no CPU path")])
def test_attention_refusals(change, error, says):
    import tilemaxsim_amd as tms
    given = {**dict(q=Q, k=K, v=K, offsets=O), **change}
    with pytest.raises(error, match=says.replace("(", r"\(").replace(")", r"\)")):
        tms.packed_attention(given.pop("q"), given.pop("k"), given.pop("v"), given.pop("offsets"), **given)


# ---------------------------------------------------------------- gated projection

# tms_gated_linear(x, N, d, w_gate, w_up, F, dtype, activation, ws, ws_bytes, h, stream)
GATED = dict(x=256, N=100, d=64, w_gate=256, w_up=256, F=32, dtype=BF16, activation=0, ws=256, ws_bytes=1 << 40, h=256, stream=None)
GATED_REFUSED = [
    (dict(N=-1), 1, "negative"), (dict(d=-1), 1, "negative"), (dict(F=-1), 1, "negative"), (dict(dtype=4), 2, "dtype"),
    (dict(activation=3), 1, "activation"), (dict(d=0), 1, "no elements"), (dict(d=65537), 2, "65536"), (dict(N=(1 << 24) + 1), 2, "2^24"),
    (dict(F=(1 << 20) + 1), 2, "2^20"), (dict(x=None), 1, "NULL"), (dict(w_gate=None), 1, "NULL"), (dict(w_up=None), 1, "NULL"),
    (dict(x=264), 1, "16-byte"), (dict(w_gate=258), 1, "16-byte"), (dict(w_up=8), 1, "16-byte"),
    (dict(d=77, ws=None), 1, "workspace"), (dict(dtype=F32, N=200, ws=None), 1, "workspace"), (dict(d=77, ws=272), 1, "256-byte"),
    (dict(d=77, ws_bytes=10), 1, "workspace")]


@pytest.mark.parametrize("change,status,says", GATED_REFUSED + [(dict(h=None), 1, "NULL"), (dict(h=8), 1, "16-byte"), (dict(N=0), 0, ""), (dict(F=0), 0, "")])
def test_gated_c_abi(change, status, says):
    rc, msg = call("tms_gated_linear", *{**GATED, **change}.values())
    assert rc == status and (rc == 0 or (says in msg and "tms_gated_linear" in msg))


@pytest.mark.parametrize("change,status,says", GATED_REFUSED + [
    (dict(grad=None), 1, "NULL"), (dict(grad=8), 1, "16-byte"), (dict(dx=8), 1, "16-byte"), (dict(ws=None), 1, "workspace"), (dict(N=0), 0, ""),
    (dict(F=0), 0, ""), (dict(dx=None, dg=None, du=None), 0, "")])
def test_gated_grad_c_abi(change, status, says):
    args = {k: v for k, v in GATED.items() if k not in ("ws", "ws_bytes", "h", "stream")}
    args.update(grad=256, ws=256, ws_bytes=1 << 40, dx=256, dg=256, du=256, stream=None)
    rc, msg = call("tms_gated_linear_grad", *{**args, **change}.values())
    assert rc == status and (rc == 0 or (says in msg and "tms_gated_linear_grad" in msg))


def test_gated_sizes():
    from tilemaxsim_amd import _lib
    from tilemaxsim_amd.gated import FEW_TOKENS
    size = _lib.load().tms_gated_workspace_size
    assert size(0, 64, 32, BF16, 1) == 0 and size(5, 0, 32, BF16, 1) == 0 and size(5, 64, -1, F32, 0) == 0
    assert size(1000, 64, 32, BF16, 0) == 0 and size(1000, 77, 32, BF16, 0) > 0
    for dtype in (F16, BF16, F32):
        assert size(FEW_TOKENS, 77, 33, dtype, 0) == 0  # the Python layer asks for none
    assert size(FEW_TOKENS + 1, 77, 33, BF16, 0) > 0 and size(129, 77, 33, F32, 0) > 0
    assert size(1000, 64, 100, BF16, 1) >= 1000 * 2 * 128 * 2


@pytest.mark.parametrize("change,error,says", [
    (dict(x=1), TypeError, "Tensor"), (dict(x=bf(64, 3)), ValueError, "d"), (dict(x=bf(())), ValueError, "d"), (dict(wu=bf(5, 8)), ValueError, "d"),
    (dict(wg=bf(8), wu=bf(8)), ValueError, "d"), (dict(x=bf(4, 0), wg=bf(3, 0), wu=bf(3, 0)), ValueError, "no elements"),
    (dict(activation="relu"), ValueError, "activation"), (dict(wu=bf(6, 8).half()), TypeError, "float16"),
    (dict(x=bf(4, 8).double(), wg=bf(6, 8).double(), wu=bf(6, 8).double()), TypeError, "float16"), (dict(), ValueError, "no CPU path")])
def test_gated_refusals(change, error, says):
    import tilemaxsim_amd as tms
    given = {**dict(x=bf(4, 8), wg=bf(6, 8), wu=bf(6, 8), activation="silu"), **change}
    with pytest.raises(error, match=says):
        tms.gated_linear(*given.values())


# ---------------------------------------------------------------- AdamW

class Tensor(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("p", "g", "copy")] + [(n, ctypes.c_int64) for n in ("n", "at")]
                + [(n, ctypes.c_int32) for n in ("index", "p_dtype", "g_dtype", "copy_dtype")])


class State(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("m", "v", "m_exp", "v_exp", "steps", "factors", "norm", "lr_at")]
                + [(n, ctypes.c_int64) for n in ("size", "counters", "bits")]
                + [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "decay", "max_norm")])


KB = 1 << 10
STATE = dict(m=256, v=256, m_exp=256, v_exp=256, steps=256, factors=256, norm=None, lr_at=None, size=1024, counters=8, bits=8, lr=1e-3,
             beta1=0.9, beta2=0.999, eps=1e-8, decay=0.01, max_norm=0.0)
ONE = dict(p=64 * KB, g=128 * KB, copy=None, n=100, at=0, index=0, p_dtype=F32, g_dtype=BF16, copy_dtype=F16)


def adamw(tensors, **state):
    table = (Tensor * len(tensors))(*(Tensor(**t) for t in tensors))
    kept = State(**{**STATE, **state})
    return call("tms_adamw_step", ctypes.addressof(table), len(tensors), ctypes.addressof(kept), None)


@pytest.mark.parametrize("state,status,says", [
    (dict(size=-1), 1, "negative"), (dict(counters=-1), 1, "negative"), (dict(bits=16), 2, "8 or 32"), (dict(lr=-1.0), 1, "lr"), (dict(lr=NAN), 1, "lr"),
    (dict(beta1=1.0), 1, "betas"), (dict(beta2=-0.1), 1, "betas"), (dict(eps=-1.0), 1, "eps"), (dict(decay=INF), 1, "decay"),
    (dict(norm=256, max_norm=-1.0), 1, "max_norm"), (dict(norm=256, max_norm=NAN), 1, "max_norm"),
    (dict(m=None), 1, "NULL"), (dict(v=None), 1, "NULL"), (dict(steps=None), 1, "NULL"), (dict(factors=None), 1, "NULL"), (dict(m_exp=None), 1, "NULL"),
    (dict(m=264), 1, "aligned"), (dict(factors=8), 1, "aligned"), (dict(steps=4), 1, "aligned")])
def test_adamw_c_abi_state(state, status, says):
    rc, msg = adamw([ONE], **state)
    assert rc == status and says in msg and "tms_adamw_step" in msg


@pytest.mark.parametrize("tensors,status,says", [
    ([dict(n=-1)], 1, "negative"), ([dict(at=-128)], 1, "negative"), ([dict(index=-1)], 1, "negative"), ([dict(p_dtype=3)], 2, "fp16"),
    ([dict(g_dtype=-1)], 2, "fp16"), ([dict(copy=256 * KB, copy_dtype=9)], 2, "fp16"), ([dict(p=None)], 1, "NULL"), ([dict(g=None)], 1, "NULL"),
    ([dict(at=64)], 1, "place of its own"), ([dict(n=1025)], 1, "place of its own"), ([dict(at=1024)], 1, "place of its own"), ([dict(index=8)], 1, "place of its own"),
    ([dict(), dict(p=192 * KB, at=128)], 1, "place of its own"),  # the same counter
    ([dict(), dict(p=192 * KB, index=1)], 1, "place of its own"),  # the same states
    ([dict(n=129), dict(p=192 * KB, at=128, index=1)], 1, "place of its own"),
    ([dict(at=512), dict(p=192 * KB, index=1)], 1, "place of its own"),  # in no order
    ([dict(), dict(at=128, index=1)], 1, "overlap"),  # one parameter twice, as tied weights are listed
    ([dict(g=64 * KB + 40)], 1, "overlap"), ([dict(copy=64 * KB)], 1, "overlap"), ([dict(copy=128 * KB + 198)], 1, "overlap"),
    ([dict(), dict(p=256 * KB, g=64 * KB + 396, at=128, index=1, n=2)], 1, "overlap"),
    ([dict(copy=256 * KB), dict(p=256 * KB + 199, at=128, index=1)], 1, "overlap")])
def test_adamw_c_abi_tensors(tensors, status, says):
    rc, msg = adamw([{**ONE, **t} for t in tensors])
    assert rc == status and says in msg and "tms_adamw_step" in msg


def test_adamw_c_abi_none():
    state = State(**STATE)
    for count, status in ((0, 0), (2, 1), (-1, 1)):
        assert call("tms_adamw_step", None, count, ctypes.addressof(state), None)[0] == status
    assert call("tms_adamw_step", None, 0, None, None)[0] == 1
    for args, word in (((256, 256, 256, 256, 100, 256, 256, None), "blocks"), ((256, 256, 256, 256, -128, 256, 256, None), "blocks"),
                       ((None, 256, 256, 256, 128, 256, 256, None), "NULL"), ((256, 256, 256, 256, 128, 256, 8, None), "aligned")):
        rc, msg = call("tms_adamw_moments", *args)
        assert rc == 1 and word in msg
    assert call("tms_adamw_moments", None, None, None, None, 0, None, None, None)[0] == 0


def fake_state(shapes, bits=32):
    """A state without a GPU, for what is refused before one is needed."""
    import tilemaxsim_amd as tms
    s = tms.AdamWState.__new__(tms.AdamWState)
    s.bits, s.shapes = bits, [tuple(x) for x in shapes]
    s.sizes = [torch.Size(x).numel() for x in s.shapes]
    s.places = [128 * i for i in range(len(shapes))]
    s.size = 128 * len(shapes)
    s.m, s.v = torch.zeros(s.size), torch.zeros(s.size)
    s.m_exp = s.v_exp = None
    s.steps = torch.zeros(len(shapes), dtype=torch.int64)
    return s


@pytest.mark.parametrize("change,error,says", [
    (dict(state=None), TypeError, "AdamWState"), (dict(grads=[torch.zeros(3)]), ValueError, "2 parameters, 1 gradients"),
    (dict(copies=[None]), ValueError, "1 copies"), (dict(betas=(1.0, 0.9)), ValueError, "betas"), (dict(betas=(0.9, -0.1)), ValueError, "betas"),
    (dict(eps=-1.0), ValueError, "eps"), (dict(weight_decay=NAN), ValueError, "weight_decay"), (dict(lr=-1.0), ValueError, "lr"), (dict(lr=NAN), ValueError, "lr"),
    (dict(norm=torch.zeros(())), ValueError, "together"), (dict(max_norm=1.0), ValueError, "together"),
    (dict(norm=torch.zeros(()), max_norm=-1.0), ValueError, "max_norm"), (dict(norm=3.0, max_norm=1.0), TypeError, "Tensor"),
    (dict(params=[torch.zeros(3), 5]), TypeError, "parameters"), (dict(grads=[torch.zeros(3).double(), torch.zeros(2, 2)]), TypeError, "float16"),
    (dict(grads=[torch.zeros(3), torch.zeros(4)]), ValueError, r"gradients\[1\]"), (dict(params=[torch.zeros(2), torch.zeros(2, 2)]), ValueError, r"parameters\[0\]"),
    (dict(copies=[torch.zeros(2), None]), ValueError, r"copies\[0\]"), (dict(lr=torch.zeros(2)), ValueError, "lr"), (dict(lr=torch.zeros((), dtype=torch.float64)), ValueError, "lr"),
    (dict(norm=torch.zeros(2), max_norm=1.0), ValueError, "norm")])
def test_adamw_refusals(change, error, says, monkeypatch):
    import tilemaxsim_amd as tms
    from tilemaxsim_amd import adamw as module
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: None if t.device.type == "cpu" else t.device.index)
    given = {**dict(params=[torch.zeros(3), torch.zeros(2, 2)], grads=[torch.zeros(3), torch.zeros(2, 2)], state=fake_state([(3,), (2, 2)])), **change}
    monkeypatch.setattr(module._lib, "launch", lambda *a: pytest.fail("launched"))
    with pytest.raises(error, match=says):
        tms.adamw_(**given)


def test_adamw_state_refusals():
    import tilemaxsim_amd as tms
    for args, error, says in ((([torch.zeros(3)], 16), NotImplementedError, "8 or 32"), (([],), ValueError, "no parameters"), (([3],), TypeError, "Tensor"),
                              (([torch.zeros(3).long()],), TypeError, "float16"), (([torch.zeros(3)],), ValueError, "no CPU path")):
        with pytest.raises(error, match=says):
            tms.AdamWState(*args)
    s = fake_state([(3,)])
    for bad in ({}, {"steps": s.steps, "m": s.m}, {"steps": s.steps, "m": s.m, "v": s.v, "m_exp": s.m}):
        with pytest.raises(ValueError, match="expected"):
            s.load_state_dict(bad)
    with pytest.raises(ValueError, match="m must be"):
        s.load_state_dict({"steps": s.steps, "m": torch.zeros(3), "v": s.v})
    with pytest.raises(ValueError, match="v must be"):
        s.load_state_dict({"steps": s.steps, "m": s.m, "v": s.v.double()})
    s.load_state_dict({"steps": s.steps + 3, "m": s.m + 1, "v": s.v + 2})
    assert s.steps.tolist() == [3] and bool((s.m == 1).all()) and s.moments()[1] is s.v and s.views(s.m)[0].shape == (3,)


def test_forward_mode_is_refused():
    import tilemaxsim_amd as tms
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(10, 2, 32), torch.ones(10, 2, 32))
        with pytest.raises(NotImplementedError, match="forward mode"):
            tms.packed_attention(dual, dual, dual, torch.tensor([0, 10]))
        x = forward_ad.make_dual(torch.zeros(4, 8), torch.ones(4, 8))
        with pytest.raises(NotImplementedError, match="forward mode"):
            tms.gated_linear(x, torch.zeros(3, 8), torch.zeros(3, 8))


# ---------------------------------------------------------------- rules

@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    so = str(tmp_path_factory.mktemp("rules") / "rules.so")
    build = subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(REPO, "tilemaxsim_amd", "csrc"),
                            os.path.join(REPO, "tests", "encoder_rules_c.cpp"), "-o", so], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    lib = ctypes.CDLL(so)
    i64 = ctypes.c_int64
    lib.attn_slots_of.restype = lib.attn_parts_of.restype = i64
    lib.attn_slots_of.argtypes = [i64] * 3
    lib.attn_wide_of.argtypes = [i64] * 3
    lib.attn_parts_of.argtypes = [i64] * 4
    lib.gated_few_of.argtypes = [i64, i64, i64, ctypes.c_int]
    lib.gemm_split_of.argtypes = [i64, i64, i64, ctypes.c_int, ctypes.POINTER(i64)]
    return lib


def test_tiles_have_numbers_of_their_own(rules):
    """A text's tiles are numbered from floor(begin / rows) + its place on: none is shared, none is behind the last."""
    rng = random.Random(0)
    for rows, _ in itertools.product((64, 128), range(60)):
        B = rng.choice((0, 1, 2, 7, 200))
        most = rng.choice((0, 1, 63, 64, 65, 1000))
        lens = [rng.randint(0, 5)] + [rng.randint(0, most) for _ in range(B)] + [rng.randint(0, 300)]  # with what stands around the texts
        at, used = 0, set()
        for t, n in enumerate(lens):
            mine = {at // rows + t + j for j in range(-(-n // rows))}
            assert not mine & used
            used |= mine
            at += n
        assert max(used, default=-1) < rules.attn_slots_of(at, B, rows)


def test_parts_divide_the_heads(rules):
    for T, B, kv, many in itertools.product((1, 100, 5000, 1 << 20), (1, 40, 4000), (1, 2, 12), (1, 2, 3, 7, 12, 64)):
        parts = rules.attn_parts_of(T, B, kv, many)
        assert 1 <= parts <= many and many % parts == 0
        if rules.attn_slots_of(T, B, 64) * kv >= 512:
            assert parts == 1
    assert rules.attn_wide_of(16384, 2, 12) and not rules.attn_wide_of(16384, 128, 12) and not rules.attn_wide_of(2048, 1, 8)


def test_few_tokens(rules):
    """More tokens or larger weights never bring the kernel of few tokens back."""
    sizes = [(8, 8), (768, 2048), (1024, 2816), (2048, 5504), (4096, 11008), (65536, 1 << 20)]
    for f32 in (0, 1):
        few = [[rules.gated_few_of(N, d, F, f32) for d, F in sizes] for N in range(1, 140)]
        assert few[0][:4] == [1] * 4 and not any(few[128])
        assert all(a >= b for row in few for a, b in zip(row, row[1:])) and all(a >= b for one, other in zip(few, few[1:]) for a, b in zip(one, other))
    assert rules.gated_few_of(64, 1021, 4096, 0) and not rules.gated_few_of(65, 1021, 4096, 0)


def test_splits(rules):
    out = (ctypes.c_int64 * 2)()
    for m, n, k, planes in itertools.product((8, 256, 1024, 4096), (1, 500, 16384), (64, 1408, 8192, 1 << 20), (1, 3)):
        rules.gemm_split_of(m, n, k, planes, out)
        size, splits = out
        assert 0 <= size <= 2 and splits >= 1 and (splits == 1 or splits * 2 <= k // 64) and not (planes == 3 and size == 0)
    rules.gemm_split_of(256, 500, 1408, 3, out)
    assert out[1] > 1  # few tiles
    rules.gemm_split_of(1024, 1 << 20, 8192, 1, out)
    assert list(out) == [0, 1]


# ---------------------------------------------------------------- one token, one head, tangents

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_strides_of_one_token_or_head_do_not_matter(dtype):
    """Whatever stride a dimension of one element has, the C entry gets one that it takes, without a copy."""
    import struct
    from tilemaxsim_amd import attention
    step = 16 // torch.empty(0, dtype=dtype).element_size()

    def strides(*ts):
        given = attention._describe(*ts, torch.tensor([0, ts[0].shape[0]]), None, None, 1.0, 0.0)
        return struct.unpack("@3P6q3P5q2dq", given)[3:9]

    wide, tall = torch.zeros(1, 4 * 64 + 3, dtype=dtype), torch.zeros(5, 1, 64, dtype=dtype)
    views = [wide[:, :256].unflatten(1, (4, 64)), torch.zeros(1, 1, 67, dtype=dtype)[..., :64],
             torch.zeros(64, dtype=dtype).as_strided((1, 1, 64), ((1 << 22) + 8, 3, 1)), tall.as_strided((5, 1, 64), (64, 3, 1)),
             tall.as_strided((5, 1, 64), (64, 1 << 40, 1)), tall]
    for x in views:
        y = attention._rows(x)
        assert y.data_ptr() == x.data_ptr() and y.shape == x.shape
        for s in strides(y, y, y):
            assert s % step == 0
        assert all(0 <= s <= attention.MOST_STRIDE for s in strides(y, y, y)[::2])
    x = torch.zeros(2, 67, dtype=dtype)[:, None, :64]  # two tokens: an odd stride counts
    y = attention._rows(x)
    assert y.data_ptr() != x.data_ptr() and y.is_contiguous()


def test_tangents_of_slopes_are_refused():
    import tilemaxsim_amd as tms
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        slopes = forward_ad.make_dual(torch.zeros(4), torch.ones(4))
        with pytest.raises(NotImplementedError, match="forward mode"):
            tms.packed_attention(Q, K, K, O, slopes=slopes)
