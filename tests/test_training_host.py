"""CPU tests of the training operators: what the C ABI and the Python entry points refuse
before any HIP call, workspace sizes, and the rules that pick tiles and pieces
(``csrc/tms_train_rules.h``)."""
import ctypes
import itertools
import os
import shutil
import subprocess

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, BF16, F32 = 0, 1, 2
NONE, SUM, MEAN = 0, 1, 2


def call(name, *args):
    from tilemaxsim_amd import _lib
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.tms_last_error().decode()


# tms_maxsim_pairs(Qs, nQ, nq, d, D, B, nd, nway, qmask, dmask, dtype, ws, ws_bytes, scores, positions, stream)
PAIRS = dict(Qs=16, nQ=2, nq=32, d=128, D=16, B=6, nd=180, nway=0, qmask=None, dmask=None, dtype=F16, ws=None, ws_bytes=0,
             scores=16, positions=16, stream=None)


@pytest.mark.parametrize("change,status,says", [
    (dict(nQ=-1), 1, "negative"), (dict(nd=-1), 1, "negative"), (dict(nway=-3), 1, "negative"),
    (dict(dtype=3), 2, "dtype"), (dict(nway=2), 1, "nQ * nway"), (dict(nd=65536), 2, "tokens"),
    (dict(d=65537), 2, "65536"), (dict(nq=65537), 2, "65536"), (dict(nQ=65536), 2, "65535"), (dict(B=1 << 31), 2, "2^31"),
    (dict(Qs=None), 1, "NULL"), (dict(D=None), 1, "NULL"), (dict(scores=None), 1, "NULL"),
    (dict(positions=18), 1, "aligned"),
    (dict(d=77), 1, "workspace"), (dict(dtype=F32), 1, "workspace"), (dict(Qs=18), 1, "workspace"),  # rows that are laid out first
    (dict(d=77, ws=256, ws_bytes=100), 1, "workspace"), (dict(d=77, ws=264, ws_bytes=1 << 30), 1, "aligned"),
    (dict(nQ=0), 0, ""), (dict(B=0), 0, "")])
def test_pairs_c_abi(change, status, says):
    rc, msg = call("tms_maxsim_pairs", *{**PAIRS, **change}.values())
    assert rc == status and (rc == 0 or (says in msg and "tms_maxsim_pairs" in msg))


# tms_maxsim_pairs_grad(Qs, nQ, nq, d, D, B, nd, nway, positions, grad, dtype, ws, ws_bytes, dQ, dD, stream)
PAIRS_GRAD = dict(Qs=16, nQ=2, nq=32, d=128, D=16, B=6, nd=180, nway=0, positions=16, grad=16, dtype=F16, ws=None, ws_bytes=0,
                  dQ=16, dD=16, stream=None)


@pytest.mark.parametrize("change,status,says", [
    (dict(d=-1), 1, "negative"), (dict(dtype=7), 2, "dtype"), (dict(nd=65536), 2, "tokens"),
    (dict(positions=None), 1, "NULL"), (dict(grad=None), 1, "NULL"), (dict(D=None), 1, "NULL"), (dict(Qs=None), 1, "NULL"),
    (dict(positions=18), 1, "aligned"),
    (dict(nQ=64, B=4096), 1, "workspace"), (dict(nQ=64, B=4096, ws=256, ws_bytes=8), 1, "workspace"),
    (dict(nQ=64, B=4096, ws=260, ws_bytes=1 << 40), 1, "aligned"),
    (dict(dQ=None, dD=None), 0, "")])
def test_pairs_grad_c_abi(change, status, says):
    rc, msg = call("tms_maxsim_pairs_grad", *{**PAIRS_GRAD, **change}.values())
    assert rc == status and (rc == 0 or (says in msg and "tms_maxsim_pairs_grad" in msg))


def test_pairs_sizes():
    from tilemaxsim_amd import _lib
    lib = _lib.load()
    assert lib.tms_pairs_workspace_size(2, 32, 128, 6, 180, F16) == 0
    # three planes of rows of d up to a multiple of 32, queries' up to 256 bytes
    assert lib.tms_pairs_workspace_size(2, 3, 33, 6, 5, F32) == 3 * (768 + 6 * 5 * 64 * 2)
    assert lib.tms_pairs_workspace_size(2, 3, 33, 6, 5, BF16) == 768 + 6 * 5 * 64 * 2
    assert lib.tms_pairs_positions(2, 33, 6, 0) == 2 * 6 * 64 and lib.tms_pairs_positions(2, 32, 6, 3) == 6 * 32
    for bad in ((-1, 32, 128, 6, 180, F16), (2, 32, 128, 6, -1, F16)):
        assert lib.tms_pairs_workspace_size(*bad) == 0
    assert lib.tms_pairs_positions(-1, 32, 6, 0) == 0
    # over 128 blocks of query tokens, a document's sums stand in fp32 between the runs
    few, many = (lib.tms_pairs_grad_workspace_size(n, 32, 128, 6, 180, 0) for n in (128, 129))
    assert many - few >= 6 * 180 * 128 * 4
    assert lib.tms_pairs_grad_workspace_size(2, 0, 128, 6, 180, 0) == 0


SCALE = ctypes.c_double(1.0)
# tms_linear_cross_entropy(H, N, d, W, V, dtype, target, ignore, scale, reduction, ws, ws_bytes, loss, stats, stream)
LCE = dict(H=256, N=4, d=64, W=256, V=100, dtype=BF16, target=256, ignore=-100, scale=ctypes.addressof(SCALE), reduction=MEAN,
           ws=256, ws_bytes=1 << 40, loss=256, stats=256, stream=None)


def numbers(*values):
    return [ctypes.c_double(v) for v in values]


BAD_SCALES = numbers(0.0, -1.0, float("nan"), float("inf"))
LCE_REFUSED = [
    (dict(N=-1), 1, "negative"), (dict(d=-1), 1, "negative"), (dict(V=-1), 1, "negative"), (dict(dtype=5), 2, "dtype"),
    (dict(reduction=3), 1, "reduction"), (dict(scale=None), 1, "scale"), (dict(V=0), 1, "vocabulary"),
    (dict(d=65537), 2, "65536"), (dict(N=(1 << 24) + 1), 2, "2^24"), (dict(V=(1 << 28) + 1), 2, "2^28"),
    (dict(H=None), 1, "NULL"), (dict(W=None), 1, "NULL"), (dict(target=None), 1, "NULL"), (dict(stats=None), 1, "NULL"),
    (dict(H=264), 1, "16-byte"), (dict(W=258), 1, "16-byte"),
    (dict(ws=None), 1, "workspace"), (dict(ws=272), 1, "256-byte"), (dict(ws_bytes=100), 1, "workspace")]
LCE_REFUSED += [(dict(scale=ctypes.addressof(x)), 1, "scale") for x in BAD_SCALES]


@pytest.mark.parametrize("change,status,says", LCE_REFUSED + [(dict(loss=None), 1, "NULL"), (dict(N=0, reduction=NONE, loss=None), 0, "")])
def test_lce_c_abi(change, status, says):
    rc, msg = call("tms_linear_cross_entropy", *{**LCE, **change}.values())
    assert rc == status and (rc == 0 or (says in msg and "tms_linear_cross_entropy" in msg))


@pytest.mark.parametrize("change,status,says", LCE_REFUSED + [(dict(grad=None), 1, "NULL"), (dict(N=0), 0, ""), (dict(dH=None, dW=None), 0, "")])
def test_lce_grad_c_abi(change, status, says):
    args = {k: v for k, v in LCE.items() if k not in ("loss", "stats", "ws", "ws_bytes", "stream")}
    args.update(stats=256, grad=256, ws=256, ws_bytes=1 << 40, dH=256, dW=256, stream=None)
    rc, msg = call("tms_linear_cross_entropy_grad", *{**args, **change}.values())
    assert rc == status and (rc == 0 or (says in msg and "tms_linear_cross_entropy_grad" in msg))


def test_lce_workspace_sizes():
    from tilemaxsim_amd import _lib
    size = _lib.load().tms_lce_workspace_size
    assert size(0, 64, 100, BF16, 1) == 0 and size(4, -1, 100, BF16, 1) == 0 and size(4, 64, 0, BF16, 0) == 0
    for N, d, V in ((1, 768, 32000), (500, 256, 8000), (8192, 768, 131072)):
        fwd, bwd = size(N, d, V, BF16, 0), size(N, d, V, BF16, 1)
        assert 0 < fwd < N * V * 4 / 8 + (1 << 16)  # an eighth of the logits at most
        assert bwd < (1 << 31) and size(N, d, V, F32, 1) > bwd
    assert size(4, 77, 100, BF16, 0) > size(4, 80, 100, BF16, 0)  # odd rows are laid out first


class Grad(ctypes.Structure):
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p), ("n", ctypes.c_int64), ("src_dtype", ctypes.c_int32), ("dst_dtype", ctypes.c_int32)]


@pytest.mark.parametrize("entry,status,says", [
    ((16, 16, -1, F32, F32), 1, "negative"), ((16, 16, 5, 9, F32), 2, "fp16"), ((None, 16, 5, F32, F32), 1, "NULL"),
    ((16, 16, (1 << 44) + 1, F32, F32), 2, "large")])
def test_clip_c_abi(entry, status, says):
    table = (Grad * 2)(Grad(16, 16, 0, F16, F16), Grad(*entry))
    at, most = ctypes.addressof(table), numbers(1.0, -1.0, float("nan"))
    for name, args in (("tms_grad_norm", (at, 2, 2, 16, 1 << 20, 16, None)),
                       ("tms_grad_clip", (at, 2, 2, ctypes.addressof(most[0]), 16, 1 << 20, 16, None))):
        rc, msg = call(name, *args)
        assert rc == status and says in msg and name in msg
    good = ctypes.addressof((Grad * 1)(Grad(16, 16, 5, F32, F32)))
    for args, word in (((good, -1, 2, 16, 1 << 20, 16, None), "negative"), ((good, 1, 1, 16, 1 << 20, 16, None), "norm_type"),
                       ((None, 1, 2, 16, 1 << 20, 16, None), "NULL"), ((good, 1, 2, None, 1 << 20, 16, None), "workspace"),
                       ((good, 1, 2, 16, 8, 16, None), "workspace"), ((good, 1, 2, 16, 1 << 20, None, None), "NULL")):
        rc, msg = call("tms_grad_norm", *args)
        assert rc == 1 and word in msg


def test_clip_c_abi_of_the_scaled_tensors():
    keep = (Grad * 1)(Grad(16, None, 5, F32, F32)), (Grad * 1)(Grad(16, 16, 5, F32, 4)), (Grad * 1)(Grad(16, 16, 5, F32, F32))
    tables = [ctypes.addressof(t) for t in keep]
    most = numbers(1.0, -1.0, float("nan"))
    for table, limit, status, word in ((tables[0], most[0], 1, "NULL"), (tables[1], most[0], 2, "fp16"), (tables[2], most[1], 1, "max_norm"),
                                       (tables[2], most[2], 1, "max_norm")):
        rc, msg = call("tms_grad_clip", table, 1, 2, ctypes.addressof(limit), 16, 1 << 20, 16, None)
        assert rc == status and word in msg
    rc, msg = call("tms_grad_clip", tables[2], 1, 2, None, 16, 1 << 20, 16, None)
    assert rc == 1 and "max_norm" in msg


def test_clip_workspace_size():
    from tilemaxsim_amd import _lib
    size = _lib.load().tms_grad_workspace_size
    assert size(-1) == size(0) == size(1) == size(200_000) and size(1_000_000) > size(1)  # a partial a launch at least


def test_maxsim_pairs_python_errors():
    import tilemaxsim_amd as tms
    Q, D = torch.ones(2, 4, 32), torch.ones(3, 5, 32)
    with pytest.raises(TypeError, match="Qs"):
        tms.maxsim_pairs([1], D)
    with pytest.raises(ValueError, match="nQ, Nq, d"):
        tms.maxsim_pairs(Q[0], D)
    with pytest.raises(ValueError, match="width 32 != D width 31"):
        tms.maxsim_pairs(Q, D[..., :31])
    with pytest.raises(ValueError, match="documents for 3 queries"):
        tms.maxsim_pairs(Q, torch.ones(3, 2, 5, 32))
    with pytest.raises(TypeError, match="Qs is torch.float32, D is torch.float16"):
        tms.maxsim_pairs(Q, D.half())
    with pytest.raises(TypeError):
        tms.maxsim_pairs(Q.double(), D.double())
    with pytest.raises(ValueError, match="D_mask"):
        tms.maxsim_pairs(Q, D, torch.ones(3, 4, dtype=torch.bool))
    with pytest.raises(TypeError, match="Q_mask"):
        tms.maxsim_pairs(Q, D, None, torch.ones(2, 4))
    with pytest.raises(NotImplementedError, match="65535"):
        tms.maxsim_pairs(torch.ones(1, 1, 1), torch.ones(1, 65536, 1))
    with pytest.raises(ValueError, match="no CPU path"):
        tms.maxsim_pairs(Q, D)


def test_linear_cross_entropy_python_errors():
    import tilemaxsim_amd as tms
    H, W, t = torch.ones(3, 8), torch.ones(10, 8), torch.tensor([0, 1, 2])
    f = tms.linear_cross_entropy
    with pytest.raises(TypeError, match="target"):
        f(H, W, [0, 1, 2])
    with pytest.raises(ValueError, match=r"weight \(V, d\)"):
        f(H, W[:, :7], t)
    with pytest.raises(ValueError, match="target must be"):
        f(H, W, t[:2])
    with pytest.raises(ValueError, match="reduction"):
        f(H, W, t, reduction="max")
    for scale in (0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            f(H, W, t, scale=scale)
    for kind in (torch.float32, torch.bool):
        with pytest.raises(TypeError, match="integer"):
            f(H, W, t.to(kind))
    with pytest.raises(TypeError, match="weight is torch.float16"):
        f(H, W.half(), t)
    with pytest.raises(TypeError):
        f(H.double(), W.double(), t)
    with pytest.raises(ValueError, match="empty vocabulary"):
        f(H, W[:0], t)
    with pytest.raises(ValueError, match="no CPU path"):
        f(H, W, t)


def test_clip_python_errors():
    import tilemaxsim_amd as tms
    g = torch.ones(3)
    with pytest.raises(NotImplementedError, match="norm_type"):
        tms.grad_norm([g], 1.0)
    with pytest.raises(TypeError, match="expected tensors, got int"):
        tms.grad_norm([g, 3])
    with pytest.raises(TypeError, match="float64"):
        tms.grad_norm([g.double()])
    with pytest.raises(ValueError, match="no CPU path"):
        tms.grad_norm([None, g])
    for most in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            tms.clip_grad_norm_([g], most)
    with pytest.raises(ValueError, match="1 gradients and 2 tensors"):
        tms.clip_grad_norm_([g], 1.0, out=[g, g])
    with pytest.raises(ValueError, match="no CPU path"):
        tms.clip_grad_norm_(g, 1.0)
    assert float(tms.grad_norm([])) == 0 and float(tms.clip_grad_norm_([None], 1.0)) == 0


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    so = str(tmp_path_factory.mktemp("rules") / "train_rules.so")
    build = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                            os.path.join(REPO, "tilemaxsim_amd", "csrc"), os.path.join(REPO, "tests", "train_rules_c.cpp"), "-o", so],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    lib = ctypes.CDLL(so)
    i64, integer = ctypes.c_int64, ctypes.c_int
    lib.gemm_size_of.argtypes = [i64] * 3
    lib.gemm_time.argtypes = [integer] + [i64] * 4
    lib.gemm_time.restype = ctypes.c_double
    lib.lce_plan_of.argtypes = [i64, i64, i64, integer, ctypes.POINTER(i64)]
    return lib


def test_plan_bounds(plan):
    """Pieces cover the vocabulary, P fits its 2^29 terms (or is one block of 256 columns),
    and the sums of the splits are bounded."""
    out = (ctypes.c_int64 * 7)()
    sizes = (1, 2, 63, 64, 65, 255, 256, 257, 500, 1024, 1229, 8192, 100_000, 1 << 24)
    for N, V, d, planes in itertools.product(sizes, (1, 2, 255, 256, 257, 8000, 30011, 131_072, 1 << 20, 1 << 28), (0, 1, 8, 77, 768, 65536), (1, 3)):
        plan.lce_plan_of(N, V, d, planes, out)
        dp, rows, piece, splits, size_p, size_h, size_w = out
        assert dp % 8 == 0 and d <= dp < d + 9
        assert rows == 64 if N <= 64 else rows % 256 == 0 and N <= rows < N + 256
        assert piece % 256 == 0 and 256 <= piece <= -(-V // 256) * 256
        assert rows * piece * planes <= 1 << 29 or piece == 256
        assert 1 <= splits <= 64 and all(0 <= s <= 2 for s in (size_p, size_h, size_w))
        steps = piece // 64 * (6 if planes == 3 else 1)
        assert splits == 1 or splits * 2 <= steps


def test_plan_of_large_and_small_products(plan):
    assert plan.gemm_size_of(131_072, 8192, 12) == 0  # the large tile once it fills the chip
    assert plan.gemm_size_of(64, 64, 12) == 2
    out = (ctypes.c_int64 * 7)()
    plan.lce_plan_of(8192, 131_072, 768, 1, out)
    assert out[2] <= 65536 and out[4] == 0  # 1 GB of P at most, in large tiles
    plan.lce_plan_of(1024, 16384, 128, 1, out)
    assert out[2] == 16384 and out[3] > 1  # one piece, and dH's few tiles split over the vocabulary
    for size in (0, 1, 2):
        assert plan.gemm_time(size, 4096, 4096, 64, 1) >= plan.gemm_time(size, 256, 256, 64, 1)
