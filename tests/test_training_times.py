"""CPU test: fp32 cross entropy picks its tiles (``csrc/tms_train_rules.h``) by the times that its products take: tiles of
64 x 64 of three planes have one workgroup a CU, those of 16-bit operands four."""
import ctypes
import itertools
import os
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    so = str(tmp_path_factory.mktemp("rules") / "lce_rules.so")
    build = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(REPO, "tilemaxsim_amd", "csrc"),
                            os.path.join(REPO, "tests", "lce_rules_c.cpp"), "-o", so], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    lib = ctypes.CDLL(so)
    i64, integer = ctypes.c_int64, ctypes.c_int
    lib.logits_size_of.argtypes = [i64, i64, i64, integer]
    lib.terms_time.argtypes = lib.product_time.argtypes = [integer, i64, i64, i64, integer, i64]
    lib.terms_time.restype = lib.product_time.restype = ctypes.c_double
    lib.plan_of.argtypes = [i64, i64, i64, integer, ctypes.POINTER(i64)]
    return lib


@pytest.mark.parametrize("N,V,d,large", [
    (500, 8000, 64, 7.48), (1024, 4000, 128, 11.56), (1000, 4000, 256, 18.16), (1000, 4000, 1024, 59.07), (2000, 8000, 64, 16.36), (2000, 8000, 256, 43.67),
    (128, 30000, 128, 11.60)])
def test_many_tiles_are_large(rules, N, V, d, large):
    """Measured in microseconds, tiles of 128; those of 64 took a fifth to a half longer."""
    assert rules.logits_size_of(N, V, d, 3) == 1
    assert abs(rules.terms_time(1, V, N, d, 3, 1) - large) <= 0.15 * large


@pytest.mark.parametrize("N,V,d,small", [
    (300, 500, 64, 3.96), (500, 2000, 64, 4.28), (400, 4000, 64, 6.20), (400, 4000, 256, 12.12), (600, 4000, 1024, 50.35), (700, 2000, 768, 27.36)])
def test_few_tiles_are_small(rules, N, V, d, small):
    """The same where tiles of 64 took less than those of 128."""
    assert rules.logits_size_of(N, V, d, 3) == 2
    assert abs(rules.terms_time(2, V, N, d, 3, 1) - small) <= 0.15 * small


def test_one_price(rules):
    """The plan's tiles are the ones that take least by the price of the products that the gated projection goes by, too."""
    out = (ctypes.c_int64 * 7)()
    for N, V, d in itertools.product((65, 500, 1024, 2048, 8192), (500, 4000, 30000), (64, 128, 768)):
        rules.plan_of(N, V, d, 3, out)
        dp, rows, piece, splits, size_p, size_h, size_w = out

        def time(size, m, n, k, s=1):
            t = rules.product_time(size, m, n, k, 3, s)
            assert t == rules.terms_time(size, m, n, k, 3, s)
            return t

        for size, m, n, k, s in ((size_p, piece, N, dp, 1), (size_w, dp, piece, N, 1), (size_h, dp, N, piece, splits)):
            assert time(size, m, n, k, s) == min(time(1, m, n, k, s), time(2, m, n, k, s))
