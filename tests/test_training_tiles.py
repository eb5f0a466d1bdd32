"""CPU test: the tiles that the training operators' rules pick (``csrc/tms_train_rules.h``) fit the
buffers whatever the measured times say."""
import ctypes
import itertools
import os
import re
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("times", ["(double)size", "-(double)size", "1.0", "(double)((m + 255) / 256 * (size + 1))", "measured"])
def test_tiles_fit_the_softmax_buffer(tmp_path, times):
    """The softmax of a piece is stored in whole tiles: its rows and columns are whole tiles of
    the form that the rules pick, also if the times behind them were others."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    with open(os.path.join(REPO, "tilemaxsim_amd", "csrc", "tms_train_rules.h")) as f:
        text = f.read()
    head = re.search(r"inline double gemm_us\([^)]*\) \{\n", text)
    if times != "measured":
        text = text[:head.end()] + f"  return {times};\n" + text[head.end():]
    (tmp_path / "tms_train_rules.h").write_text(text)
    shutil.copy(os.path.join(REPO, "tests", "train_rules_c.cpp"), tmp_path)
    so = str(tmp_path / "rules.so")
    build = subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(tmp_path), str(tmp_path / "train_rules_c.cpp"), "-o", so],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    lib = ctypes.CDLL(so)
    i64 = ctypes.c_int64
    lib.lce_plan_of.argtypes = [i64, i64, i64, ctypes.c_int, ctypes.POINTER(i64)]
    out = (i64 * 7)()
    for N, V, d, planes in itertools.product((1, 2, 63, 64, 65, 128, 255, 257, 1229, 100_000), (1, 255, 257, 8000, 131_072, 1 << 22), (1, 64, 768), (1, 3)):
        lib.lce_plan_of(N, V, d, planes, out)
        _, rows, piece, _, size_p, _, _ = out
        side = {0: 256, 1: 128, 2: 64}[size_p]
        assert rows % side == 0 and piece % side == 0, (N, V, d, planes, list(out))
