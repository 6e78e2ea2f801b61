"""The GPU tests of unusual calls of the operators on the CPU emulator (what needs the GPU's sizes left out by name)."""
import ctypes
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_gpu_tests_of_operator_calls_pass_on_the_emulator():
    from tests.emu.build_emu import build
    build()
    cmd = [sys.executable, "-m", "pytest", "tests/test_gpu_operator_calls.py", "-m", "gpu", "-q", "--tb=short", "-p",
           "no:cacheprovider", "-k", "not beyond"]
    r = subprocess.run(cmd, cwd=ROOT, env=dict(os.environ, BGMOE_EMULATE="1", OMP_NUM_THREADS="2"), capture_output=True, text=True,
                       timeout=1500)
    tail = (r.stdout + r.stderr)[-3000:]
    assert r.returncode == 0, tail
    assert " passed" in r.stdout and "failed" not in r.stdout.splitlines()[-1], tail


def test_a_grouped_product_too_large_for_its_second_launch_is_refused_before_the_first():
    from batchgen_amd import _lib
    p, h = ctypes.c_void_p(64), _lib.lib()
    n, m, groups = 1 << 22, 10000, 63                     # 141 m-tiles of 128 rows x 32768 column tiles
    assert h.bgmoe_int8_grouped_gemm(p, p, p, 16 * n, p, n, p, p, groups, m, n, 16, p, 0, None) != 0
    assert "too large for one launch" in h.bgmoe_last_error().decode()
    assert h.bgmoe_int8_fused_s1(p, p, p, 16 * n, p, n, p, 16 * n, p, n, p, p, groups, m, n // 2 + 64, 16, p, 0, None) != 0
    assert "too large for one launch" in h.bgmoe_last_error().decode()
