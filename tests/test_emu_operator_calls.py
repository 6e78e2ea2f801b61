"""The GPU tests of unusual calls of the operators on the CPU emulator (what needs the GPU's sizes left out by name)."""
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
