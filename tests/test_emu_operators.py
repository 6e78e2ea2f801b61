"""The GPU test files of the token sort, the gated residual norm and the int8 products on the CPU emulator (as
tests/test_emu_rehearsal.py does for the older ones; graph captures skip themselves), and the C ABI's refusals, which
need no device: every argument error is found before anything is launched."""
import ctypes
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FILES = [("tests/test_gpu_token_sort.py", "not 3000"), ("tests/test_gpu_gated_residual_norm.py", "not 1100"),
         ("tests/test_gpu_int8_moe_block.py", ""), ("tests/test_gpu_int8.py", "not 20000 and not 7168 and not 512] and not largest_sums")]


@pytest.fixture(scope="module")
def rehearsals():
    from concurrent.futures import ThreadPoolExecutor
    from tests.emu.build_emu import build
    build()
    env = dict(os.environ, BGMOE_EMULATE="1", OMP_NUM_THREADS="2")

    def run(item):
        cmd = [sys.executable, "-m", "pytest", item[0], "-m", "gpu", "-q", "--tb=short", "-p", "no:cacheprovider", "-k", item[1]]
        return subprocess.run(cmd, cwd=ROOT, env=env, capture_output=True, text=True, timeout=1500)
    with ThreadPoolExecutor(len(FILES)) as ex:
        return dict(zip([f for f, _ in FILES], ex.map(run, FILES)))


@pytest.mark.parametrize("path", [f for f, _ in FILES], ids=[os.path.basename(f) for f, _ in FILES])
def test_gpu_test_files_pass_on_the_emulator(rehearsals, path):
    r = rehearsals[path]
    tail = (r.stdout + r.stderr)[-3000:]
    assert r.returncode == 0, tail
    assert " passed" in r.stdout and "failed" not in r.stdout.splitlines()[-1], tail


P = ctypes.c_void_p(64)          # a pointer that is never followed: the call is refused before


def refused(fn, *args, says):
    from batchgen_amd import _lib
    h = _lib.lib()
    assert getattr(h, fn)(*args) != 0, (fn, args)
    assert says in h.bgmoe_last_error().decode(), h.bgmoe_last_error()


def test_token_sort_refusals():
    f = "bgmoe_token_sort_index"
    refused(f, P, 0, 4, 0, 0, 4, 1, P, P, P, None, 0, None, says="bad sizes")
    refused(f, P, 0, 4, 2, 0, 4, 12, P, P, P, None, 0, None, says="power of two")
    refused(f, P, 0, 4, 2, 0, 1025, 1, P, P, P, None, 0, None, says="num_local_experts")
    refused(f, P, 0, 4, 2, -1, 4, 1, P, P, P, None, 0, None, says="expert_start")
    refused(f, P, 0, 1 << 30, 2, 0, 4, 1, P, P, P, None, 0, None, says="exceed int32")
    refused(f, P, 0, 4, 2, 0, 4, 1, P, None, P, None, 0, None, says="null output")
    refused(f, None, 0, 4, 2, 0, 4, 1, P, P, P, None, 0, None, says="null topk_ids")
    refused(f, P, 0, 1 << 16, 2, 0, 4, 1, P, P, P, None, 0, None, says="workspace")
    f = "bgmoe_token_sort_rows"
    refused(f, P, 16, 16, -1, 2, P, P, P, 4, 8, 0, P, None, says="negative")
    refused(f, P, 16, 16, 4, 33, P, P, P, 4, 8, 0, P, None, says="top-k")
    refused(f, None, 16, 16, 4, 2, P, P, P, 4, 8, 0, P, None, says="null pointer")
    f = "bgmoe_token_unsort"
    refused(f, P, 3, P, P, 4, 2, 8, P, None, says="element type")
    refused(f, P, 0, P, P, 4, 0, 8, P, None, says="top-k")
    refused(f, P, 0, None, P, 4, 2, 8, P, None, says="null pointer")
    f = "bgmoe_token_unsort_backward"
    refused(f, P, P, 9, P, P, 4, 2, 8, P, P, 4, 8, P, P, None, says="element type")
    refused(f, P, None, 0, P, P, 4, 2, 8, P, P, 4, 8, P, P, None, says="needs the rows")
    refused(f, P, P, 0, P, P, 4, 2, 8, None, P, 4, 8, P, P, None, says="null pointer")


def test_gated_norm_refusals():
    f = "bgmoe_gated_residual_norm"

    def args(**kw):
        a = dict(block=P, residual=P, dtype=0, post=P, gate=None, mode=0, scale=1.0, pre=P, fp32=0, rows=2, h=64, eps=1e-5, y=P,
                 normed=P, q=None, qs=None, i1=None, i2=None, st=None)
        a.update(kw)
        return tuple(a.values())
    refused(f, *args(dtype=4), says="element type")
    refused(f, *args(h=16385), says="row width")
    refused(f, *args(h=0), says="row width")
    refused(f, *args(mode=1), says="do not agree")
    refused(f, *args(mode=7, gate=P), says="gate_mode")
    refused(f, *args(y=None), says="null pointer")
    refused(f, *args(block=None), says="null pointer")
    refused(f, *args(pre=None), says="without pre_weight")
    refused(f, *args(normed=None), says="without an output")
    refused(f, *args(q=P), says="come together")
    f = "bgmoe_gated_residual_norm_backward"

    def back(**kw):
        a = dict(block=P, residual=P, dtype=0, post=P, gate=None, mode=0, scale=1.0, pre=P, fp32=0, rows=2, h=64, i1=P, i2=P, dy=P,
                 dn=P, db=P, dr=P, dpost=P, dgate=None, dpre=P, ws=P, nbytes=1 << 20, st=None)
        a.update(kw)
        return tuple(a.values())
    refused(f, *back(rows=0), says="no rows")
    refused(f, *back(post=None), says="d_post without")
    refused(f, *back(pre=None), says="d_pre without")
    refused(f, *back(dgate=P), says="d_gate without")
    refused(f, *back(i1=None), says="inv_post")
    refused(f, *back(nbytes=100), says="workspace")
    refused(f, *back(ws=None), says="workspace")
    refused(f, *back(pre=None, dpre=None), says="d_normed without")


def test_int8_refusals():
    refused("bgmoe_int8_quant_rows", P, 5, 64, 2, 64, P, P, None, says="element type")
    refused("bgmoe_int8_quant_rows", P, 0, 64, 2, 0, P, P, None, says="empty rows")
    refused("bgmoe_int8_quant_rows", P, 0, 64, 2, 64, None, P, None, says="null pointer")
    f = "bgmoe_int8_gemm"

    def args(**kw):
        a = dict(x=P, ldx=64, xs=P, w=P, ws=P, bias=None, m=4, n=8, k=64, out=P, dt=0, ldo=8, st=None)
        a.update(kw)
        return tuple(a.values())
    refused(f, *args(k=40), says="multiple of 16")
    refused(f, *args(k=131072), says="multiple of 16")
    refused(f, *args(m=-1), says="bad sizes")
    refused(f, *args(dt=3), says="output type")
    refused(f, *args(x=None), says="null pointer")
    refused(f, *args(w=ctypes.c_void_p(72)), says="16 bytes")
    refused(f, *args(ldx=72), says="16 bytes")
    refused(f, *args(ldx=48), says="x_row_stride")
    refused(f, *args(ldo=7), says="out_row_stride")
    refused("bgmoe_int8_linear", P, 0, 64, P, P, None, 4, 8, 64, P, 0, 8, None, 0, None, says="workspace")
    refused("bgmoe_int8_linear", P, 0, 64, P, P, None, 4, 8, 64, P, 0, 8, ctypes.c_void_p(8), 1 << 20, None, says="aligned")
    f = "bgmoe_int8_grouped_gemm"
    refused(f, P, P, P, 512, P, 8, P, P, 0, 4, 8, 64, P, 0, None, says="groups")
    refused(f, P, P, P, 520, P, 8, P, P, 1, 4, 8, 64, P, 0, None, says="16 bytes")
    refused(f, P, P, P, 512, P, 8, None, P, 1, 4, 8, 64, P, 0, None, says="null pointer")
    refused("bgmoe_int8_fused_s1", P, P, P, 512, P, 8, None, 512, P, 8, P, P, 1, 4, 8, 64, P, 0, None, says="null pointer")


@pytest.mark.parametrize("mode", [1, 2], ids=["loads land late", "loads land late, ordinary loads counted"])
@pytest.mark.parametrize("schedule", [0, 1, 2])
@pytest.mark.parametrize("m,n,k", [(5, 70, 1296), (33, 64, 800), (70, 40, 64), (200, 130, 656), (300, 300, 144)])
def test_int8_rings_wait_for_what_they_read(mode, schedule, m, n, k):
    """The asynchronous loads landing as late as the kernels' own waits allow, with the largest skew between waves that
    the barriers allow, in guarded buffers: a wait that is too lenient gives wrong sums, an access out of range ends the
    test process with a message."""
    import numpy as np
    from tests import emu
    h = emu.load()
    rng = np.random.default_rng(m + k)
    x, w = (emu.guarded(rng.integers(-128, 128, s, dtype=np.int8)) for s in ((m, k), (n, k)))
    xs, ws = (emu.guarded(rng.uniform(0.5, 1.5, s).astype(np.float32)) for s in (m, n))
    out = emu.guarded(np.zeros((m, n), np.float32))
    h.emu_set_async_mode(mode)
    h.emu_set_schedule(schedule)
    try:
        emu.ok(h, h.bgmoe_int8_gemm(emu.p(x), k, emu.p(xs), emu.p(w), emu.p(ws), None, m, n, k, emu.p(out), 2, n, None))
    finally:
        h.emu_set_async_mode(0)
        h.emu_set_schedule(0)
    want = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float32) * xs[:, None] * ws[None, :]
    assert np.array_equal(out, want)
