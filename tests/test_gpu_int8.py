"""int8 row quantiser and products: the integer sum is exact, so the whole error is that of a few fp32 roundings and one
rounding to the output type."""
import pytest
import torch

from tests import operator_ref as ref
from tests.conftest import emulating

pytestmark = pytest.mark.gpu


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def ints(seed, *shape):
    return torch.randint(-128, 128, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.int8)


def scales(seed, *shape):
    return (0.5 + torch.rand(*shape, generator=torch.Generator().manual_seed(seed))) * 0.01


def quant_ref(x):
    """The definition in IEEE fp32."""
    xf = x.float()
    s = xf.abs().amax(-1).clamp_min(1e-30) / 127.0
    return torch.round(xf / s.unsqueeze(-1)).clamp(-127, 127).to(torch.int8), s


def product(x, xs, w, ws):
    """Exact integer product in fp64 (|sum| < 2^31), scaled."""
    return (x.to(ref.F64) @ w.to(ref.F64).t()) * xs.to(ref.F64)[:, None] * ws.to(ref.F64)


def check_product(got, want, bias, what):
    total = want if bias is None else want + bias.to(ref.F64)
    # sum to fp32, two scalings, bias: four half steps of what they act on, then the output's own
    tol = 4 * ref.U32 * (want.abs() + (0 if bias is None else bias.to(ref.F64).abs()))
    ref.assert_within(got, total, tol + ref.half_step(got.dtype, total.abs() + tol), what)


# ---- quantiser ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (3, 16), (5, 1001), (2, 8192), (2, 8200), (1, 16384), (2, 16400)], ids=str)
def test_quantiser_is_the_fp32_formula_bit_for_bit(dev, dtype, shape):
    from batchgen_amd.quantization.int8 import int8_quant_rows
    x = rand(1, *shape, dtype=dtype) * 3
    x[0, : shape[1] // 2] = 0
    if shape[0] > 2:
        x[2] = 0
    q, s = int8_quant_rows(x.to(dev))
    q_ref, s_ref = quant_ref(x)
    assert torch.equal(q.cpu(), q_ref) and torch.equal(s.cpu(), s_ref)
    wide = torch.zeros(shape[0], shape[1] + 5, dtype=dtype)
    wide[:, 3:3 + shape[1]] = x
    q2, s2 = int8_quant_rows(wide.to(dev)[:, 3:3 + shape[1]])
    assert torch.equal(q2, q) and torch.equal(s2, s)


def test_quantiser_edges(dev):
    from batchgen_amd.quantization.int8 import int8_quant_rows
    x = torch.zeros(6, 40)
    x[0, 3] = float("nan")
    x[1, 3] = float("-inf")
    x[2] = torch.arange(40) * 1e-38                       # far below the floor
    x[3] = torch.finfo(torch.float32).max
    x[4] = torch.tensor([1.0, -1.0] * 20) * 127
    x[4, 1::4] = 0.5                                      # ties go to even
    x[4, 2::4] = 1.5
    q, s = int8_quant_rows(x.to(dev))
    assert not bool(torch.isfinite(s[:2]).any())
    q_ref, s_ref = quant_ref(x[2:])
    assert torch.equal(q[2:].cpu(), q_ref) and torch.equal(s[2:].cpu(), s_ref)
    lead, ls = int8_quant_rows(x[2:].view(2, 2, 40).to(dev))
    assert lead.shape == (2, 2, 40) and ls.shape == (2, 2) and torch.equal(lead.view(4, 40).cpu(), q_ref)
    assert int8_quant_rows(x[:0].to(dev))[1].shape == (0,)


# ---- dense -------------------------------------------------------------------------------------------------------------
# m, n, k: one token, tile edges on every side, K tails inside a stage, many rows
DENSE = [(1, 64, 256), (1, 33, 16), (2, 1, 48), (16, 64, 512), (17, 65, 272), (31, 100, 1024), (33, 129, 496), (64, 64, 1296),
         (65, 31, 64), (130, 257, 304), (257, 300, 144), (300, 512, 256), (20, 8200, 64), (33, 8200, 80), (700, 1300, 528), (1100, 700, 400)]


@pytest.mark.parametrize("shape", DENSE, ids=str)
def test_dense_product(dev, shape):
    from batchgen_amd.quantization.int8 import int8_linear
    m, n, k = shape
    x, w, xs, ws = ints(2, m, k), ints(3, n, k), scales(4, m), scales(5, n)
    want = product(x, xs, w, ws)
    bias = rand(6, n)
    for i, dtype in enumerate(ref.DTYPES):
        b = bias if (m + i) % 2 else None
        got = int8_linear(x.to(dev), w.to(dev), ws.to(dev), bias=None if b is None else b.to(dev), x_scale=xs.to(dev),
                          out_dtype=dtype)
        assert got.dtype == dtype
        check_product(got, want, b, f"int8_linear {shape} {dtype}")


# rows, elements between them, element the first starts at
@pytest.mark.parametrize("view", [(3, 64, 5), (1, 71, 3), (3, 72, 0), (3, 80, 16), (40, 70, 1), (2, 1 << 24, 0)], ids=str)
def test_rows_at_any_address_and_stride(dev, view):
    from batchgen_amd.quantization.int8 import int8_linear
    m, stride, first = view
    base = ints(50, (m - 1) * stride + 64 + first).to(dev)
    x = base.as_strided((m, 64), (stride, 1), first)
    w, xs, ws = ints(51, 33, 64).to(dev), scales(52, m).to(dev), scales(53, 33).to(dev)
    check_product(int8_linear(x, w, ws, x_scale=xs), product(*(t.cpu() for t in (x, xs, w, ws))), None, f"view {view}")
    xb = torch.randn(base.shape, generator=torch.Generator().manual_seed(54)).to(dev, torch.bfloat16).as_strided((m, 64), (stride, 1), first)
    assert torch.equal(int8_linear(xb, w, ws), int8_linear(xb.cpu().contiguous().to(dev), w, ws))


@pytest.mark.parametrize("shape", [(1, 200, 4096), (5, 64, 20000), (2, 100, 16400), (100, 70, 7168)], ids=str)
def test_dense_product_long_k(dev, shape):
    from batchgen_amd.quantization.int8 import int8_linear
    m, n, k = shape
    x, w, xs, ws = ints(7, m, k), ints(8, n, k), scales(9, m), scales(10, n)
    got = int8_linear(x.to(dev), w.to(dev), ws.to(dev), x_scale=xs.to(dev), out_dtype=torch.float32)
    check_product(got, product(x, xs, w, ws), None, f"long K {shape}")


def test_largest_sums_do_not_wrap(dev):
    from batchgen_amd.quantization.int8 import int8_linear
    k = 131056                                            # the largest multiple of 16 that is taken
    x = torch.full((2, k), -128, dtype=torch.int8)
    w = torch.full((3, k), -128, dtype=torch.int8)
    w[1] = 127
    one = torch.ones(3)
    got = int8_linear(x.to(dev), w.to(dev), one.to(dev), x_scale=one[:2].to(dev), out_dtype=torch.float32)
    check_product(got, product(x, one[:2], w, one), None, "largest sums")


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 96, 512), (7, 130, 1040), (70, 64, 272), (300, 260, 160)], ids=str)
def test_linear_quantises_and_multiplies(dev, dtype, shape):
    from batchgen_amd.quantization.int8 import int8_linear, int8_quant_rows
    m, n, k = shape
    x, w, ws, bias = rand(11, m, k, dtype=dtype), ints(12, n, k), scales(13, n), rand(14, n)
    got = int8_linear(x.to(dev), w.to(dev), ws.to(dev), bias=bias.to(dev))
    q, s = quant_ref(x)
    check_product(got, product(q, s, w, ws), bias, f"linear {shape}")
    q2, s2 = int8_quant_rows(x.to(dev))
    two = int8_linear(q2, w.to(dev), ws.to(dev), bias=bias.to(dev), x_scale=s2, out_dtype=dtype)
    assert torch.equal(got, two)
    lead = int8_linear(x.to(dev).view(1, m, k), w.to(dev), ws.to(dev), bias=bias.to(dev))
    assert lead.shape == (1, m, n) and torch.equal(lead[0], got)
    out = torch.empty_like(got)
    assert int8_linear(x.to(dev), w.to(dev), ws.to(dev), bias=bias.to(dev), out=out) is out and torch.equal(out, got)


def test_a_row_does_not_depend_on_its_batch(dev):
    """Whatever kernel the row count selects: the sum is an integer."""
    from batchgen_amd.quantization.int8 import int8_linear
    x, w, ws = rand(15, 400, 528, dtype=torch.bfloat16).to(dev), ints(16, 272, 528).to(dev), scales(17, 272).to(dev)
    whole = int8_linear(x, w, ws)
    for m in (1, 3, 16, 17, 40, 64, 65, 128, 129, 256, 257):
        assert torch.equal(int8_linear(x[:m], w, ws), whole[:m]), m
    wide = torch.zeros(400, 600, dtype=torch.bfloat16, device=x.device)
    wide[:, 7:535] = x
    assert torch.equal(int8_linear(wide[:, 7:535], w, ws), whole)
    q, s = torch.zeros(40, 1024, dtype=torch.int8, device=x.device), torch.ones(40, device=x.device)
    q[:, 16:544] = ints(18, 40, 528).to(dev)
    q[:, 5:6] = 9
    a = int8_linear(q[:, 16:544], w, ws, x_scale=s)
    assert torch.equal(a, int8_linear(q[:, 16:544].contiguous(), w, ws, x_scale=s))
    b = int8_linear(q[:, 5:533], w, ws, x_scale=s)        # rows at no 16-byte address are copied first
    assert torch.equal(b, int8_linear(q[:, 5:533].contiguous(), w, ws, x_scale=s))


def test_non_finite_token_gives_nan_in_its_row_only(dev):
    from batchgen_amd.quantization.int8 import int8_linear
    x, w, ws = rand(19, 5, 64), ints(20, 40, 64).to(dev), scales(21, 40).to(dev)
    clean = int8_linear(x.to(dev), w, ws)
    x[1, 7], x[3, 9] = float("nan"), float("inf")
    got = int8_linear(x.to(dev), w, ws)
    assert torch.equal(got[[0, 2, 4]], clean[[0, 2, 4]])
    assert not bool(torch.isfinite(got[[1, 3]]).any())


# ---- grouped -----------------------------------------------------------------------------------------------------------
# counts per expert, n, k
GROUPED = [
    ([1], 64, 256),
    ([0, 3, 0, 16, 17], 96, 272),
    ([33, 0, 64, 65, 5], 33, 144),
    ([0, 0, 0], 64, 64),
    ([130, 1, 300], 130, 256),
    ([257, 0, 40, 512], 272, 400),
]


def layout(counts, align, gap):
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + (c + align - 1) // align * align)
    return cu, cu[-1] + gap


@pytest.mark.parametrize("case", GROUPED, ids=str)
@pytest.mark.parametrize("align", [1, 16])
def test_grouped_product_and_fused_stage_1(dev, case, align):
    from batchgen_amd.moe.grouped_int8_moe import int8_fused_s1, int8_grouped_gemm
    counts, n, k = case
    e = len(counts)
    cu, rows = layout(counts, align, 3)
    x, xs = ints(22, rows, k), scales(23, rows)
    w, ws = ints(24, e, 2 * n, k), scales(25, e, 2 * n)
    seqlens, cus = torch.tensor(counts, dtype=torch.int32), torch.tensor(cu, dtype=torch.int32)
    want = torch.zeros(rows, 2 * n, dtype=ref.F64)
    live = torch.zeros(rows, dtype=torch.bool)
    for g, c in enumerate(counts):
        sl = slice(cu[g], cu[g] + c)
        want[sl] = product(x[sl], xs[sl], w[g], ws[g])
        live[sl] = True
    xs_dirty = xs.clone()
    xs_dirty[~live] = float("nan")                        # rows of no expert are not read ...
    xd, xsd, wd, wsd, sd, cd = (t.to(dev) for t in (x, xs_dirty, w, ws, seqlens, cus))
    for dtype in ref.DTYPES:
        held = torch.full((rows, 2 * n), 5.0, dtype=dtype, device=dev)
        got = int8_grouped_gemm(xd, xsd, wd, wsd, sd, cd, out=held)
        assert got is held and bool((held[~live.to(dev)] == 5.0).all())          # ... and not written
        check_product(got.cpu()[live], want[live], None, f"grouped {case} {dtype}")
        # gate and up as halves of the stack
        held = torch.full((rows, n), 5.0, dtype=dtype, device=dev)
        got = int8_fused_s1(xd, xsd, wd[:, :n], wsd[:, :n], wd[:, n:], wsd[:, n:], sd, cd, out=held)
        assert bool((held[~live.to(dev)] == 5.0).all())
        g64, u64 = want[live][:, :n], want[live][:, n:]
        h64 = g64 * torch.sigmoid(g64) * u64
        # gate and up: three half steps each; exp(-g) of an argument that is off by |g| half steps: the hardware
        # exponential's own ulp, the product with log2 e; sum, division, product: at most (4 |g| + 16) half steps
        tol = (4 * g64.abs() + 16) * ref.U32 * h64.abs() + torch.finfo(torch.float32).smallest_normal
        ref.assert_within(got.cpu()[live], h64, tol + ref.half_step(dtype, h64.abs() + tol), f"fused {case} {dtype}")


def test_counts_that_reach_past_the_rows_are_cut(dev):
    from batchgen_amd.moe.grouped_int8_moe import int8_grouped_gemm
    x, xs, w, ws = ints(26, 20, 64), scales(27, 20), ints(28, 2, 48, 64), scales(29, 2, 48)
    seqlens, cu = torch.tensor([8, 1000], dtype=torch.int32), torch.tensor([0, 8, 1008], dtype=torch.int32)
    got = int8_grouped_gemm(*(t.to(dev) for t in (x, xs, w, ws, seqlens, cu)))
    want = torch.cat([product(x[:8], xs[:8], w[0], ws[0]), product(x[8:], xs[8:], w[1], ws[1])])
    check_product(got, want, None, "cut counts")
    none = int8_grouped_gemm(*(t.to(dev) for t in (x, xs, w, ws, -seqlens, cu)), out=torch.ones(20, 48, device=dev))
    assert bool((none == 1).all())


def test_streams_and_empty_calls(dev):
    from batchgen_amd.moe.grouped_int8_moe import int8_grouped_gemm
    from batchgen_amd.quantization.int8 import int8_linear
    x, w, ws = rand(30, 100, 512, dtype=torch.bfloat16).to(dev), ints(31, 192, 512).to(dev), scales(32, 192).to(dev)
    want = int8_linear(x, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [int8_linear(x, w, ws) for _ in range(3)]
    here = [int8_linear(x, w, ws) for _ in range(3)]      # two calls at once share no scratch
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got + here)
    assert int8_linear(x[:0], w, ws).shape == (0, 192) and int8_linear(x, w[:0], ws[:0]).shape == (100, 0)
    z = torch.zeros(2, dtype=torch.int32, device=dev)
    out = int8_grouped_gemm(ints(33, 0, 64).to(dev), scales(34, 0).to(dev), ints(35, 2, 32, 64).to(dev),
                            scales(36, 2, 32).to(dev), z, z)
    assert out.shape == (0, 32)


@pytest.mark.skipif(emulating(), reason="graph capture needs the GPU")
@pytest.mark.parametrize("m", [1, 24, 200])
def test_in_a_graph(dev, m):
    from batchgen_amd.quantization.int8 import int8_linear
    x, w, ws = rand(37, m, 1024, dtype=torch.bfloat16).to(dev), ints(38, 320, 1024).to(dev), scales(39, 320).to(dev)
    int8_linear(x, w, ws)
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(int8_linear(x, w, ws))
        graphs.append(graph)
    for seed in (40, 41, 42):
        x.copy_(rand(seed, m, 1024))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = int8_linear(x, w, ws)
        assert all(torch.equal(h, want) for h in held)


def test_refusals(dev):
    from batchgen_amd.moe.grouped_int8_moe import int8_fused_s1, int8_grouped_gemm
    from batchgen_amd.quantization.int8 import int8_linear, int8_quant_rows
    x, w, ws = rand(43, 4, 64).to(dev), ints(44, 32, 64).to(dev), scales(45, 32).to(dev)
    q, s = int8_quant_rows(x)
    for bad in (lambda: int8_quant_rows(x.double()), lambda: int8_quant_rows(x.clone().requires_grad_(True)),
                lambda: int8_quant_rows(x, out=torch.empty(4, 63, dtype=torch.int8, device=dev)),
                lambda: int8_quant_rows(x, scale=torch.empty(3, device=dev)),
                lambda: int8_linear(x[:, :48], w, ws), lambda: int8_linear(x, w.float(), ws), lambda: int8_linear(x, w, ws[:31]),
                lambda: int8_linear(x[:, :40], w[:, :40].contiguous(), ws), lambda: int8_linear(x, w, ws, bias=ws[:3]),
                lambda: int8_linear(q, w, ws), lambda: int8_linear(x, w, ws, x_scale=s), lambda: int8_linear(q, w, ws, x_scale=s[:3]),
                lambda: int8_linear(x, w, ws, out_dtype=torch.float64), lambda: int8_linear(x, w, ws, out=torch.empty(4, 31, device=dev)),
                lambda: int8_linear(x.clone().requires_grad_(True), w, ws), lambda: int8_linear(x, w.t(), ws),
                lambda: int8_linear(torch.zeros(1, 131072, device=dev), torch.zeros(1, 131072, dtype=torch.int8, device=dev),
                                    ws[:1])):
        with pytest.raises(RuntimeError):
            bad()
    wide = (1 << 32) + 64                                 # its low 32 bits are a valid K
    for bad in (lambda: int8_quant_rows(x[0, 0].expand(1, wide)),
                lambda: int8_linear(q[0, 0].expand(1, wide), torch.empty(0, wide, dtype=torch.int8, device=dev), ws[:0], x_scale=s[:1]),
                lambda: int8_grouped_gemm(torch.empty(0, wide, dtype=torch.int8, device=dev), s[:0],
                                          torch.empty(1, 0, wide, dtype=torch.int8, device=dev), ws[:0].view(1, 0),
                                          torch.zeros(1, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev))):
        with pytest.raises(RuntimeError):
            bad()
    we, wse = w.view(1, 32, 64), ws.view(1, 32)
    n1 = torch.tensor([4], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    for bad in (lambda: int8_grouped_gemm(x, s, we, wse, n1, cu), lambda: int8_grouped_gemm(q, s[:3], we, wse, n1, cu),
                lambda: int8_grouped_gemm(q, s, w, ws, n1, cu), lambda: int8_grouped_gemm(q, s, we, wse[:, :31], n1, cu),
                lambda: int8_grouped_gemm(q, s, we, wse, n1.long(), cu), lambda: int8_grouped_gemm(q, s, we, wse, n1[:0], cu),
                lambda: int8_grouped_gemm(q, s, we, wse, n1, cu, out=torch.empty(4, 31, device=dev)),
                lambda: int8_grouped_gemm(q, s, we.transpose(1, 2), wse, n1, cu),
                lambda: int8_fused_s1(q, s, we, wse, we[:, :16], wse[:, :16], n1, cu)):
        with pytest.raises(RuntimeError):
            bad()
