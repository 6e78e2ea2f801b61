"""The gated residual norm against 64 bits: types, odd widths, every gate layout, missing norms, gradients against the
formula and against differences, the int8 form against the row quantiser."""
import pytest
import torch

from tests import operator_ref as ref
from tests.conftest import emulating

pytestmark = pytest.mark.gpu

EPS = 1e-5
SHAPES = [(1, 1), (3, 7), (2, 64), (5, 65), (17, 1001), (4, 7168), (2, 8192), (2, 8200), (1, 16384), (3, 16383)]
GATES = ["none", "channel", "token", "full"]


def api():
    from batchgen_amd.attention import gated_residual_norm
    return gated_residual_norm


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def operands(rows, h, dtype, gate, param=None, seed=1):
    param = param or dtype
    g = None
    if gate != "none":
        shape = {"channel": (h,), "token": (rows, 1), "full": (rows, h)}[gate]
        g = torch.sigmoid(rand(seed + 4, *shape)).to(param)
    return (rand(seed, rows, h, dtype=dtype) * 3, rand(seed + 1, rows, h, dtype=dtype) * 2,
            (1 + 0.2 * rand(seed + 2, h)).to(param), g, (1 + 0.2 * rand(seed + 3, h)).to(param))


def to(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


def call(dev, block, residual, post, gate, pre, scale):
    b, r, p, g, w = to(dev, block, residual, post, gate, pre)
    return api().gated_residual_rmsnorm(b, r, post_weight=p, gate=g, residual_scale=scale, pre_weight=w, eps=EPS)


def check_forward(got_y, got_n, dtype, ops, scale):
    block, residual, post, gate, pre = ops
    y, n, e_y, e_n = ref.norm_forward(block, residual, post, gate, scale, pre, EPS)
    ref.assert_within(got_y, y, e_y + ref.half_step(dtype, y) * (1 + ref.U32), "y")
    if pre is None:
        assert got_n is None
    else:
        ref.assert_within(got_n, n, e_n + ref.half_step(dtype, n.abs() + e_n), "normed")


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_forward(dev, shape, dtype):
    for i, gate in enumerate(GATES):
        ops = operands(*shape, dtype, gate, seed=10 * i + 1)
        check_forward(*call(dev, *ops, 0.7), dtype, ops, 0.7)


@pytest.mark.parametrize("missing", [(2,), (4,), (2, 4), (2, 3, 4)], ids=str)
def test_without_either_norm(dev, missing):
    ops = list(operands(6, 250, torch.bfloat16, "channel"))
    for i in missing:
        ops[i] = None
    check_forward(*call(dev, *ops, -1.5), torch.bfloat16, ops, -1.5)


@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 65), (33, 250), (17, 1001), (4, 8200), (1100, 24)], ids=str)
@pytest.mark.parametrize("dtype,param", [(torch.bfloat16, None), (torch.float16, torch.float32), (torch.float32, None)], ids=str)
@pytest.mark.parametrize("gate", GATES)
def test_gradients(dev, shape, dtype, param, gate):
    rows, h = shape
    ops = operands(rows, h, dtype, gate, param)
    dy, dn = rand(21, rows, h, dtype=dtype), rand(22, rows, h, dtype=dtype)
    check_grads(dev, ops, dtype, 0.7, dy, dn)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("only", range(5))
def test_gradient_of_one_leaf_alone(dev, only, gate):
    ops = operands(37, 264, torch.bfloat16, gate)
    if ops[only] is not None:
        dy, dn = rand(27, 37, 264, dtype=torch.bfloat16), rand(28, 37, 264, dtype=torch.bfloat16)
        check_grads(dev, ops, torch.bfloat16, 0.7, None if only == 4 else dy, dn, only)   # pre_weight acts on normed alone


# the widest rows, and several rows per block at a width between the two register layouts' limits
@pytest.mark.parametrize("shape,dtype,gate", [((5, 16384), torch.bfloat16, "channel"), ((3, 16384), torch.float32, "full"),
                                              ((700, 7168), torch.bfloat16, "channel"), ((515, 8192), torch.float16, "token")], ids=str)
def test_gradients_of_wide_rows(dev, shape, dtype, gate):
    check_grads(dev, operands(*shape, dtype, gate), dtype, 0.7, rand(25, *shape, dtype=dtype), rand(26, *shape, dtype=dtype))


@pytest.mark.parametrize("which", ["dy only", "dn only", "no post", "no pre", "neither norm"])
def test_gradients_of_partial_calls(dev, which):
    ops = list(operands(9, 130, torch.float32, "token"))
    dy, dn = rand(23, 9, 130), rand(24, 9, 130)
    if which in ("no post", "neither norm"):
        ops[2] = None
    if which in ("no pre", "neither norm"):
        ops[4], dn = None, None
    if which == "dy only":
        dn = None
    if which == "dn only":
        dy = None
    check_grads(dev, ops, torch.float32, -0.3, dy, dn)


def check_grads(dev, ops, dtype, scale, dy, dn, only=None):
    leaves = [None if t is None else t.clone().to(dev).requires_grad_(only in (None, i)) for i, t in enumerate(ops)]
    block, residual, post, gate, pre = leaves
    y, n = api().gated_residual_rmsnorm(block, residual, post_weight=post, gate=gate, residual_scale=scale, pre_weight=pre,
                                        eps=EPS)
    outs = [(o, g.to(dev)) for o, g in ((y, dy), (n, dn)) if g is not None]
    wanted = [t for t in leaves if t is not None and t.requires_grad]
    grads = torch.autograd.grad([o for o, _ in outs], wanted, [g for _, g in outs], allow_unused=False)
    want, mag = ref.norm_grads(*ops[:4], scale, ops[4], EPS, dy, dn)
    names = [m for m, t in zip(("block", "residual", "post", "gate", "pre"), leaves) if t is not None and t.requires_grad]
    c = ref.grad_roundings(ops[0].size(0))
    for name, leaf, got in zip(names, wanted, grads):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        tol = c * ref.U32 * mag[name]
        ref.assert_within(got, want[name], tol + ref.half_step(leaf.dtype, want[name].abs() + tol), f"gradient of {name}")


def test_gradient_against_differences(dev):
    """Directional differences of the op itself; the truncation error is that of the same quotient in 64 bits."""
    rows, h, scale, step = 5, 96, 0.8, 2.0 ** -6
    ops = operands(rows, h, torch.float32, "full")
    cy, cn = rand(31, rows, h), rand(32, rows, h)
    leaves = [t.clone().to(dev).requires_grad_(True) for t in ops]

    def f(ts):
        y, n = api().gated_residual_rmsnorm(ts[0], ts[1], post_weight=ts[2], gate=ts[3], residual_scale=scale,
                                            pre_weight=ts[4], eps=EPS)
        return y, n

    def loss64(ts):
        y, n, e_y, e_n = ref.norm_forward(*[t.to(ref.F64) for t in ts[:4]], scale, ts[4].to(ref.F64), EPS)
        noise = ((e_y + ref.half_step(torch.float32, y)) * cy.abs() + (e_n + ref.half_step(torch.float32, n)) * cn.abs()).sum()
        return (y * cy.to(ref.F64)).sum() + (n * cn.to(ref.F64)).sum(), noise
    y, n = f(leaves)
    grads = torch.autograd.grad((y, n), leaves, (cy.to(dev), cn.to(dev)))
    want, mag = ref.norm_grads(*ops[:4], scale, ops[4], EPS, cy, cn)
    for i, name in enumerate(("block", "residual", "post", "gate", "pre")):
        v = torch.sign(rand(40 + i, *ops[i].shape)) * 2.0 ** -1        # a power of two: x + step * v rounds by half a step
        up = [t + step * v if j == i else t for j, t in enumerate(ops)]
        down = [t - step * v if j == i else t for j, t in enumerate(ops)]
        with torch.no_grad():
            parts = [f([t.to(dev) for t in side]) for side in (up, down)]
        loss = [(p.cpu().to(ref.F64) * cy).sum() + (q.cpu().to(ref.F64) * cn).sum() for p, q in parts]
        (up64, noise_up), (down64, noise_down) = loss64(up), loss64(down)
        quotient, quotient64 = (loss[0] - loss[1]) / (2 * step), (up64 - down64) / (2 * step)
        slope = (grads[i].cpu().to(ref.F64) * v).sum()
        slope64 = (want[name] * v).sum()
        allowed = (quotient64 - slope64).abs() + (noise_up + noise_down) / (2 * step)
        allowed += ref.grad_roundings(rows) * ref.U32 * (mag[name] * v.abs()).sum()
        assert (quotient - slope).abs() <= allowed, (name, quotient, slope, allowed)


@pytest.mark.parametrize("shape", [(1, 16), (7, 1001), (16, 7168), (2, 16384)], ids=str)
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_int8_form_is_the_quantiser_of_the_stored_rows(dev, shape, dtype):
    from batchgen_amd.quantization.int8 import int8_quant_rows
    ops = operands(*shape, dtype, "channel")
    ops[0][0] = 0.0                                       # a zero block row: y = residual
    if shape[0] > 2:
        ops[1][2] = 0.0
        ops[0][2] = 0.0                                   # a zero row through both norms: scale of the floor, q = 0
    b, r, p, g, w = to(dev, *ops)
    y, n = api().gated_residual_rmsnorm(b, r, post_weight=p, gate=g, residual_scale=0.7, pre_weight=w, eps=EPS)
    y8, n8, q, s = api().gated_residual_rmsnorm_int8_quant(b, r, post_weight=p, gate=g, residual_scale=0.7, pre_weight=w,
                                                           eps=EPS)
    q_ref, s_ref = int8_quant_rows(n)
    assert torch.equal(y, y8) and torch.equal(n, n8) and torch.equal(q, q_ref) and torch.equal(s, s_ref)
    # the running residual updated in place
    keep = r.clone()
    y9, _, q9, _ = api().gated_residual_rmsnorm_int8_quant(b, keep, post_weight=p, gate=g, residual_scale=0.7, pre_weight=w,
                                                           eps=EPS, out=keep)
    assert y9 is keep and torch.equal(keep, y) and torch.equal(q9, q)


def test_non_finite_rows_stay_in_their_row(dev):
    ops = operands(4, 72, torch.float32, "none")
    ops[0][1, 5] = float("nan")
    ops[1][2, 6] = float("inf")
    b, r, p, g, w = to(dev, *ops)
    y, n, q, s = api().gated_residual_rmsnorm_int8_quant(b, r, post_weight=p, pre_weight=w, eps=EPS)
    clean = operands(4, 72, torch.float32, "none")
    y0, n0 = call(dev, clean[0], clean[1], clean[2], None, clean[4], 1.0)
    for row in (0, 3):
        assert torch.equal(y[row], y0[row]) and torch.equal(n[row], n0[row]) and bool(torch.isfinite(s[row]))
    for row in (1, 2):
        assert bool(torch.isnan(n[row]).any()) and not bool(torch.isfinite(s[row]))


def test_leading_axes_strides_and_streams(dev):
    b, r, p, g, w = to(dev, *operands(12, 88, torch.bfloat16, "channel"))
    want = api().gated_residual_rmsnorm(b, r, post_weight=p, gate=g, pre_weight=w)
    got = api().gated_residual_rmsnorm(b.view(3, 4, 88), r.view(3, 4, 88), post_weight=p, gate=g, pre_weight=w)
    assert all(torch.equal(x.view(12, 88), z) for x, z in zip(got, want)) and got[0].shape == (3, 4, 88)
    wide = torch.zeros(12, 100, dtype=b.dtype, device=b.device)
    wide[:, 3:91] = b
    got = api().gated_residual_rmsnorm(wide[:, 3:91], r, post_weight=p, gate=g, pre_weight=w)
    assert all(torch.equal(x, z) for x, z in zip(got, want))
    token = torch.rand(12, 1).to(dev, b.dtype)
    got = api().gated_residual_rmsnorm(b.view(3, 4, 88), r.view(3, 4, 88), gate=token.view(3, 4, 1), pre_weight=w)
    flat = api().gated_residual_rmsnorm(b, r, gate=token, pre_weight=w)
    assert torch.equal(got[1].view(12, 88), flat[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = api().gated_residual_rmsnorm(b, r, post_weight=p, gate=g, pre_weight=w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, z) for x, z in zip(got, want))
    # no rows
    empty = torch.zeros(0, 88, dtype=b.dtype, device=b.device).requires_grad_(True)
    pl = p.clone().requires_grad_(True)
    y, n = api().gated_residual_rmsnorm(empty, empty, post_weight=pl, pre_weight=w)
    grads = torch.autograd.grad((y.sum() + n.sum()), (empty, pl))
    assert grads[0].shape == (0, 88) and not bool(grads[1].any())


@pytest.mark.skipif(emulating(), reason="graph capture needs the GPU")
def test_forward_and_backward_in_a_graph(dev):
    rows, h = 40, 264
    leaves = [t.to(dev).requires_grad_(True) for t in operands(rows, h, torch.bfloat16, "channel")]
    cy, cn = rand(51, rows, h, dtype=torch.bfloat16).to(dev), rand(52, rows, h, dtype=torch.bfloat16).to(dev)

    def step():
        y, n = api().gated_residual_rmsnorm(leaves[0], leaves[1], post_weight=leaves[2], gate=leaves[3], residual_scale=0.7,
                                            pre_weight=leaves[4], eps=EPS)
        return (y.detach(), n.detach()) + torch.autograd.grad((y, n), leaves, (cy, cn))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, held = [], []
    for _ in range(2):                                    # two graphs that are replayed one into the other's gaps
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(step())
        graphs.append(graph)
    for seed in (53, 54, 55):
        with torch.no_grad():
            leaves[0].copy_(rand(seed, rows, h))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for got in held:
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_no_second_gradient(dev):
    b, r, p, g, w = [t.clone().to(dev).requires_grad_(True) for t in operands(4, 24, torch.float32, "channel")]
    y, n = api().gated_residual_rmsnorm(b, r, post_weight=p, gate=g, pre_weight=w)
    first = torch.autograd.grad((y.sum(), n.square().sum()), (b, p), create_graph=True)
    y, n = api().gated_residual_rmsnorm(b, r, post_weight=p, gate=g, pre_weight=w)
    plain = torch.autograd.grad((y.sum(), n.square().sum()), (b, p))
    assert all(torch.equal(u, v) for u, v in zip(first, plain))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first[0].sum(), b)


def test_refusals(dev):
    f, q = api().gated_residual_rmsnorm, api().gated_residual_rmsnorm_int8_quant
    b, r, p, g, w = to(dev, *operands(4, 24, torch.bfloat16, "channel"))
    for bad in (lambda: f(b, r[:2]), lambda: f(b, r.float()), lambda: f(b.double(), r.double()), lambda: f(b, r, post_weight=p[:8]),
                lambda: f(b, r, post_weight=p.half()), lambda: f(b, r, gate=g[:8]), lambda: f(b, r, gate=g.view(1, 24)),
                lambda: f(torch.zeros(1, 16392, device=dev), torch.zeros(1, 16392, device=dev)),
                lambda: q(b, r), lambda: q(b, r, pre_weight=w, out=r.float()), lambda: q(b, r, pre_weight=w, out=r[:2]),
                lambda: q(b, r, pre_weight=w.clone().requires_grad_(True))):
        with pytest.raises(RuntimeError):
            bad()
