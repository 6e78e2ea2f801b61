"""Token sort and unsort against plain loops in 64 bits: element types, odd widths, strides, padding tokens, experts
elsewhere, garbage in rows that hold no pair, gradients against the formula and against differences."""
import pytest
import torch

from tests import operator_ref as ref
from tests.conftest import emulating

pytestmark = pytest.mark.gpu

# n, k, h, e_total, e, start, align
SHAPES = [
    (0, 2, 8, 4, 4, 0, 1),
    (1, 1, 1, 1, 1, 0, 1),
    (1, 8, 130, 16, 16, 0, 1),
    (5, 3, 7, 6, 6, 0, 4),
    (33, 4, 257, 16, 4, 8, 16),
    (64, 32, 24, 64, 64, 0, 1),
    (130, 9, 515, 40, 40, 0, 8),
    (300, 8, 96, 600, 300, 150, 1),          # more local experts than the one-block index takes
]


def make_ids(n, k, e_total, dtype, seed, pad=0.0):
    g = torch.Generator().manual_seed(seed)
    if k <= e_total:
        ids = torch.rand(n, e_total, generator=g).topk(k, dim=1).indices
    else:
        ids = torch.randint(0, e_total, (n, k), generator=g)
    ids = ids.to(dtype)
    if pad and n:
        ids[torch.rand(n, generator=g) < pad] = -1
    return ids


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def api():
    from batchgen_amd.moe import token_sort
    return token_sort


def plan_of(ids, e, start, align, dev):
    plan = api().token_sort_plan(ids.to(dev), e, expert_start=start, row_align=align)
    counts, cu, pos = ref.sort_plan(ids, e, start, align)
    assert plan.counts.cpu().tolist() == counts and plan.cu_seqlens.cpu().tolist() == cu
    assert torch.equal(plan.topk_pos.cpu().long(), pos)
    assert plan.capacity >= cu[-1]
    return plan, counts, cu, pos


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", ref.DTYPES + [torch.int8], ids=str)
def test_sort_places_every_row_and_zeroes_the_rest(dev, shape, dtype):
    n, k, h, e_total, e, start, align = shape
    ids = make_ids(n, k, e_total, torch.int64 if n % 2 else torch.int32, 1, pad=0.1)
    plan, counts, cu, pos = plan_of(ids, e, start, align, dev)
    x = (rand(2, n, h) * 50).to(dtype)
    want = torch.zeros(plan.capacity, h, dtype=dtype)
    for t in range(n):
        for j in range(k):
            if pos[t, j] >= 0:
                want[pos[t, j]] = x[t]
    assert torch.equal(api().sort_tokens(x.to(dev), plan).cpu(), want)
    # a caller's buffer: rows without a pair keep what they held
    held = torch.full((plan.capacity, h), 7, dtype=dtype)
    out = held.clone().to(dev)
    live = torch.zeros(plan.capacity, dtype=torch.bool)
    live[pos[pos >= 0]] = True
    assert api().sort_tokens(x.to(dev), plan, out=out) is out
    assert torch.equal(out.cpu(), torch.where(live[:, None], want, held))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("weighted", [True, False])
def test_unsort_and_both_gradients(dev, shape, dtype, weighted):
    n, k, h, e_total, e, start, align = shape
    ids = make_ids(n, k, e_total, torch.int32 if n % 2 else torch.int64, 3, pad=0.1)
    plan, counts, cu, pos = plan_of(ids, e, start, align, dev)
    here = pos >= 0
    y = rand(4, plan.capacity, h, dtype=dtype)
    live = torch.zeros(plan.capacity, dtype=torch.bool)
    live[pos[here]] = True
    y[~live] = float("nan")                              # rows of no pair may hold anything
    w = torch.rand(n, k, generator=torch.Generator().manual_seed(5)) if weighted else None
    if weighted:
        w[~here] = float("inf")                          # and so may the weights of pairs without a row
    yd = y.clone().to(dev).requires_grad_(True)
    wd = w.clone().to(dev).requires_grad_(True) if weighted else None
    out = api().unsort_tokens(yd, plan, wd)
    want, mag = ref.unsort(y, pos, w)
    ref.assert_within(out, want, k * ref.U32 * mag + ref.half_step(dtype, want), "unsort")
    with torch.no_grad():
        again = api().unsort_tokens(yd, plan, wd, out=torch.empty_like(out))
    assert torch.equal(again, out.detach())

    g = rand(6, n, h, dtype=dtype)
    grads = torch.autograd.grad(out, [yd] + ([wd] if weighted else []), g.to(dev))
    dy = torch.zeros(plan.capacity, h, dtype=ref.F64)
    dw = torch.zeros(n, k, dtype=ref.F64)
    dw_mag = torch.zeros(n, k, dtype=ref.F64)
    for t in range(n):
        for j in range(k):
            if here[t, j]:
                dy[pos[t, j]] = (w[t, j].to(ref.F64) if weighted else 1.0) * g[t].to(ref.F64)
                terms = g[t].to(ref.F64) * y[pos[t, j]].to(ref.F64)
                dw[t, j], dw_mag[t, j] = terms.sum(), terms.abs().sum()
    # one product p, exact in 64 bits (24 + 24 bits).  The fp32 product and the rounding of it to fp16 may be one
    # instruction that rounds p once (error half a step of p) or two that round p to fp32 first (another U32 |p|)
    ref.assert_within(grads[0], dy, ref.U32 * dy.abs() + ref.half_step(dtype, dy), "row gradient")
    if weighted:
        assert grads[1].dtype == torch.float32
        # a dot product: at most h products and sums on any path
        ref.assert_within(grads[1], dw, (h + 1) * ref.U32 * dw_mag, "weight gradient")

    # the gradient of sort is the unweighted unsort
    x = rand(7, n, h, dtype=dtype).to(dev).requires_grad_(True)
    rows = api().sort_tokens(x, plan)
    d_rows = rand(8, plan.capacity, h, dtype=dtype)
    d_rows[~live] = float("nan")
    (dx,) = torch.autograd.grad(rows, x, d_rows.to(dev))
    want, mag = ref.unsort(d_rows, pos, None)
    ref.assert_within(dx, want, k * ref.U32 * mag + ref.half_step(dtype, want), "token gradient")


def test_gradients_against_differences(dev):
    """unsort is linear in the rows and in the weights, so a difference quotient is exact but for rounding."""
    n, k, h, e = 24, 4, 50, 8
    ids = make_ids(n, k, e, torch.int64, 9)
    plan = api().token_sort_plan(ids.to(dev), e)
    x = rand(10, n, h).to(dev).requires_grad_(True)
    w = torch.rand(n, k, generator=torch.Generator().manual_seed(11)).to(dev).requires_grad_(True)
    c = rand(12, n, h).to(dev)

    def f(x_, w_):
        rows = api().sort_tokens(x_, plan)
        return api().unsort_tokens(rows, plan, w_)
    gx, gw = torch.autograd.grad(f(x, w), (x, w), c)
    for leaf, grad, args in ((x, gx, lambda d: (x + d, w)), (w, gw, lambda d: (x, w + d))):
        v = rand(13, *leaf.shape).to(dev)
        with torch.no_grad():
            up, down = f(*args(0.5 * v)), f(*args(-0.5 * v))
        quotient = ((up.double() - down.double()) * c.double()).sum().cpu()
        slope = (grad.double() * v.double()).sum().cpu()
        # every output is off by at most 2 k half steps of the magnitudes that enter it (inputs' own rounding included)
        noise = 4 * k * ref.U32 * ((up.abs() + down.abs() + 4).double() * c.abs().double()).sum().cpu() * k
        noise += (h + k) * 2 * ref.U32 * (grad.abs().double() * v.abs().double()).sum().cpu() * 4
        assert abs(quotient - slope) <= noise, (quotient, slope, noise)


def test_strided_and_unaligned_inputs(dev):
    n, k, h, e = 19, 3, 45, 5
    ids = make_ids(n, k, e, torch.int32, 14)
    plan = api().token_sort_plan(ids.to(dev).t().contiguous().t(), e)      # ids that are not contiguous
    for dtype in ref.DTYPES:
        wide = rand(15, n, h + 9, dtype=dtype).to(dev)
        for x in (wide[:, 1:h + 1], wide[:, 9:], rand(16, h, n, dtype=dtype).to(dev).t()):
            rows = api().sort_tokens(x, plan)
            assert torch.equal(rows, api().sort_tokens(x.contiguous(), plan))
            back = api().unsort_tokens(rows.t().contiguous().t(), plan)
            assert torch.equal(back, api().unsort_tokens(rows, plan))
            xl = x.detach().clone()
            leaf = wide.detach().requires_grad_(True)
            (g,) = torch.autograd.grad(api().sort_tokens(leaf[:, 1:h + 1], plan).float().sum(), leaf)
            assert torch.equal(g[:, 1:h + 1].cpu(), torch.full((n, h), float(k), dtype=dtype))
            assert not bool(g[:, 0].any()) and not bool(g[:, h + 1:].any())
            del xl
    # weights of another type are cast, with their gradient
    w = torch.rand(n, k).to(dev, torch.bfloat16).requires_grad_(True)
    rows = api().sort_tokens(rand(17, n, h).to(dev), plan)
    (gw,) = torch.autograd.grad(api().unsort_tokens(rows, plan, w).sum(), w)
    assert gw.dtype == torch.bfloat16 and gw.shape == w.shape


def test_repeated_expert_and_every_token_on_one_expert(dev):
    ids = torch.tensor([[2, 2, 2], [0, 2, 2], [-1, 5, 2 ** 40]])
    plan, counts, cu, pos = plan_of(ids, 4, 0, 1, dev)
    x = rand(18, 3, 20).to(dev).requires_grad_(True)
    rows = api().sort_tokens(x, plan)
    out = api().unsort_tokens(rows, plan, torch.full((3, 3), 0.5).to(dev))
    want = torch.stack([1.5 * x[0], 1.5 * x[1], 0 * x[2]]).detach().cpu()
    ref.assert_within(out, want.double(), 4 * ref.U32 * want.double().abs(), "repeated experts")
    ids = torch.zeros(5000, 1, dtype=torch.int32)
    plan, counts, cu, pos = plan_of(ids, 3, 0, 64, dev)
    x = rand(19, 5000, 4).to(dev)
    assert torch.equal(api().sort_tokens(x, plan)[:5000], x)


def test_many_pairs_take_the_chunked_index(dev):
    n, k, e = 3000, 4, 64                                # beyond what one block indexes
    ids = make_ids(n, k, e, torch.int64, 20, pad=0.05)
    plan, counts, cu, pos = plan_of(ids, e, 0, 8, dev)
    x = rand(21, n, 16, dtype=torch.bfloat16).to(dev)
    rows = api().sort_tokens(x, plan)
    w = torch.ones(n, k).to(dev) / k
    assert torch.equal(api().unsort_tokens(rows, plan, w)[(pos >= 0).all(1).to(dev)], x[(pos >= 0).all(1).to(dev)])


def test_same_bits_every_time_and_on_another_stream(dev):
    n, k, h, e = 700, 6, 320, 32
    ids = make_ids(n, k, e, torch.int64, 22).to(dev)
    x = rand(23, n, h, dtype=torch.bfloat16).to(dev).requires_grad_(True)
    w = torch.rand(n, k).to(dev).requires_grad_(True)
    c = rand(24, n, h, dtype=torch.bfloat16).to(dev)

    def once():
        plan = api().token_sort_plan(ids, e)
        rows = api().sort_tokens(x, plan)
        out = api().unsort_tokens(rows, plan, w)
        return (rows, out) + torch.autograd.grad(out, (x, w), c)
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.skipif(emulating(), reason="graph capture needs the GPU")
def test_forward_and_backward_in_a_graph(dev):
    n, k, h, e = 96, 4, 264, 16
    ids = make_ids(n, k, e, torch.int64, 25).to(dev)
    x = rand(26, n, h, dtype=torch.bfloat16).to(dev).requires_grad_(True)
    w = torch.rand(n, k).to(dev).requires_grad_(True)
    c = rand(27, n, h, dtype=torch.bfloat16).to(dev)

    def step():
        plan = api().token_sort_plan(ids, e)
        out = api().unsort_tokens(api().sort_tokens(x, plan), plan, w)
        return (out.detach(),) + torch.autograd.grad(out, (x, w), c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (28, 29, 30):
        ids.copy_(make_ids(n, k, e, torch.int64, seed))
        with torch.no_grad():
            x.copy_(rand(seed, n, h))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_no_second_gradient(dev):
    """A gradient of a gradient is refused where it is asked for, not answered with a wrong one."""
    ids = make_ids(6, 2, 4, torch.int64, 31).to(dev)
    plan = api().token_sort_plan(ids, 4)
    x = rand(32, 6, 8).clone().to(dev).requires_grad_(True)
    w = torch.rand(6, 2).to(dev).requires_grad_(True)
    out = api().unsort_tokens(api().sort_tokens(x, plan), plan, w)
    gx, gw = torch.autograd.grad(out.square().sum(), (x, w), create_graph=True)
    plain = torch.autograd.grad(api().unsort_tokens(api().sort_tokens(x, plan), plan, w).square().sum(), (x, w))
    assert torch.equal(gx, plain[0]) and torch.equal(gw, plain[1])
    for g in (gx, gw):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x, retain_graph=True)


def test_refusals(dev):
    t = api()
    ids = torch.zeros(4, 2, dtype=torch.int32, device=dev)
    for bad in (lambda: t.token_sort_plan(ids.float(), 4), lambda: t.token_sort_plan(ids[0], 4),
                lambda: t.token_sort_plan(torch.zeros(2, 33, dtype=torch.int32, device=dev), 4),
                lambda: t.token_sort_plan(ids, 0), lambda: t.token_sort_plan(ids, 1025),
                lambda: t.token_sort_plan(ids, 4, row_align=3), lambda: t.token_sort_plan(ids, 4, row_align=0),
                lambda: t.token_sort_plan(ids, 4, expert_start=-1),
                # sizes whose low 32 bits are valid
                lambda: t.token_sort_plan(ids[:1, :1].expand((1 << 32) + 4, 1), 4), lambda: t.token_sort_plan(ids, (1 << 32) + 4),
                lambda: t.token_sort_plan(ids, 4, expert_start=1 << 32), lambda: t.token_sort_plan(ids, 4, row_align=1 << 32),
                lambda: t.sort_tokens(torch.zeros(1, 1, device=dev).expand(4, (1 << 32) + 4), t.token_sort_plan(ids, 4))):
        with pytest.raises(RuntimeError):
            bad()
    plan = t.token_sort_plan(ids, 4)
    x = torch.zeros(4, 8, device=dev)
    rows = torch.zeros(plan.capacity, 8, device=dev)
    for bad in (lambda: t.sort_tokens(x[:3], plan), lambda: t.sort_tokens(x[0], plan), lambda: t.sort_tokens(x.double(), plan),
                lambda: t.sort_tokens(x, plan, out=rows[:-1]), lambda: t.sort_tokens(x, plan, out=rows.half()),
                lambda: t.sort_tokens(x.requires_grad_(True), plan, out=rows),
                lambda: t.unsort_tokens(rows[:-1], plan), lambda: t.unsort_tokens(rows.to(torch.int8), plan),
                lambda: t.unsort_tokens(rows, plan, torch.zeros(4, 3, device=dev)),
                lambda: t.unsort_tokens(rows, plan, torch.zeros(4, 2, dtype=torch.int32, device=dev)),
                lambda: t.unsort_tokens(rows.requires_grad_(True), plan, out=torch.zeros(4, 8, device=dev))):
        with pytest.raises(RuntimeError):
            bad()
