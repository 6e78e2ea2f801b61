"""Ways of calling the token sort, the int8 products and the gated residual norm other than plainly with fresh operands."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def sort_api():
    from batchgen_amd.moe import token_sort
    return token_sort


def norm_api():
    from batchgen_amd.attention import gated_residual_norm
    return gated_residual_norm


def plan_for(dev, n=6, k=2, e=4, seed=1, **kw):
    ids = torch.randint(0, e, (n, k), generator=torch.Generator().manual_seed(seed))
    return sort_api().token_sort_plan(ids.to(dev), e, **kw)


# ---- a gradient of a gradient ---------------------------------------------------------------------------------------
NAMES = ("block", "residual", "post", "gate", "pre")


def norm_leaves(dev, h=24, needed=NAMES, without=()):
    ts = dict(block=rand(1, 4, h), residual=rand(2, 4, h), post=1 + 0.1 * rand(3, h), gate=torch.sigmoid(rand(4, h)),
              pre=1 + 0.1 * rand(5, h))
    return {m: None if m in without else t.to(dev).requires_grad_(m in needed) for m, t in ts.items()}


def norm_of(v):
    return norm_api().gated_residual_rmsnorm(v["block"], v["residual"], post_weight=v["post"], gate=v["gate"], pre_weight=v["pre"])


@pytest.mark.parametrize("of", NAMES)
@pytest.mark.parametrize("with_respect_to", NAMES)
@pytest.mark.parametrize("through", ["y", "normed"])
def test_norm_penalty_is_refused_with_a_constant_cotangent(dev, of, with_respect_to, through):
    """d/d(with_respect_to) of |d out.sum() / d(of)|^2 + sum(with_respect_to): the first term's share may be left out only
    where it is zero, by the same derivative of the plain formula in 64 bits."""
    def plain(v):
        i1 = torch.rsqrt(v["block"].square().mean(-1, keepdim=True) + 1e-5)
        y = v["residual"] + v["gate"] * (v["block"] * i1 * v["post"])
        return y, y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5) * v["pre"]

    def loss(v, f):
        out = f(v)[0 if through == "y" else 1]
        (g,) = torch.autograd.grad(out.sum(), v[of], create_graph=True, allow_unused=True)
        return v[with_respect_to].sum() + (0 if g is None else g.square().sum())
    v64 = {m: t.detach().cpu().double().requires_grad_(True) for m, t in norm_leaves("cpu").items()}
    (want,) = torch.autograd.grad(loss(v64, plain), v64[with_respect_to])
    depends = bool((want - 1).abs().max() > 1e-9)         # (a zero share is an exact zero but for rounding)
    v = norm_leaves(dev)
    total = loss(v, norm_of)
    if depends:
        with pytest.raises(RuntimeError, match="no gradient of its own"):
            torch.autograd.grad(total, v[with_respect_to])
    else:
        (got,) = torch.autograd.grad(total, v[with_respect_to])
        assert torch.equal(got, torch.ones_like(got))


@pytest.mark.parametrize("without", [("post",), ("gate",), ("post", "gate")], ids=str)
def test_norm_penalty_without_optional_operands(dev, without):
    v = norm_leaves(dev, without=without)
    y, n = norm_of(v)
    (g,) = torch.autograd.grad(n.sum(), v["block"], create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        (g.square().sum() + v["block"].sum()).backward()
    # y alone: linear in block without a norm behind it, and constant there if nothing else needs a gradient
    v = norm_leaves(dev, needed=("block",), without=without)
    (g,) = torch.autograd.grad(norm_of(v)[0].sum(), v["block"], create_graph=True)
    assert g.requires_grad == ("post" not in without)


def test_unsort_penalty_is_refused_with_a_constant_cotangent(dev):
    t, plan = sort_api(), plan_for(dev)
    rows, w = rand(7, plan.capacity, 8).to(dev).requires_grad_(True), rand(8, 6, 2).to(dev).requires_grad_(True)
    g_rows, g_w = torch.autograd.grad(t.unsort_tokens(rows, plan, w).sum(), (rows, w), create_graph=True)
    for g, leaf in ((g_rows, w), (g_w, rows)):            # d_rows depends on the weights, d_weights on the rows
        with pytest.raises(RuntimeError, match="no gradient of its own"):
            torch.autograd.grad(g.square().sum() + leaf.sum(), leaf, retain_graph=True)
    # through the sort: a token's gradient depends on the weights too
    x = rand(9, 6, 8).to(dev).requires_grad_(True)
    (g,) = torch.autograd.grad(t.unsort_tokens(t.sort_tokens(x, plan), plan, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(g.square().sum() + w.sum(), w)


def test_constant_first_gradients_stay_constants(dev):
    """Linear operations: with a constant cotangent and constant other operands nothing is refused."""
    t, plan = sort_api(), plan_for(dev)
    x, w = rand(10, 6, 8).to(dev).requires_grad_(True), rand(11, 6, 2).to(dev)
    rows = t.sort_tokens(x, plan)
    for out in (rows, t.unsort_tokens(rows, plan), t.unsort_tokens(rows, plan, w)):
        (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
        (again,) = torch.autograd.grad(out.sum(), x, retain_graph=True)
        assert not g.requires_grad and torch.equal(g, again)
        (total,) = torch.autograd.grad(x.sum() + g.square().sum(), x)
        assert torch.equal(total, torch.ones_like(total))
    # a cotangent that needs a gradient: refused, as before
    c = rand(12, plan.capacity, 8).to(dev).requires_grad_(True)
    (g,) = torch.autograd.grad(t.sort_tokens(x, plan), x, c, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(g.sum(), c)


# ---- forward mode ---------------------------------------------------------------------------------------------------
def calls_with_one_marked_operand(dev, mark):
    """(name, call) for every public operation and floating operand of it; ``mark`` makes the operand what is tested."""
    from batchgen_amd.moe.grouped_int8_moe import int8_fused_s1, int8_grouped_gemm
    from batchgen_amd.quantization.int8 import int8_linear, int8_quant_rows
    t, plan = sort_api(), plan_for(dev)
    i8 = lambda *s: torch.ones(*s, dtype=torch.int8, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    norm = dict(block=rand(1, 4, 32), residual=rand(2, 4, 32), post_weight=rand(3, 32), gate=rand(4, 32), pre_weight=rand(5, 32))
    ops = [
        ("sort_tokens", lambda x: t.sort_tokens(x, plan), dict(x=rand(6, 6, 8))),
        ("unsort_tokens", lambda rows, w: t.unsort_tokens(rows, plan, w), dict(rows=rand(7, plan.capacity, 8), w=rand(8, 6, 2))),
        ("unsort_tokens, cast weights", lambda rows, w: t.unsort_tokens(rows, plan, w),
         dict(rows=rand(7, plan.capacity, 8), w=rand(8, 6, 2).half())),
        ("gated_residual_rmsnorm", norm_api().gated_residual_rmsnorm, norm),
        ("gated_residual_rmsnorm_int8_quant", norm_api().gated_residual_rmsnorm_int8_quant, norm),
        ("int8_quant_rows", int8_quant_rows, dict(x=rand(9, 4, 32))),
        ("int8_linear", lambda x, ws, b: int8_linear(x, i8(8, 32), ws, bias=b), dict(x=rand(9, 4, 32), ws=rand(10, 8), b=rand(11, 8))),
        ("int8_linear, int8 rows", lambda xs, ws: int8_linear(i8(4, 32), i8(8, 32), ws, x_scale=xs), dict(xs=rand(9, 4), ws=rand(10, 8))),
        ("int8_grouped_gemm", lambda xs, ws: int8_grouped_gemm(i8(4, 32), xs, i8(1, 8, 32), ws, i32(4), i32(0, 4)),
         dict(xs=rand(9, 4), ws=rand(10, 1, 8))),
        ("int8_fused_s1", lambda xs, g, u: int8_fused_s1(i8(4, 32), xs, i8(1, 8, 32), g, i8(1, 8, 32), u, i32(4), i32(0, 4)),
         dict(xs=rand(9, 4), g=rand(10, 1, 8), u=rand(11, 1, 8))),
    ]
    for name, f, operands in ops:
        operands = {m: v.to(dev) for m, v in operands.items()}
        for marked in operands:
            yield f"{name}: {marked}", lambda f=f, o=operands, marked=marked: f(**{m: mark(v) if m == marked else v for m, v in o.items()})


def test_operands_with_a_tangent_are_refused(dev):
    from torch.autograd import forward_ad
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            for name, call in calls_with_one_marked_operand(dev, lambda v: forward_ad.make_dual(v, torch.ones_like(v))):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call()
                    pytest.fail(f"{name} dropped the tangent")
            for name, call in calls_with_one_marked_operand(dev, lambda v: v):     # none carries one: they run
                call()


# ---- a caller's output tensors --------------------------------------------------------------------------------------
def calls_with_out(dev):
    """(name, fresh tensors to write, call) for every public operation that writes a caller's tensors."""
    from batchgen_amd.moe.grouped_int8_moe import int8_fused_s1, int8_grouped_gemm
    from batchgen_amd.quantization.int8 import int8_linear, int8_quant_rows
    t, plan = sort_api(), plan_for(dev)
    i8 = lambda *s: torch.ones(*s, dtype=torch.int8, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    f = lambda seed, *s: rand(seed, *s).to(dev)
    zeros = lambda *s: torch.zeros(*s, device=dev)
    return [
        ("sort_tokens", [zeros(plan.capacity, 8)], lambda o: t.sort_tokens(f(1, 6, 8), plan, out=o)),
        ("unsort_tokens", [zeros(6, 8)], lambda o: t.unsort_tokens(f(1, plan.capacity, 8), plan, f(2, 6, 2), out=o)),
        ("norm", [zeros(4, 32)], lambda o: norm_api().gated_residual_rmsnorm_int8_quant(f(1, 4, 32), f(2, 4, 32),
                                                                                        pre_weight=f(3, 32), out=o)),
        ("quantiser", [i8(4, 32), zeros(4)], lambda q, s: int8_quant_rows(f(1, 4, 32), out=q, scale=s)),
        ("linear", [zeros(4, 8)], lambda o: int8_linear(f(1, 4, 32), i8(8, 32), f(2, 8), out=o)),
        ("linear, int8 rows", [zeros(4, 8)], lambda o: int8_linear(i8(4, 32), i8(8, 32), f(2, 8), x_scale=f(3, 4), out=o)),
        ("grouped", [zeros(4, 8)], lambda o: int8_grouped_gemm(i8(4, 32), f(1, 4), i8(1, 8, 32), f(2, 1, 8), i32(4), i32(0, 4), out=o)),
        ("fused", [zeros(4, 8)], lambda o: int8_fused_s1(i8(4, 32), f(1, 4), i8(1, 8, 32), f(2, 1, 8), i8(1, 8, 32), f(3, 1, 8),
                                                         i32(4), i32(0, 4), out=o)),
    ]


def test_an_earlier_graph_notices_that_its_tensor_was_overwritten(dev):
    for name, outs, call in calls_with_out(dev):
        for i, o in enumerate(outs):
            if not o.is_floating_point():
                continue
            leaf = o.clone().requires_grad_(True)
            held = leaf * 1.0                             # what an earlier graph saves
            loss = held.square().sum()
            with torch.no_grad():
                call(*(held if j == i else p for j, p in enumerate(outs)))
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
                pytest.fail(f"{name}: the backward pass used the new values")


def test_outputs_that_require_a_gradient_are_refused_in_grad_mode(dev):
    from torch.autograd import forward_ad
    for name, outs, call in calls_with_out(dev):
        for i, o in enumerate(outs):
            versions = [p._version for p in outs]
            if o.is_floating_point():
                with pytest.raises(RuntimeError, match="must not require"):
                    call(*(p.clone().requires_grad_(True) if j == i else p for j, p in enumerate(outs)))
                    pytest.fail(f"{name} took an output that requires a gradient")
                with pytest.raises(RuntimeError, match="no forward-mode derivative"), forward_ad.dual_level():
                    call(*(forward_ad.make_dual(p, torch.ones_like(p)) if j == i else p for j, p in enumerate(outs)))
            assert versions == [p._version for p in outs]                # refused: nothing written
        with torch.no_grad():
            call(*(p.clone().requires_grad_(p.is_floating_point()) for p in outs))
        call(*outs)
        assert all(p._version > 0 for p in outs), name


def test_outputs_of_inference_mode(dev):
    """Inference tensors have no version counter; ordinary ones are written in inference mode too."""
    with torch.inference_mode():
        cases = calls_with_out(dev)
        for _, outs, call in cases:
            call(*outs)
    ordinary = calls_with_out(dev)
    for (name, outs, call), (_, plain, same) in zip(cases, ordinary):
        call(*outs)                                       # and outside of it, where no autograd can hold them
        with torch.inference_mode():
            same(*plain)
        assert all(torch.equal(a, b) for a, b in zip(outs, plain)), name


def test_outputs_that_share_memory_with_an_operand(dev):
    from batchgen_amd.moe.grouped_int8_moe import int8_grouped_gemm
    from batchgen_amd.quantization.int8 import int8_linear, int8_quant_rows
    t, norm8 = sort_api(), norm_api().gated_residual_rmsnorm_int8_quant
    plan = t.token_sort_plan((torch.arange(63, -1, -1) % 8).view(64, 1).to(dev), 8)       # as many rows as tokens
    x = rand(1, 64, 16).to(dev)
    w = rand(2, 64, 1).to(dev)
    both = rand(3, 65 * 16).to(dev)
    q = torch.ones(16, 16, dtype=torch.int8, device=dev)
    ones = torch.ones(16, device=dev)
    one = torch.tensor([16], dtype=torch.int32, device=dev)
    seam = rand(4, 5, 32).to(dev)
    pre = torch.ones(32, device=dev)
    for bad in (lambda: t.sort_tokens(x, plan, out=x), lambda: t.unsort_tokens(x, plan, out=x),
                lambda: t.sort_tokens(both[:1024].view(64, 16), plan, out=both[16:].view(64, 16)),
                lambda: t.sort_tokens(both.as_strided((64, 4), (16, 1)), plan, out=both[:256].view(64, 4)),
                lambda: t.unsort_tokens(both[16:].view(64, 16), plan, out=both[:1024].view(64, 16)),
                lambda: t.unsort_tokens(rand(5, 64, 1).to(dev), plan, w, out=w),
                lambda: t.unsort_tokens(rand(5, 64, 1).to(dev), plan, out=plan.topk_pos.view(torch.float32)),
                lambda: norm8(seam[:4], seam[:4].clone(), pre_weight=pre, out=seam[1:]),
                lambda: norm8(seam[:4].clone(), seam[1:], pre_weight=pre, out=seam[:4]),
                lambda: norm8(seam[:1], seam[1:2], pre_weight=pre, out=pre.view(1, 32)),
                lambda: norm8(seam[:2].half(), seam[1:3].half(), gate=pre, pre_weight=seam[4], out=pre.view(torch.float16).view(2, 32)),
                lambda: int8_quant_rows(x, out=x.view(torch.int8)[:16].view(64, 16)),
                lambda: int8_quant_rows(x, scale=x[:4].view(64)),
                lambda: int8_quant_rows(x[:1, :4], out=ones[:1].view(torch.int8).view(1, 4), scale=ones[:1]),
                lambda: int8_linear(x[:1], q, ones, out=ones.view(1, 16)),
                lambda: int8_linear(x[:1], q, ones, bias=pre[:16], out=pre[:16].view(1, 16)),
                lambda: int8_linear(both.view(torch.int8)[:256].view(16, 16), q, ones, x_scale=ones, out=both[:256].view(16, 16)),
                lambda: int8_grouped_gemm(q, ones, q[:8].view(1, 8, 16), ones[:8].view(1, 8), one, one, out=q.view(torch.bfloat16).view(16, 8)),
                lambda: int8_grouped_gemm(q, ones, q[:1].view(1, 1, 16), ones[:1].view(1, 1), one, one, out=ones.view(16, 1))):
        before = [v.clone() for v in (x, w, both, q, ones, one, seam, pre, plan.topk_pos)]
        with pytest.raises(RuntimeError, match="share memory|whole memory"):
            bad()
        for a, b in zip(before, (x, w, both, q, ones, one, seam, pre, plan.topk_pos)):
            assert torch.equal(a, b)                      # refused before anything was written


def test_outputs_that_may_be_an_operand(dev):
    """The whole of block, residual or a full gate; the input of a product that is quantised first; memory beside an operand."""
    from batchgen_amd.quantization.int8 import int8_linear
    t, norm8 = sort_api(), norm_api().gated_residual_rmsnorm_int8_quant
    block, residual, gate, pre = (rand(s, 4, 32).to(dev) for s in (1, 2, 3, 4))
    want = norm8(block, residual, gate=gate, pre_weight=pre[0])
    for i in range(3):
        ops = [v.clone() for v in (block, residual, gate)]
        got = norm8(*ops[:2], gate=ops[2], pre_weight=pre[0], out=ops[i])
        assert got[0] is ops[i] and all(torch.equal(a, b) for a, b in zip(got, want)), i
    # a residual that is copied because it is not contiguous does not share memory with the output any more
    wide = torch.zeros(4, 64, device=dev)
    wide[:, ::2] = residual
    got = norm8(block, wide[:, ::2], gate=gate, pre_weight=pre[0], out=wide.view(-1)[:128].view(4, 32))
    assert torch.equal(got[0], want[0])
    x, w, ws = rand(5, 4, 32).to(dev), torch.ones(32, 32, dtype=torch.int8, device=dev), rand(6, 32).to(dev)
    want = int8_linear(x, w, ws)
    assert torch.equal(int8_linear(x, w, ws, out=x), want)
    plan = plan_for(dev)
    one = rand(7, 6 * 8 + plan.capacity * 8).to(dev)
    x = one[:48].view(6, 8)
    want = t.sort_tokens(x.clone(), plan)
    rows = t.sort_tokens(x, plan, out=one[48:].view(-1, 8).zero_())
    assert torch.equal(rows, want)


# ---- sizes ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [0, 1, 6])
def test_rows_of_width_zero(dev, n):
    t, plan = sort_api(), plan_for(dev, n=n)
    x = torch.zeros(n, 0, device=dev, requires_grad=True)
    w = rand(1, n, 2).to(dev).requires_grad_(True)
    rows = t.sort_tokens(x, plan)
    out = t.unsort_tokens(rows, plan, w)
    assert rows.shape == (plan.capacity, 0) and out.shape == (n, 0)
    gx, gw = torch.autograd.grad(out.sum(), (x, w))
    assert gx.shape == (n, 0) and gw.shape == (n, 2) and not bool(gw.any())
    held = torch.zeros(plan.capacity, 0, device=dev, requires_grad=True)
    (g,) = torch.autograd.grad(t.unsort_tokens(held, plan, w.detach()).sum(), held)
    assert g.shape == (plan.capacity, 0)


# ---- memory held for the backward pass -------------------------------------------------------------------------------
@pytest.mark.parametrize("rows_need,weights_need", [(True, None), (True, False), (False, True), (True, True)])
def test_unsort_saves_what_its_gradient_reads(dev, rows_need, weights_need):
    t, plan = sort_api(), plan_for(dev)
    rows = rand(1, plan.capacity, 8).to(dev).requires_grad_(rows_need)
    w = None if weights_need is None else rand(2, 6, 2).to(dev).requires_grad_(weights_need)
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda v: held.append(v.shape) or v, lambda v: v):
        out = t.unsort_tokens(rows, plan, w)
    assert held == ([rows.shape] if weights_need else []) + ([w.shape] if w is not None and rows_need else [])
    c = rand(3, 6, 8).to(dev)
    leaves = [v for v in (rows, w) if v is not None and v.requires_grad]
    grads = torch.autograd.grad(out, leaves, c)
    every = [rows.detach().requires_grad_(True), rand(2, 6, 2).to(dev) if w is None else w.detach().clone()]
    every[1].requires_grad_(True)
    want = torch.autograd.grad(t.unsort_tokens(every[0], plan, None if w is None else every[1]), every, c, allow_unused=True)
    for g, v in zip(grads, leaves):
        assert torch.equal(g, want[0 if v is rows else 1])


# ---- many groups, large weight stacks --------------------------------------------------------------------------------
def int8_operands(dev, rows, e, n, k, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.empty(e, n, k, dtype=torch.int8, device=dev)
    for part in w:                                        # one expert at a time: what randint makes is copied
        part.copy_(torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8, device=dev))
    return (torch.randint(-128, 128, (rows, k), generator=g, dtype=torch.int8, device=dev),
            0.5 + torch.rand(rows, generator=g, device=dev), w, 0.5 + torch.rand(e, n, generator=g, device=dev))


def offsets(counts, dev):
    c = torch.tensor(counts, dtype=torch.int32)
    cu = torch.zeros(len(counts) + 1, dtype=torch.int32)
    cu[1:] = c.cumsum(0)
    return c.to(dev), cu.to(dev), cu.tolist()


def check_groups(dev, counts, n, k, seed, groups=None):
    """Grouped and fused products against the dense product and the fused product of each expert by itself: the same
    integers, scaled by the same operations."""
    from batchgen_amd.moe.grouped_int8_moe import int8_fused_s1, int8_grouped_gemm
    from batchgen_amd.quantization.int8 import int8_linear
    c, cu, at = offsets(counts, dev)
    x, xs, w, ws = int8_operands(dev, at[-1], len(counts), n, k, seed)
    got = int8_grouped_gemm(x, xs, w, ws, c, cu, out_dtype=torch.float32)
    half = n // 2
    fused = int8_fused_s1(x, xs, w[:, :half], ws[:, :half], w[:, half:2 * half], ws[:, half:2 * half], c, cu, out_dtype=torch.float32)
    for g in range(len(counts)) if groups is None else groups:
        sl = slice(at[g], at[g + 1])
        if not counts[g]:
            continue
        assert torch.equal(got[sl], int8_linear(x[sl], w[g], ws[g], x_scale=xs[sl], out_dtype=torch.float32)), (g, counts[g])
        one, zero = offsets([counts[g]], dev)[:2]
        alone = int8_fused_s1(x[sl], xs[sl], w[g:g + 1, :half], ws[g:g + 1, :half], w[g:g + 1, half:2 * half],
                              ws[g:g + 1, half:2 * half], one, zero, out_dtype=torch.float32)
        assert torch.equal(fused[sl], alone), (g, counts[g])


def test_against_the_definition_once(dev):
    """What the comparisons of this section rest on: the dense product and one group's fused product against 64 bits."""
    from batchgen_amd.moe.grouped_int8_moe import int8_fused_s1
    from batchgen_amd.quantization.int8 import int8_linear
    from tests import operator_ref as ref
    x, xs, w, ws = int8_operands(dev, 40, 1, 66, 80, 1)
    one, cu, _ = offsets([40], dev)
    x64, w64 = x.cpu().double() * xs.cpu().double()[:, None], w[0].cpu().double() * ws[0].cpu().double()[:, None]
    want = x64 @ w64.t()
    got = int8_linear(x, w[0], ws[0], x_scale=xs, out_dtype=torch.float32)
    # sum to fp32 and two scalings: three half steps (fp64's own error is 2^-29 of one)
    ref.assert_within(got, want, 4 * ref.U32 * want.abs() + 1e-6 * ref.U32, "dense")
    fused = int8_fused_s1(x, xs, w[:, :33], ws[:, :33], w[:, 33:], ws[:, 33:], one, cu, out_dtype=torch.float32)
    g64, u64 = want[:, :33], want[:, 33:]
    h64 = g64 * torch.sigmoid(g64) * u64
    tol = (4 * g64.abs() + 16) * ref.U32 * h64.abs() + torch.finfo(torch.float32).smallest_normal
    ref.assert_within(fused, h64, tol + ref.half_step(torch.float32, h64.abs() + tol), "fused")


@pytest.mark.parametrize("groups", [64, 65, 200, 1024])
def test_many_groups(dev, groups):
    """More groups than the lanes that scan their tile counts: the last of each 64 and the first of the next hold rows."""
    counts = [0] * groups
    for i, v in ((0, 33), (1, 1), (63, 130), (64, 40), (65, 17), (127, 35), (128, 70), (199, 34), (511, 3), (960, 36), (1023, 129)):
        if i < groups:
            counts[i] = v
    counts[-1] = max(counts[-1], 34)
    check_groups(dev, counts, 34, 48, 7)


def test_many_groups_in_the_large_tiles_beyond_the_emulator(dev):
    g = torch.Generator().manual_seed(8)
    counts = (torch.randint(0, 420, (130,), generator=g) * (torch.rand(130, generator=g) < 0.9)).tolist()
    assert sum(counts) > 160 * len(counts)
    check_groups(dev, counts, 260, 272, 9)


def test_weight_stacks_beyond_the_last_level_cache(dev):
    """More than 256 MB of weights are streamed past the cache: whole stages and a K tail, one and two token tiles."""
    check_groups(dev, [0, 1, 16, 17, 32], 4001, 16016, 10)
    check_groups(dev, [40, 1, 0, 65, 32], 4001, 16016, 11)


def test_weight_stacks_beyond_32_bits(dev):
    for counts in ([0, 2, 0, 20], [1, 0, 0, 70]):         # the last expert's weights start at 4.9e9 bytes
        check_groups(dev, counts, 100000, 16384, 12)
        torch.cuda.empty_cache()


@pytest.mark.parametrize("create_graph", [False, True])
def test_checkpointed_block(dev, create_graph):
    """Under torch's checkpointing a backward pass may read what was saved only once."""
    from torch.utils.checkpoint import checkpoint
    t, plan = sort_api(), plan_for(dev)
    v = norm_leaves(dev, h=8)
    x, w = rand(1, 6, 8).to(dev).requires_grad_(True), rand(2, 6, 2).to(dev).requires_grad_(True)

    def block(x_, w_):
        out = t.unsort_tokens(t.sort_tokens(x_, plan), plan, w_)
        return norm_of(dict(v, block=out[:4]))[1]
    leaves = (x, w, v["post"], v["gate"])
    want = torch.autograd.grad(block(x, w).sum(), leaves)
    got = torch.autograd.grad(checkpoint(block, x, w, use_reentrant=False).sum(), leaves, create_graph=create_graph)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", ["residual_scale", "eps"])
def test_numbers_that_require_a_gradient_are_refused(dev, name):
    from torch.autograd import forward_ad
    block, residual, pre = rand(1, 4, 8).to(dev), rand(2, 4, 8).to(dev), rand(3, 8).to(dev)
    value = torch.tensor(0.5, device=dev)
    for f in (norm_api().gated_residual_rmsnorm, norm_api().gated_residual_rmsnorm_int8_quant):
        want = f(block, residual, pre_weight=pre, **{name: 0.5})
        for plain in (value, value.cpu(), 0.5):           # a constant is a number
            assert all(torch.equal(a, b) for a, b in zip(f(block, residual, pre_weight=pre, **{name: plain}), want))
        assert f(block, residual, pre_weight=pre, **{name: 1})[0].shape == block.shape
        with pytest.raises(RuntimeError, match="has no gradient"):
            f(block, residual, pre_weight=pre, **{name: value.clone().requires_grad_(True)})
        with pytest.raises(RuntimeError, match="forward-mode"), forward_ad.dual_level():
            f(block, residual, pre_weight=pre, **{name: forward_ad.make_dual(value, value)})
        with torch.no_grad():
            assert torch.equal(f(block, residual, pre_weight=pre, **{name: value.clone().requires_grad_(True)})[0], want[0])


def test_outputs_that_are_no_tensor_are_refused(dev):
    for name, outs, call in calls_with_out(dev):
        for i in range(len(outs)):
            with pytest.raises(RuntimeError, match="must be"):
                call(*(o.cpu().numpy() if j == i else o for j, o in enumerate(outs)))
                pytest.fail(name)
