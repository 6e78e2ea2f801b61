"""The operators as a model uses them together: a mixture-of-experts block served in int8 (norm -> int8 rows -> sorted
tokens -> experts -> back with weights -> norm), each stage checked against its definition on the stage's own inputs,
and the trainable block (norm -> sort -> experts -> unsort -> norm), whose gradient is that of its parts in sequence."""
import pytest
import torch

from tests import operator_ref as ref
from tests.conftest import emulating

pytestmark = pytest.mark.gpu
EPS = 1e-5


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def quantised(seed, e, n, k):
    w = rand(seed, e, n, k) * 0.05
    s = w.abs().amax(2) / 127
    return torch.round(w / s[..., None]).to(torch.int8), s


def block(dev, n, h, inter, e_total, e, start, k, align, out_buffers):
    """One served block on n tokens; returns every stage's tensors."""
    from batchgen_amd.attention.gated_residual_norm import gated_residual_rmsnorm_int8_quant
    from batchgen_amd.moe.grouped_int8_moe import int8_fused_s1, int8_grouped_gemm
    from batchgen_amd.moe.token_sort import sort_tokens, token_sort_plan, unsort_tokens
    from batchgen_amd.quantization.int8 import int8_quant_rows
    bf = torch.bfloat16
    t = dict(attn=rand(1, n, h, dtype=bf), res=rand(2, n, h, dtype=bf), post=(1 + 0.1 * rand(3, h)).to(bf),
             pre=(1 + 0.1 * rand(4, h)).to(bf), gate=torch.sigmoid(rand(5, h)).to(bf))
    ids = torch.rand(n, e_total, generator=torch.Generator().manual_seed(6)).topk(k, 1).indices.to(torch.int32)
    if n > 3:
        ids[1] = -1                                       # a padding token of the batch
    t["ids"], t["w"] = ids, torch.softmax(rand(7, n, k), 1)
    t["gu"], t["gus"] = quantised(8, e, 2 * inter, h)
    t["down"], t["downs"] = quantised(9, e, h, inter)
    d = {name: v.clone().to(dev) for name, v in t.items()}

    def run():
        y, normed, q, qs = gated_residual_rmsnorm_int8_quant(d["attn"], d["res"], post_weight=d["post"], gate=d["gate"],
                                                             residual_scale=0.8, pre_weight=d["pre"], eps=EPS)
        plan = token_sort_plan(d["ids"], e, expert_start=start, row_align=align)
        kw = [{}, {}] if not out_buffers else [dict(out=torch.zeros(plan.capacity, h, dtype=torch.int8, device=dev)),
                                               dict(out=torch.zeros(plan.capacity, 1, device=dev))]
        rows, rs = sort_tokens(q, plan, **kw[0]), sort_tokens(qs.view(-1, 1), plan, **kw[1])
        hidden = int8_fused_s1(rows, rs, d["gu"][:, :inter], d["gus"][:, :inter], d["gu"][:, inter:], d["gus"][:, inter:],
                               plan.counts, plan.cu_seqlens, out=torch.zeros(plan.capacity, inter, dtype=bf, device=dev))
        hq, hs = int8_quant_rows(hidden)
        out = int8_grouped_gemm(hq, hs, d["down"], d["downs"], plan.counts, plan.cu_seqlens,
                                out=torch.zeros(plan.capacity, h, dtype=bf, device=dev))
        moe = unsort_tokens(out, plan, d["w"])
        y2, n2, q2, qs2 = gated_residual_rmsnorm_int8_quant(moe, y, post_weight=d["post"], pre_weight=d["pre"], eps=EPS)
        return dict(y=y, normed=normed, q=q, qs=qs, rows=rows, rs=rs, hidden=hidden, hq=hq, hs=hs, out=out, moe=moe, y2=y2,
                    n2=n2, q2=q2, qs2=qs2, pos=plan.topk_pos, counts=plan.counts, cu=plan.cu_seqlens)
    return t, d, run


@pytest.mark.parametrize("n,h,inter,e_total,e,start,k,align,buffers", [
    (1, 64, 32, 8, 8, 0, 2, 1, False), (5, 96, 48, 8, 4, 2, 3, 16, True), (70, 160, 80, 12, 12, 0, 4, 8, False),
    (300, 272, 144, 6, 3, 0, 2, 1, True)])
def test_served_block_stage_by_stage(dev, n, h, inter, e_total, e, start, k, align, buffers):
    t, d, run = block(dev, n, h, inter, e_total, e, start, k, align, buffers)
    g = {name: v.cpu() for name, v in run().items()}
    bf = torch.bfloat16
    y, nn, e_y, e_n = ref.norm_forward(t["attn"], t["res"], t["post"], t["gate"], 0.8, t["pre"], EPS)
    ref.assert_within(g["y"], y, e_y + ref.half_step(bf, y) * (1 + ref.U32), "first residual")
    ref.assert_within(g["normed"], nn, e_n + ref.half_step(bf, nn.abs() + e_n), "first norm")
    counts, cu, pos = ref.sort_plan(t["ids"], e, start, align)
    assert g["counts"].tolist() == counts and g["cu"].tolist() == cu and torch.equal(g["pos"].long(), pos)
    for tok in range(n):
        for j in range(k):
            if pos[tok, j] >= 0:
                assert torch.equal(g["rows"][pos[tok, j]], g["q"][tok]) and g["rs"][pos[tok, j], 0] == g["qs"][tok]
    for x in range(e):
        sl = slice(cu[x], cu[x] + counts[x])
        # the integer sums first, which 64 bits hold exactly (scaled operands would leave noise where a sum is 0)
        both = (g["rows"][sl].to(ref.F64) @ t["gu"][x].to(ref.F64).t()) * g["rs"][sl].to(ref.F64) * t["gus"][x].to(ref.F64)
        g64, u64 = both[:, :inter], both[:, inter:]
        h64 = g64 * torch.sigmoid(g64) * u64
        tol = (4 * g64.abs() + 16) * ref.U32 * h64.abs() + torch.finfo(torch.float32).smallest_normal
        ref.assert_within(g["hidden"][sl], h64, tol + ref.half_step(bf, h64.abs() + tol), "gate and up")
        s = g["hidden"][sl].float().abs().amax(-1).clamp_min(1e-30) / 127.0 if counts[x] else torch.zeros(0)
        assert torch.equal(g["hs"][sl], s)
        assert torch.equal(g["hq"][sl], torch.round(g["hidden"][sl].float() / s[:, None]).to(torch.int8))
        o64 = (g["hq"][sl].to(ref.F64) @ t["down"][x].to(ref.F64).t()) * s.to(ref.F64)[:, None] * t["downs"][x].to(ref.F64)
        tol = 4 * ref.U32 * o64.abs()
        ref.assert_within(g["out"][sl], o64, tol + ref.half_step(bf, o64.abs() + tol), "down")
    want, mag = ref.unsort(g["out"], pos, t["w"])
    ref.assert_within(g["moe"], want, k * ref.U32 * mag + ref.half_step(bf, want), "back with weights")
    y, nn, e_y, e_n = ref.norm_forward(g["moe"], g["y"], t["post"], None, 1.0, t["pre"], EPS)
    ref.assert_within(g["y2"], y, e_y + ref.half_step(bf, y) * (1 + ref.U32), "second residual")
    ref.assert_within(g["n2"], nn, e_n + ref.half_step(bf, nn.abs() + e_n), "second norm")


@pytest.mark.skipif(emulating(), reason="graph capture needs the GPU")
def test_served_block_in_a_graph(dev):
    """Captured once, replayed with other tokens and other routes in between eager calls."""
    t, d, run = block(dev, 96, 160, 96, 8, 8, 0, 2, 1, False)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for seed in (11, 12, 13):
        d["attn"].copy_(rand(seed, 96, 160))
        d["ids"].copy_(torch.rand(96, 8, generator=torch.Generator().manual_seed(seed)).topk(2, 1).indices)
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        for name in held:
            assert torch.equal(held[name], want[name]), name


def test_trainable_block(dev):
    """Gradients through the whole block are those of its parts called one after the other with the cotangents that
    autograd hands on: the same kernels, so the same bits."""
    from batchgen_amd.attention.gated_residual_norm import gated_residual_rmsnorm
    from batchgen_amd.moe.token_sort import sort_tokens, token_sort_plan, unsort_tokens
    n, h, e, k = 60, 72, 6, 3
    leaves = {name: v.clone().to(dev).requires_grad_(True) for name, v in dict(
        x=rand(1, n, h), res=rand(2, n, h), post=1 + 0.1 * rand(3, h), pre=1 + 0.1 * rand(4, h), gate=torch.sigmoid(rand(5, h)),
        w=torch.softmax(rand(6, n, k), 1), mats=0.1 * rand(7, e, h, h)).items()}
    ids = torch.rand(n, e, generator=torch.Generator().manual_seed(8)).topk(k, 1).indices.to(dev)
    plan = token_sort_plan(ids, e, row_align=4)
    cu, counts = plan.cu_seqlens.tolist(), plan.counts.tolist()

    def experts(rows, mats):
        return torch.cat([rows[cu[i]:cu[i + 1]] @ mats[i] for i in range(e)] + [rows[cu[e]:]])
    L = leaves
    y, nrm = gated_residual_rmsnorm(L["x"], L["res"], post_weight=L["post"], gate=L["gate"], residual_scale=0.5,
                                    pre_weight=L["pre"])
    rows = sort_tokens(nrm, plan)
    done = experts(rows, L["mats"])
    moe = unsort_tokens(done, plan, L["w"])
    y2, n2 = gated_residual_rmsnorm(moe, y, post_weight=L["post"], pre_weight=L["pre"])
    cy, cn = rand(9, n, h).to(dev), rand(10, n, h).to(dev)
    whole = torch.autograd.grad((y2, n2), list(L.values()), (cy, cn), retain_graph=True)
    # piece by piece
    moe_c, y_c, post2, pre2 = [v.detach().requires_grad_(True) for v in (moe, y, L["post"], L["pre"])]
    y2b, n2b = gated_residual_rmsnorm(moe_c, y_c, post_weight=post2, pre_weight=pre2)
    d_moe, d_y, d_post2, d_pre2 = torch.autograd.grad((y2b, n2b), (moe_c, y_c, post2, pre2), (cy, cn))
    done_c, w_c = done.detach().requires_grad_(True), L["w"].detach().requires_grad_(True)
    d_done, d_w = torch.autograd.grad(unsort_tokens(done_c, plan, w_c), (done_c, w_c), d_moe)
    live = torch.zeros(plan.capacity, dtype=torch.bool, device=rows.device)
    for i in range(e):
        live[cu[i]:cu[i] + counts[i]] = True
    assert not bool(d_done[~live].any()) and not bool(rows.detach()[~live].any())      # padding rows carry nothing
    rows_c, mats_c = rows.detach().requires_grad_(True), L["mats"].detach().requires_grad_(True)
    d_rows, d_mats = torch.autograd.grad(experts(rows_c, mats_c), (rows_c, mats_c), d_done)
    n_c = nrm.detach().requires_grad_(True)
    (d_n,) = torch.autograd.grad(sort_tokens(n_c, plan), n_c, d_rows)
    first = [L[name].detach().requires_grad_(True) for name in ("x", "res", "post", "pre", "gate")]
    ya, na = gated_residual_rmsnorm(first[0], first[1], post_weight=first[2], gate=first[4], residual_scale=0.5,
                                    pre_weight=first[3])
    d_x, d_res, d_post, d_pre, d_gate = torch.autograd.grad((ya, na), first, (d_y, d_n))
    for got, want in zip(whole, (d_x, d_res, d_post + d_post2, d_pre + d_pre2, d_gate, d_w, d_mats)):
        assert torch.equal(got, want) or torch.allclose(got, want, rtol=2 * ref.U32, atol=0)       # one sum of two terms


@pytest.mark.skipif(emulating(), reason="tens of GB")
def test_offsets_past_32_bits(dev):
    """Operands of more than 2^32 bytes (and 2^31 elements): the last rows come out as they do on their own."""
    from batchgen_amd.attention.gated_residual_norm import gated_residual_rmsnorm, gated_residual_rmsnorm_int8_quant
    from batchgen_amd.moe.token_sort import sort_tokens, token_sort_plan, unsort_tokens
    from batchgen_amd.quantization.int8 import int8_linear, int8_quant_rows
    n, k, h, e = 40000, 8, 8192, 64
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(n, h, device=dev, generator=g, dtype=torch.bfloat16).requires_grad_(True)
    ids = torch.rand(n, e, device=dev, generator=g).topk(k, 1).indices
    plan = token_sort_plan(ids, e)
    rows = sort_tokens(x, plan)
    assert rows.numel() * 2 > 1 << 32
    back = unsort_tokens(rows, plan)
    assert torch.equal(back, 8 * x.detach())              # eight equal terms: exact
    (dx,) = torch.autograd.grad(back, x, torch.ones_like(back))
    assert bool((dx == 8).all())
    last = plan.topk_pos[-1].long()
    assert torch.equal(rows.detach()[last], x.detach()[-1:].expand(k, h))
    del rows, back, dx, x
    torch.cuda.empty_cache()
    m, kk, nn = 620000, 7168, 48
    q = torch.randint(-127, 128, (m, kk), device=dev, generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (nn, kk), device=dev, generator=g, dtype=torch.int8)
    s, ws = torch.rand(m, device=dev, generator=g), torch.rand(nn, device=dev, generator=g)
    out = int8_linear(q, w, ws, x_scale=s)
    assert torch.equal(out[-300:], int8_linear(q[-300:].clone(), w, ws, x_scale=s[-300:].clone()))
    del q, out
    torch.cuda.empty_cache()
    r, hh = 300000, 8192
    b, res = (torch.randn(r, hh, device=dev, generator=g, dtype=torch.bfloat16).requires_grad_(True) for _ in range(2))
    pre = torch.rand(hh, device=dev, generator=g).to(torch.bfloat16)
    y, nrm = gated_residual_rmsnorm(b, res, post_weight=pre, pre_weight=pre)
    db, dr = torch.autograd.grad((y, nrm), (b, res), (y.detach(), nrm.detach()))
    tail = [t.detach()[-5:].clone().requires_grad_(True) for t in (b, res)]
    ty, tn = gated_residual_rmsnorm(*tail, post_weight=pre, pre_weight=pre)
    tdb, tdr = torch.autograd.grad((ty, tn), tail, (ty.detach(), tn.detach()))
    # another number of vectors per thread: another order of the row sums, at most a step of the output type away
    for got, want in ((y[-5:], ty), (nrm[-5:], tn), (db[-5:], tdb), (dr[-5:], tdr)):
        want = want.detach().to("cpu", ref.F64)
        ref.assert_within(got, want, 2 * ref.half_step(torch.bfloat16, want) * (1 + 2 ** -7) + 2 ** -16 * want.abs().max(), "tail")
    del y, nrm, db, dr
    q, qs = int8_quant_rows(b.detach())
    tq, tqs = int8_quant_rows(b.detach()[-5:].clone())
    assert torch.equal(q[-5:], tq) and torch.equal(qs[-5:], tqs)
    del q
    with torch.no_grad():
        q8 = gated_residual_rmsnorm_int8_quant(b, res, post_weight=pre, pre_weight=pre)
        tq = int8_quant_rows(q8[1][-5:].clone())
        assert torch.equal(q8[2][-5:], tq[0]) and torch.equal(q8[3][-5:], tq[1])
