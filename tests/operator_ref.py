"""Plain 64-bit forms of the token sort, the int8 products and the gated residual norm, and the rounding bounds their
tests use.  A rounding to type t is off by at most half a step, finfo(t).eps / 2 relative to the value, or half the
smallest subnormal."""
import torch

U32 = 2.0 ** -24                       # half a step of fp32
F64 = torch.float64
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def half_step(t, value):
    """Largest error of one rounding of ``value`` to type ``t``."""
    f = torch.finfo(t)
    return value.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def assert_within(got, want, tol, what):
    err = (got.detach().to("cpu", F64) - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst error {float(err[bad].max()):.3g} "
                                 f"where {float(tol.expand_as(err)[bad].min()):.3g} is allowed")


# ---- token sort ------------------------------------------------------------------------------------------------------
def sort_plan(ids, e, start=0, align=1):
    """-> counts, cu (lists), pos [N, K] int64 with -1 for pairs without a row."""
    n, k = ids.shape
    buckets = [[] for _ in range(e)]
    for i, v in enumerate(ids.cpu().reshape(-1).tolist()):
        if 0 <= v - start < e:
            buckets[v - start].append(i)
    pos = torch.full((n * k,), -1, dtype=torch.int64)
    cu = [0]
    for b in buckets:
        for j, i in enumerate(b):
            pos[i] = cu[-1] + j
        cu.append(cu[-1] + (len(b) + align - 1) // align * align)
    return [len(b) for b in buckets], cu, pos.reshape(n, k)


def unsort(rows, pos, w):
    """fp64 sum and the sum of magnitudes (for the rounding bound)."""
    n, k = pos.shape
    out = torch.zeros(n, rows.size(1), dtype=F64)
    mag = torch.zeros_like(out)
    for t in range(n):
        for j in range(k):
            if pos[t, j] >= 0:
                term = (1.0 if w is None else w[t, j].to(F64)) * rows[pos[t, j]].to(F64)
                out[t] += term
                mag[t] += term.abs()
    return out, mag


# ---- gated residual norm ---------------------------------------------------------------------------------------------
# A row's sum of squares is a chain of at most 16 fused multiply-adds, six shuffle steps and 16 waves' sums: fewer than
# 64 roundings, all of positive terms.  Its square root's inverse is therefore off by at most 32 + 3 half steps.
NORM_C = 40


def norm_forward(block, residual, post, gate, scale, pre, eps):
    """fp64 (y, n) and bounds of the fp32 evaluation, without the outputs' own rounding."""
    b, r = block.to(F64), residual.to(F64)
    p = b if post is None else b / torch.sqrt((b * b).mean(-1, keepdim=True) + eps) * post.to(F64)
    add = scale * p * (1.0 if gate is None else gate.to(F64))
    y = r + add
    e_y = U32 * (NORM_C * add.abs() + y.abs())
    if pre is None:
        return y, None, e_y, None
    i2 = 1.0 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    n = y * i2 * pre.to(F64)
    rel = (e_y * e_y).mean(-1, keepdim=True).sqrt() * i2
    e_n = (i2 * pre.to(F64)).abs() * e_y + n.abs() * (NORM_C * U32 + rel)
    return y, n, e_y, e_n


def norm_grads(block, residual, post, gate, scale, pre, eps, dy, dn):
    """fp64 gradients from autograd, and for each the sum of the magnitudes of its terms (the cancelling sums of the
    formula with every term taken positive), by which rounding errors are bounded."""
    names = ("block", "residual", "post", "gate", "pre")
    v = {m: None if t is None else t.detach().to("cpu", F64).requires_grad_(True)
         for m, t in zip(names, (block, residual, post, gate, pre))}
    y, n, _, _ = norm_forward(v["block"], v["residual"], v["post"], v["gate"], scale, v["pre"], eps)
    total = 0.0
    if dy is not None:
        total = total + (y * dy.to(F64)).sum()
    if dn is not None:
        total = total + (n * dn.to(F64)).sum()
    leaves = [m for m in names if v[m] is not None]
    g = dict(zip(leaves, torch.autograd.grad(total, [v[m] for m in leaves], allow_unused=True)))
    with torch.no_grad():
        b, y = v["block"].abs(), y.abs()
        i1 = 1.0 if post is None else 1.0 / torch.sqrt((b * b).mean(-1, keepdim=True) + eps)
        bh, w1 = b * i1, 1.0 if post is None else v["post"].abs()
        sg = abs(scale) * (1.0 if gate is None else v["gate"].abs())
        my = torch.zeros_like(b) if dy is None else dy.to(F64).abs()
        mag = {}
        if dn is not None:
            i2 = 1.0 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
            t, yh = dn.to(F64).abs() * v["pre"].abs(), y * i2
            my = my + i2 * (t + yh * (t * yh).mean(-1, keepdim=True))
            mag["pre"] = (dn.to(F64).abs() * yh).reshape(-1, b.size(-1)).sum(0)
        elif pre is not None:
            mag["pre"] = torch.zeros(b.size(-1), dtype=F64)
        mag["residual"] = my
        dp = sg * my
        mag["block"] = i1 * (dp * w1 + (bh * (dp * w1 * bh).mean(-1, keepdim=True) if post is not None else 0.0))
        if post is not None:
            mag["post"] = (dp * bh).reshape(-1, b.size(-1)).sum(0)
        if gate is not None:
            m = abs(scale) * bh * w1 * my
            if gate.shape == (b.size(-1),):
                m = m.reshape(-1, b.size(-1)).sum(0)
            elif gate.size(-1) == 1 and b.size(-1) != 1:
                m = m.sum(-1, keepdim=True)
            mag["gate"] = m
    return {m: torch.zeros_like(v[m]) if g[m] is None else g[m] for m in leaves}, mag


# the largest number of roundings on a path from an input to a gradient: three sums over a row (64 each) that enter one
# another, the two inverse roots (35 each), about 20 products, and for the weights a sum over rows (one per row of a
# block and one per block)
def grad_roundings(rows):
    return 3 * 64 + 2 * 35 + 20 + min(rows, 1024) + 64
