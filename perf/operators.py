"""Measured cases of three operators around a mixture-of-experts block, each in its plain form (elementary torch
operations, 32 bits) and as this package's calls:

* ``linear`` / ``experts``: matrix products in 8-bit integers with one scale per token and one per output channel
  (``int8_linear``, ``int8_grouped_gemm``, ``int8_fused_s1``);
* ``sort``: tokens sorted by expert and brought back with their routing weights, forward and gradient
  (``token_sort_plan``, ``sort_tokens``, ``unsort_tokens``);
* ``norm``: the RMSNorm behind a block, its gate and residual scale, the residual sum and the RMSNorm in front of the
  next block in one pass, forward, gradient and the form that also hands the next product its int8 rows
  (``gated_residual_rmsnorm``, ``gated_residual_rmsnorm_int8_quant``).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decode step through a 7168 -> 4096 projection: latency and the weights' stream
        dict(name="linear_one_token", kind="linear", m=1, k=7168, n=4096, dtype="bf16", bias=False),
        # a small batch through a layer whose sizes divide nothing: ragged tiles, bias, half precision
        dict(name="linear_odd", kind="linear", m=77, k=1424, n=1001, dtype="fp16", bias=True),
        # a prefill chunk through the same projection as the single token
        dict(name="linear_prefill", kind="linear", m=8192, k=7168, n=4096, dtype="bf16", bias=False),
        # decode, 256 tokens routed to 8 of 256 experts, 32 of them here: gate and up of about 8 rows each
        dict(name="experts_decode", kind="experts", rows=256, e=32, k=7168, n=2048, fused=True, skew=0.0),
        # a prefill chunk's share of the same layer: gate and up, 512 rows per expert on average, mildly skewed
        dict(name="experts_prefill", kind="experts", rows=16384, e=32, k=7168, n=2048, fused=True, skew=0.3),
        # the down projection under skewed routing: hot experts, and experts without a row
        dict(name="experts_down_skewed", kind="experts", rows=4095, e=64, k=2048, n=7168, fused=False, skew=1.2),
        # a decode batch of an expert-parallel rank: 32 of 256 experts are local, rows go into a kept buffer
        dict(name="sort_decode", kind="sort", n=256, k=8, h=7168, e_total=256, e=32, start=64, dtype="bf16", train=False),
        # a training step's odd remainder batch in 32 bits
        dict(name="sort_train_odd", kind="sort", n=1003, k=6, h=1001, e_total=64, e=64, start=0, dtype="fp32", train=True),
        # a training step over 16384 tokens, all experts local
        dict(name="sort_train", kind="sort", n=16384, k=8, h=7168, e_total=256, e=256, start=0, dtype="bf16", train=True),
        # a small decode batch between two blocks, int8 rows for the next projection
        dict(name="norm_decode_int8", kind="norm", rows=16, h=7168, dtype="bf16", gate="channel", train=False, int8=True),
        # odd width and row count in half precision, one gate value per token, with gradients
        dict(name="norm_train_odd", kind="norm", rows=333, h=1001, dtype="fp16", gate="token", train=True, int8=False),
        # a training step over 16384 tokens, one learned gate value per channel
        dict(name="norm_train", kind="norm", rows=16384, h=7168, dtype="bf16", gate="channel", train=True, int8=False),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "experts", "experts", "sort", "sort", "sort", "norm", "norm", "norm"])
    if kind == "linear":
        m, k, n = _log(rng, 1, 8192), 16 * _log(rng, 4, 448), _log(rng, 33, 7168)
        m = min(m, max(1, 8192 * 7168 * 4096 // (k * n)))
        return dict(kind=kind, m=m, k=k, n=n, dtype=rng.choice(["bf16", "fp16"]), bias=rng.random() < 0.4)
    if kind == "experts":
        e, k, fused = _log(rng, 1, 64), 16 * _log(rng, 8, 448), rng.random() < 0.5
        n = _log(rng, 48, 2048 if fused else 7168)
        rows = _log(rng, 1, 16384)
        if e * k * n * (2 if fused else 1) > 32 * 7168 * 4096:
            e = max(1, 32 * 7168 * 4096 // (k * n * (2 if fused else 1)))
        return dict(kind=kind, rows=rows, e=e, k=k, n=n, fused=fused, skew=round(rng.choice([0.0, 0.3, 0.8, 1.2]), 1))
    if kind == "sort":
        n, k, h, train = _log(rng, 1, 16384), rng.randint(1, 16), _log(rng, 17, 7168), rng.random() < 0.6
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        n = min(n, max(1, 16384 * 8 * 7168 * 2 // (k * h * SIZE[dtype])))
        e_total = max(k, _log(rng, 4, 512))
        e = e_total if train else max(1, e_total // rng.choice([1, 2, 8]))
        start = 0 if e == e_total else rng.randint(0, e_total - e)
        return dict(kind=kind, n=n, k=k, h=h, e_total=e_total, e=e, start=start, dtype=dtype, train=train)
    rows, h, train = _log(rng, 1, 16384), _log(rng, 65, 8192), rng.random() < 0.6
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    int8 = not train and rng.random() < 0.6
    if int8:
        h, dtype = max(80, h // 16 * 16), rng.choice(["bf16", "fp16"])      # rows that an int8 product takes
    rows = min(rows, max(1, 16384 * 7168 * 2 // (h * SIZE[dtype])))
    return dict(kind=kind, rows=rows, h=h, dtype=dtype, gate=rng.choice(["none", "channel", "token", "full"]), train=train,
                int8=int8)


# ----------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _int8(g, *shape):
    """What quantising normal values leaves: a rounded normal distribution, at most 127."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda").mul_(34.0).round_().clamp_(-127, 127))
    return out


def prepare(case, seed):
    g, c = _gen(seed), dict(case)
    kind = c["kind"]
    if kind == "linear":
        # activations of tokens of different size, a few channels much larger than the rest
        x = _randn(g, c["m"], c["k"]) * torch.exp(0.5 * _randn(g, c["m"], 1))
        x = x * (1.0 + 7.0 * (torch.rand(1, c["k"], generator=g, device="cuda") < 0.005))
        s = dict(x=x.to(DTYPES[c["dtype"]]), w=_int8(g, c["n"], c["k"]),
                 ws=(0.5 + torch.rand(c["n"], generator=g, device="cuda")) * (0.02 / 34.0),
                 bias=0.1 * _randn(g, c["n"]) if c["bias"] else None)
    elif kind == "experts":
        e, r = c["e"], c["rows"]
        popularity = torch.arange(1, e + 1, device="cuda", dtype=torch.float32).pow(-c["skew"])
        popularity = popularity[torch.randperm(e, generator=g, device="cuda")]
        ids = torch.multinomial(popularity, r, replacement=True, generator=g)
        counts = torch.bincount(ids, minlength=e)
        cu = torch.zeros(e + 1, dtype=torch.int64, device="cuda")
        cu[1:] = torch.cumsum(counts, 0)
        s = dict(x=_int8(g, r, c["k"]), xs=(0.5 + torch.rand(r, generator=g, device="cuda")) / 34.0,
                 w=_int8(g, e, c["n"], c["k"]),
                 ws=(0.5 + torch.rand(e, c["n"], generator=g, device="cuda")) * (0.02 / 34.0),
                 seqlens=counts.to(torch.int32), cu=cu.to(torch.int32), most=int(counts.max()))
        if c["fused"]:
            s["w1"] = _int8(g, e, c["n"], c["k"])
            s["ws1"] = (0.5 + torch.rand(e, c["n"], generator=g, device="cuda")) * (0.02 / 34.0)
    elif kind == "sort":
        n, k, dt = c["n"], c["k"], DTYPES[c["dtype"]]
        # top-k of random scores with a per-expert preference: distinct experts per token, uneven load
        score = _randn(g, n, c["e_total"]) + 0.5 * _randn(g, 1, c["e_total"])
        ids = torch.topk(score, k, dim=1).indices
        if not c["train"]:
            ids = ids.to(torch.int32)
            ids[torch.rand(n, generator=g, device="cuda") < 0.03] = -1          # padding tokens of a decode bucket
        w = torch.softmax(_randn(g, n, k), dim=1)
        s = dict(ids=ids, w=w, x=_randn(g, n, c["h"]).to(dt), y=_randn(g, n * k, c["h"]).to(dt))
        if c["train"]:
            s["dout"] = _randn(g, n, c["h"]).to(dt)
            s["drows"] = _randn(g, n * k, c["h"]).to(dt)
            for name in ("x", "y", "w"):
                s[name].requires_grad_(True)
        else:
            s["rows"] = torch.zeros(n * k, c["h"], dtype=dt, device="cuda")
    else:
        rows, h, dt = c["rows"], c["h"], DTYPES[c["dtype"]]
        s = dict(block=(_randn(g, rows, h) * torch.exp(0.5 * _randn(g, rows, 1))).to(dt),
                 residual=(2.0 * _randn(g, rows, h)).to(dt),
                 post=(1.0 + 0.2 * _randn(g, h)).to(dt), pre=(1.0 + 0.2 * _randn(g, h)).to(dt),
                 scale=0.7, gate=None)
        if c["gate"] != "none":
            shape = {"channel": (h,), "token": (rows, 1), "full": (rows, h)}[c["gate"]]
            s["gate"] = torch.sigmoid(_randn(g, *shape)).to(dt)
        if c["train"]:
            s["dy"], s["dn"] = _randn(g, rows, h).to(dt), _randn(g, rows, h).to(dt)
            for name in ("block", "residual", "post", "pre", "gate"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    s["case"] = c
    return s


# -------------------------------------------------------------------------------------------------------------- run
def run(state):
    kind = state["case"]["kind"]
    if kind == "linear":
        return _linear(state)
    if kind == "experts":
        return _experts(state)
    if kind == "sort":
        return _sort(state)
    return _norm(state)


def _linear(s):
    if own:
        from batchgen_amd.quantization.int8 import int8_linear
        return int8_linear(s["x"], s["w"], s["ws"], bias=s["bias"])
    x = s["x"].float()
    scale = x.abs().amax(1).clamp_min(1e-30) / 127.0
    q = torch.round(x / scale[:, None]).clamp(-127, 127)
    y = (q @ s["w"].float().t()) * scale[:, None] * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _experts(s):
    c = s["case"]
    if own:
        from batchgen_amd.moe.grouped_int8_moe import int8_fused_s1, int8_grouped_gemm
        if c["fused"]:
            return int8_fused_s1(s["x"], s["xs"], s["w"], s["ws"], s["w1"], s["ws1"], s["seqlens"], s["cu"])
        return int8_grouped_gemm(s["x"], s["xs"], s["w"], s["ws"], s["seqlens"], s["cu"])
    # rows of every expert side by side, padded to the longest; then one batched product
    r = torch.arange(c["rows"], device="cuda")
    e = torch.searchsorted(s["cu"][1:].long().contiguous(), r, right=True)
    slot = r - s["cu"].long()[e]
    pad = torch.zeros(c["e"], s["most"], c["k"], device="cuda")
    pad[e, slot] = s["x"].float()

    def product(w, ws):
        y = torch.bmm(pad, w.float().transpose(1, 2).contiguous())[e, slot]
        return y * s["xs"][:, None] * ws[e]
    y = product(s["w"], s["ws"])
    if c["fused"]:
        y = y / (1.0 + torch.exp(-y)) * product(s["w1"], s["ws1"])
    return y.to(torch.bfloat16)


def _sort(s):
    c = s["case"]
    if own:
        from batchgen_amd.moe.token_sort import sort_tokens, token_sort_plan, unsort_tokens
        plan = token_sort_plan(s["ids"], c["e"], expert_start=c["start"])
        if not c["train"]:
            rows = sort_tokens(s["x"], plan, out=s["rows"])
            return dict(rows=rows, out=unsort_tokens(s["y"], plan, s["w"]), counts=plan.counts, pos=plan.topk_pos)
        rows = sort_tokens(s["x"], plan)
        out = unsort_tokens(s["y"], plan, s["w"])
        dx, dy, dw = torch.autograd.grad((rows, out), (s["x"], s["y"], s["w"]), (s["drows"], s["dout"]))
        return dict(rows=rows, out=out, counts=plan.counts, pos=plan.topk_pos, dx=dx, dy=dy, dw=dw)
    n, k, e, dt = c["n"], c["k"], c["e"], s["x"].dtype
    with torch.no_grad():
        local = s["ids"].reshape(-1).long() - c["start"]
        key = torch.where((local >= 0) & (local < e), local, e)
        sorted_key, order = torch.sort(key, stable=True)
        ends = torch.searchsorted(sorted_key, torch.arange(e, device="cuda"), right=True)
        counts = torch.diff(ends, prepend=torch.zeros(1, dtype=ends.dtype, device="cuda")).to(torch.int32)
        pos = torch.empty_like(order)
        pos[order] = torch.arange(n * k, device="cuda")
        here = (key < e)
        rows = torch.where((sorted_key < e)[:, None], s["x"][order // k], torch.zeros((), dtype=dt, device="cuda"))
        yk = s["y"][pos].float().reshape(n, k, -1)
        wk = torch.where(here.reshape(n, k), s["w"], 0.0)
        out = (yk * wk[:, :, None]).sum(1).to(dt)
        told = torch.where(here, pos, -1).to(torch.int32).reshape(n, k)
        if not c["train"]:
            return dict(rows=rows, out=out, counts=counts, pos=told)
        g = s["dout"].float()
        dx = s["drows"][pos].float().reshape(n, k, -1).sum(1).to(dt)
        dw = (yk * g[:, None, :]).sum(2)
        dy = torch.empty_like(s["y"])
        dy[pos] = (wk[:, :, None] * g[:, None, :]).reshape(n * k, -1).to(dt)
        return dict(rows=rows, out=out, counts=counts, pos=told, dx=dx, dy=dy, dw=dw)


def _norm(s):
    c = s["case"]
    if own:
        from batchgen_amd.attention.gated_residual_norm import (gated_residual_rmsnorm,
                                                                gated_residual_rmsnorm_int8_quant)
        args = dict(post_weight=s["post"], gate=s["gate"], residual_scale=s["scale"], pre_weight=s["pre"], eps=EPS)
        if c["int8"]:
            y, n, q, qs = gated_residual_rmsnorm_int8_quant(s["block"], s["residual"], **args)
            return dict(y=y, n=n, q=(q * qs[:, None]).to(n.dtype))
        y, n = gated_residual_rmsnorm(s["block"], s["residual"], **args)
        if not c["train"]:
            return dict(y=y, n=n)
        leaves = [s[name] for name in ("block", "residual", "post", "pre", "gate") if s[name] is not None]
        return dict(y=y, n=n, grads=torch.autograd.grad((y, n), leaves, (s["dy"], s["dn"])))
    with torch.no_grad():
        dt, scale = s["block"].dtype, s["scale"]
        b, w1, w2 = s["block"].float(), s["post"].float(), s["pre"].float()
        gate = 1.0 if s["gate"] is None else s["gate"].float()
        i1 = torch.rsqrt((b * b).mean(1, keepdim=True) + EPS)
        p = b * i1 * w1
        y = s["residual"].float() + scale * gate * p
        i2 = torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
        n = y * i2 * w2
        if c["int8"]:
            nb = n.to(dt).float()
            qs = nb.abs().amax(1, keepdim=True).clamp_min(1e-30) / 127.0
            q = torch.round(nb / qs).clamp(-127, 127)
            return dict(y=y.to(dt), n=n.to(dt), q=(q * qs).to(dt))
        if not c["train"]:
            return dict(y=y.to(dt), n=n.to(dt))
        dn = s["dn"].float()
        yhat, t = y * i2, dn * w2
        dy = s["dy"].float() + i2 * (t - yhat * (t * yhat).mean(1, keepdim=True))
        dw2 = (dn * yhat).sum(0)
        dp = scale * gate * dy
        bhat, u = b * i1, dp * w1
        db = i1 * (u - bhat * (u * bhat).mean(1, keepdim=True))
        dw1 = (dp * bhat).sum(0)
        grads = [db.to(dt), dy.to(dt), dw1.to(dt), dw2.to(dt)]
        if s["gate"] is not None:
            dg = scale * p * dy
            dg = dg.sum(0) if c["gate"] == "channel" else dg.sum(1, keepdim=True) if c["gate"] == "token" else dg
            grads.append(dg.to(dt))
        return dict(y=y.to(dt), n=n.to(dt), grads=tuple(grads))


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "linear":
        b = c["m"] * (c["k"] + c["n"]) * SIZE[c["dtype"]] + c["n"] * c["k"] + c["n"] * (8 if c["bias"] else 4)
        return {"bytes": b, "flops": 2.0 * c["m"] * c["n"] * c["k"]}
    if c["kind"] == "experts":
        e = min(c["e"], c["rows"])                       # experts that can have a row
        mats = 2 if c["fused"] else 1
        b = c["rows"] * (c["k"] + 4 + 2 * c["n"]) + mats * e * c["n"] * (c["k"] + 4)
        return {"bytes": b, "flops": 2.0 * mats * c["rows"] * c["n"] * c["k"]}
    if c["kind"] == "sort":
        share = c["e"] / c["e_total"]                    # of the pairs: what lies here
        token, pair = c["n"] * c["h"] * SIZE[c["dtype"]], c["n"] * c["k"] * c["h"] * SIZE[c["dtype"]] * share
        index = c["n"] * c["k"] * (12 if c["train"] else 8)
        if not c["train"]:
            return {"bytes": 2 * token + 2 * pair + index + 4 * c["n"] * c["k"], "flops": 2 * pair}
        return {"bytes": 4 * token + 4 * pair + index + 8 * c["n"] * c["k"], "flops": 6 * pair}
    row = c["rows"] * c["h"] * SIZE[c["dtype"]]
    gate = row if c["gate"] == "full" else 0
    if c["train"]:                                       # block, residual, dy, dn in; y, n and two gradients out
        return {"bytes": 8 * row + 2 * gate, "flops": 30.0 * c["rows"] * c["h"]}
    return {"bytes": 4 * row + gate + (c["rows"] * (c["h"] + 4) if c["int8"] else 0), "flops": 12.0 * c["rows"] * c["h"]}


# ------------------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """The definitions in 64 bits, from the same inputs."""
    s = prepare(case, seed)
    c, d = s["case"], torch.float64
    with torch.no_grad():
        if c["kind"] == "linear":
            x = s["x"].to(d)
            step = torch.clamp(torch.max(torch.abs(x), dim=1, keepdim=True).values, min=1e-30) / 127
            levels = torch.round(x / step)
            y = torch.matmul(levels, s["w"].to(d).T) * step * s["ws"].to(d)[None, :]
            return y if s["bias"] is None else y + s["bias"].to(d)
        if c["kind"] == "experts":
            y = torch.empty(c["rows"], c["n"], dtype=d, device="cuda")
            cu = s["cu"].tolist()
            for e in range(c["e"]):
                lo, hi = cu[e], cu[e + 1]
                if hi == lo:
                    continue
                x = s["x"][lo:hi].to(d) * s["xs"][lo:hi].to(d)[:, None]
                part = torch.mm(x, (s["w"][e].to(d) * s["ws"][e].to(d)[:, None]).T)
                if c["fused"]:
                    part = part * torch.sigmoid(part) * torch.mm(x, (s["w1"][e].to(d) * s["ws1"][e].to(d)[:, None]).T)
                y[lo:hi] = part
            return y
        if c["kind"] == "sort":
            n, k, h = c["n"], c["k"], c["h"]
            ids = s["ids"].cpu().reshape(-1).tolist()
            buckets = [[] for _ in range(c["e"])]
            for i, expert in enumerate(ids):
                if 0 <= expert - c["start"] < c["e"]:
                    buckets[expert - c["start"]].append(i)
            pairs = torch.tensor([i for b in buckets for i in b], dtype=torch.int64, device="cuda")
            live, token = pairs.numel(), pairs // k
            pos = torch.full((n * k,), -1, dtype=torch.int64, device="cuda")
            pos[pairs] = torch.arange(live, device="cuda")
            counts = torch.tensor([len(b) for b in buckets], device="cuda")
            rows = torch.zeros(n * k, h, dtype=d, device="cuda")
            rows[:live] = s["x"].to(d)[token]
            wl = s["w"].to(d).reshape(-1)[pairs]
            yl = s["y"][:live].to(d)
            out = torch.zeros(n, h, dtype=d, device="cuda").index_add_(0, token, yl * wl[:, None])
            told = dict(rows=rows, out=out, counts=counts, pos=pos.reshape(n, k))
            if c["train"]:
                gl = s["dout"].to(d)[token]
                told["dx"] = torch.zeros(n, h, dtype=d, device="cuda").index_add_(0, token, s["drows"][:live].to(d))
                dw = torch.zeros(n * k, dtype=d, device="cuda")
                dw[pairs] = (gl * yl).sum(1)
                told["dw"] = dw.reshape(n, k)
                told["dy"] = gl * wl[:, None]
            return told
        names = ("block", "residual", "post", "pre", "gate")
        with torch.enable_grad():
            v = {m: None if s[m] is None else s[m].detach().to(d).requires_grad_(c["train"]) for m in names}
            normed = v["block"] / torch.sqrt(v["block"].pow(2).mean(-1, keepdim=True) + EPS) * v["post"]
            y = v["residual"] + s["scale"] * (normed if v["gate"] is None else v["gate"] * normed)
            n = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * v["pre"]
            if c["train"]:
                grads = torch.autograd.grad((y, n), [v[m] for m in names if v[m] is not None],
                                            (s["dy"].to(d), s["dn"].to(d)))
                return dict(y=y.detach(), n=n.detach(), grads=grads)
        if c["int8"]:
            held = n.to(s["block"].dtype).to(d)          # the quantiser reads the stored row
            step = torch.clamp(held.abs().amax(1, keepdim=True), min=1e-30) / 127
            return dict(y=y, n=n, q=torch.round(held / step) * step)
        return dict(y=y, n=n)
