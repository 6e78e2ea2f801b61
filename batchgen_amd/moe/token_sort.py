"""Tokens sorted by expert and brought back with their routing weights, differentiable.

The ragged dispatch and the weighted combine of ``dispatch_scatter_3d`` serve the reference's inference path (bf16,
fixed top-k, no gradient).  These are the same movement for training and for every element type:

    plan = token_sort_plan(topk_ids, num_experts)          # where each (token, slot) pair goes; stays on the device
    rows = sort_tokens(x, plan)                             # rows[plan.topk_pos[t, j]] = x[t]
    ...                                                     # the experts, over rows [cu_seqlens[e], cu_seqlens[e] + counts[e])
    out = unsort_tokens(rows, plan, topk_weights)           # out[t] = sum_j w[t, j] * rows[topk_pos[t, j]]

Gradients reach ``x``, ``rows`` and ``topk_weights``; no kernel uses atomics, so they are the same bits every time.
They have no gradient of their own and there is no forward-mode derivative: asking for either raises.
Ids outside ``[expert_start, expert_start + num_experts)`` (another rank's experts, ``-1`` on padding tokens) have no
row: they add nothing to ``out`` and their weight gets gradient 0, whatever it holds.
"""
from __future__ import annotations

from typing import Optional

import torch

from .._lib import lib, ptr
from ..kernels import _checks as ck
from ..kernels._autograd import no_second_gradient
from .dispatch_scatter_3d import ragged_row_capacity

MAX_TOP_K = 32


class TokenSortPlan:
    """``counts`` int32 ``[E]``, ``cu_seqlens`` int32 ``[E + 1]``, ``topk_pos`` int32 ``[N, K]`` (-1: no row), and the
    host-side sizes; ``capacity`` is the row count of a sorted buffer (enough for any routing)."""
    __slots__ = ("meta", "topk_pos", "num_tokens", "top_k", "num_experts", "row_align", "capacity")

    def __init__(self, meta, topk_pos, num_experts, row_align, capacity):
        self.meta, self.topk_pos = meta, topk_pos          # meta: counts, then cu_seqlens
        self.num_tokens, self.top_k = topk_pos.shape
        self.num_experts, self.row_align, self.capacity = num_experts, row_align, capacity

    @property
    def counts(self) -> torch.Tensor:
        return self.meta[:self.num_experts]

    @property
    def cu_seqlens(self) -> torch.Tensor:
        return self.meta[self.num_experts:]


def token_sort_plan(topk_ids: torch.Tensor, num_experts: int, expert_start: int = 0, row_align: int = 1) -> TokenSortPlan:
    """``topk_ids`` int32 or int64 ``[N, K]``, K <= 32.  ``num_experts`` (at most 1024) experts from ``expert_start`` on
    are local.  Every expert's rows start at a multiple of ``row_align`` (a power of two)."""
    ck.gpu(topk_ids, "topk_ids")
    ck.dtype(topk_ids, (torch.int32, torch.int64), "topk_ids")
    if topk_ids.dim() != 2 or not 1 <= topk_ids.size(1) <= MAX_TOP_K:
        ck.fail(f"topk_ids must be [N, K] with K in [1, {MAX_TOP_K}], got {tuple(topk_ids.shape)}")
    n, k = topk_ids.shape
    e, row_align = ck.int32(int(num_experts), "num_experts"), ck.int32(int(row_align), "row_align")
    ck.int32(n * k, "N*K")
    ck.int32(int(expert_start), "expert_start")
    if row_align <= 0 or row_align & (row_align - 1):
        ck.fail(f"row_align must be a positive power of two, got {row_align}")
    ids = topk_ids.contiguous()
    dev = ids.device
    meta = torch.empty(2 * max(e, 0) + 1, dtype=torch.int32, device=dev)
    pos = torch.empty((n, k), dtype=torch.int32, device=dev)
    need = int(lib().bgmoe_dispatch_workspace_bytes(n * k, e))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    ck.launch(dev, lib().bgmoe_token_sort_index, ptr(ids), int(ids.dtype == torch.int64), n, k, int(expert_start), e,
              row_align, ptr(meta), ptr(meta) + 4 * e, ptr(pos), ptr(ws), need)
    return TokenSortPlan(meta, pos, e, row_align, ragged_row_capacity(n, k, e, row_align))


def _tokens(x, plan, name, rows):
    """``x`` as ``[rows, H]`` with contiguous rows on the plan's device."""
    ck.gpu(x, name)
    ck.same_device(plan.topk_pos, x, name)
    if x.dim() != 2 or x.size(0) != rows:
        ck.fail(f"{name} must be [{rows}, H], got {tuple(x.shape)}")
    ck.int32(x.size(1), "H")
    return ck.rows_of(x, name)


def _buffer(out, like, shape, name):
    ck.cuda_tensor(like, out, like.dtype, name)
    if tuple(out.shape) != tuple(shape):
        ck.fail(f"{name} must have the shape {tuple(shape)}, got {tuple(out.shape)}")


def _run_sort(x, plan, out):
    zero_rest = out is None
    h = x.size(1)
    if out is None:
        out = torch.empty((plan.capacity, h), dtype=x.dtype, device=x.device)
    size, meta = x.element_size(), ptr(plan.meta)
    ck.launch(x.device, lib().bgmoe_token_sort_rows, ptr(x), x.stride(0) * size, h * size, plan.num_tokens,
              plan.top_k, ptr(plan.topk_pos), meta, meta + 4 * plan.num_experts, plan.num_experts, plan.capacity,
              int(zero_rest), ptr(out))
    return out


def _run_unsort(rows, plan, weights, out):
    h = rows.size(1)
    if out is None:
        out = torch.empty((plan.num_tokens, h), dtype=rows.dtype, device=rows.device)
    ck.launch(rows.device, lib().bgmoe_token_unsort, ptr(rows), ck.dtype_code(rows, "rows"), ptr(plan.topk_pos),
              ptr(weights), plan.num_tokens, plan.top_k, h, ptr(out))
    return out


def _sort_backward(ctx, d_rows):
    return _run_unsort(d_rows.contiguous(), ctx.plan, None, None)


def _unsort_backward(ctx, d_out, rows, weights):
    plan, d_out, h = ctx.plan, d_out.contiguous(), d_out.size(1)
    d_rows = d_weights = None
    if ctx.needs_input_grad[0]:
        d_rows = torch.empty((plan.capacity, h), dtype=d_out.dtype, device=d_out.device)
    if ctx.needs_input_grad[1]:
        d_weights = torch.empty((plan.num_tokens, plan.top_k), dtype=torch.float32, device=d_out.device)
    ck.launch(d_out.device, lib().bgmoe_token_unsort_backward, ptr(d_out), ptr(rows), ck.dtype_code(d_out, "d_out"),
              ptr(plan.topk_pos), ptr(weights), plan.num_tokens, plan.top_k, h, ptr(plan.meta),
              ptr(plan.meta) + 4 * plan.num_experts, plan.num_experts, plan.capacity, ptr(d_rows), ptr(d_weights))
    return d_rows, d_weights


# Grad mode is on in a backward pass only while a graph of it is being recorded (create_graph=True).
class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return _run_sort(x, plan, None)

    @staticmethod
    def backward(ctx, d_rows):
        if not torch.is_grad_enabled():
            return _sort_backward(ctx, d_rows), None
        with torch.no_grad():
            d_x = _sort_backward(ctx, d_rows)
        return no_second_gradient("sort_tokens", d_x, d_rows), None


class _Unsort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan):
        ctx.plan = plan
        # the rows' gradient reads the weights, the weights' gradient the rows
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weights if ctx.needs_input_grad[0] else None)
        return _run_unsort(rows, plan, weights, None)

    @staticmethod
    def backward(ctx, d_out):
        rows, weights = ctx.saved_tensors                 # once: checkpointing recomputes them at the first access
        if not torch.is_grad_enabled():
            return (*_unsort_backward(ctx, d_out, rows, weights), None)
        with torch.no_grad():
            d_rows, d_weights = _unsort_backward(ctx, d_out, rows, weights)
        return (no_second_gradient("unsort_tokens", d_rows, d_out, weights),
                no_second_gradient("unsort_tokens", d_weights, d_out, rows), None)


def sort_tokens(x: torch.Tensor, plan: TokenSortPlan, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [N, H]`` -> ``[plan.capacity, H]``: row ``topk_pos[t, j]`` holds token t.  Any element type of 1, 2 or 4 bytes
    moves (int8 and FP8 rows, their fp32 scales as ``[N, 1]``); bf16, fp16 and fp32 have a gradient.

    Rows that hold no pair (alignment padding, rows at or past ``cu_seqlens[E]``) are zero in a fresh result; in a
    caller's ``out`` they are left as they were.  ``out`` is for inference: it is refused where a gradient is wanted, and
    shares no memory with ``x``."""
    x = _tokens(x, plan, "x", plan.num_tokens)
    if x.element_size() not in (1, 2, 4):
        ck.fail(f"x must have elements of 1, 2 or 4 bytes, got {x.dtype}")
    ck.no_tangent("sort_tokens", x)
    wants_grad = torch.is_grad_enabled() and x.requires_grad
    if out is None:
        if wants_grad:
            ck.dtype_code(x, "x")
            return _Sort.apply(x, plan)
    else:
        _buffer(out, x, (plan.capacity, x.size(1)), "out")
        if wants_grad:
            ck.fail("sort_tokens: out= has no gradient; call it without out, or under torch.no_grad()")
        ck.writable("sort_tokens", out)
        ck.apart("sort_tokens", out, x, plan.topk_pos, plan.meta)
    rows = _run_sort(x, plan, out)
    if out is not None:
        ck.written(out)
    return rows


def unsort_tokens(rows: torch.Tensor, plan: TokenSortPlan, weights: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rows [plan.capacity, H]`` (bf16, fp16 or fp32) -> ``[N, H]``: ``sum_j weights[t, j] * rows[topk_pos[t, j]]`` in
    fp32, one rounding; a token without a row gives zeros.  ``weights [N, K]`` (fp32, or a type that is cast to it);
    None: a plain sum.  ``out`` is for inference and shares no memory with the operands."""
    rows = _tokens(rows, plan, "rows", plan.capacity)
    if not rows.is_contiguous():
        rows = rows.contiguous()
    ck.dtype_code(rows, "rows")
    if weights is not None:
        ck.gpu(weights, "weights")
        ck.same_device(rows, weights, "weights")
        if tuple(weights.shape) != (plan.num_tokens, plan.top_k) or not weights.is_floating_point():
            ck.fail(f"weights must be floating [{plan.num_tokens}, {plan.top_k}], got {weights.dtype} {tuple(weights.shape)}")
        if weights.dtype != torch.float32:
            weights = weights.float()
        if not weights.is_contiguous():
            weights = weights.contiguous()
    ck.no_tangent("unsort_tokens", rows, weights)
    wants_grad = torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad))
    if out is None:
        if wants_grad:
            return _Unsort.apply(rows, weights, plan)
    else:
        _buffer(out, rows, (plan.num_tokens, rows.size(1)), "out")
        if wants_grad:
            ck.fail("unsort_tokens: out= has no gradient; call it without out, or under torch.no_grad()")
        ck.writable("unsort_tokens", out)
        ck.apart("unsort_tokens", out, rows, weights, plan.topk_pos, plan.meta)
    tokens = _run_unsort(rows, plan, weights, out)
    if out is not None:
        ck.written(out)
    return tokens
