"""The seam between two blocks in one pass: the RMSNorm behind a block, its gate and residual scale, the residual sum
and the RMSNorm in front of the next block; differentiable, and a form that also hands the next int8 product its rows.

    p = RMSNorm(block) * post_weight                  (post_weight None: p = block)
    y = residual + residual_scale * gate * p          (gate None: 1)
    normed = RMSNorm(y) * pre_weight                  (pre_weight None: not computed)

``cuda_add_rmsnorm_fp8_quant`` is the reference's form without the first norm, the gate and the gradient; these have no
counterpart there.  fp32 throughout, each output rounded once (``normed`` from the unrounded ``y``).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .._lib import lib, ptr
from ..kernels import _checks as ck
from ..kernels._autograd import no_second_gradient
from ..quantization.int8 import no_grad_needed

MAX_HIDDEN = 16384
_NONE, _CHANNEL, _TOKEN, _FULL = range(4)


def _constant(value, name):
    """residual_scale and eps are numbers: a tensor's derivative would be lost."""
    if isinstance(value, torch.Tensor):
        ck.no_tangent(f"gated_residual_rmsnorm({name}=)", value)
        if value.requires_grad and torch.is_grad_enabled():
            ck.fail(f"{name} has no gradient: pass a number (a learned scale can be the gate)")


class _Call:
    """The checked operands of one call: 2-D views, codes and flags of the C ABI."""
    __slots__ = ("code", "rows", "h", "gate_mode", "param_fp32", "scale", "eps", "device")

    def __init__(self, block, residual, post, gate, pre, scale, eps):
        ck.gpu(block, "block")
        self.code = ck.dtype_code(block, "block")
        ck.gpu(residual, "residual")
        ck.same_device(block, residual, "residual")
        if residual.dtype != block.dtype or residual.shape != block.shape:
            ck.fail(f"residual must be {block.dtype} {tuple(block.shape)} like block, got {residual.dtype} "
                    f"{tuple(residual.shape)}")
        if block.dim() < 1 or not 1 <= block.size(-1) <= MAX_HIDDEN:
            ck.fail(f"block must be [..., H] with H in [1, {MAX_HIDDEN}], got {tuple(block.shape)}")
        h = self.h = block.size(-1)
        self.rows = block.numel() // h
        self.device = block.device
        if type(scale) is not float or type(eps) is not float:
            _constant(scale, "residual_scale")
            _constant(eps, "eps")
        self.scale, self.eps = float(scale), float(eps)
        self.param_fp32 = 0
        for bit, p, name in ((1, post, "post_weight"), (2, gate, "gate"), (4, pre, "pre_weight")):
            if p is None:
                continue
            ck.gpu(p, name)
            ck.same_device(block, p, name)
            if p.dtype == torch.float32:
                self.param_fp32 |= bit
            elif p.dtype != block.dtype:
                ck.fail(f"{name} must be {block.dtype} or float32, got {p.dtype}")
            if bit != 2 and tuple(p.shape) != (h,):
                ck.fail(f"{name} must be [{h}], got {tuple(p.shape)}")
        if gate is None:
            self.gate_mode = _NONE
        elif tuple(gate.shape) == (h,):
            self.gate_mode = _CHANNEL
        elif gate.shape == block.shape:
            self.gate_mode = _FULL
        elif gate.shape == block.shape[:-1] + (1,):
            self.gate_mode = _TOKEN
        else:
            ck.fail(f"gate must be [{h}], {tuple(block.shape[:-1]) + (1,)} or {tuple(block.shape)}, got {tuple(gate.shape)}")


def _forward(c, block, residual, post, gate, pre, y, normed, q, q_scale, inv_post, inv_pre):
    if c.rows:
        ck.launch(c.device, lib().bgmoe_gated_residual_norm, ptr(block), ptr(residual), c.code, ptr(post), ptr(gate),
                  c.gate_mode, c.scale, ptr(pre), c.param_fp32, c.rows, c.h, c.eps, ptr(y), ptr(normed), ptr(q),
                  ptr(q_scale), inv_post, inv_pre)


def _backward(ctx, saved, d_y, d_normed):
    block, residual, post, gate, pre, inv = saved
    c, need = ctx.call, ctx.needs_input_grad
    if d_y is None and d_normed is None:
        return None, None, None, None, None, None
    grads = [torch.empty_like(t) if t is not None and need[i] else None
             for i, t in enumerate((block, residual, post, gate, pre))]
    d_block, d_residual, d_post, d_gate, d_pre = grads
    if c.rows == 0:
        for g in grads:
            if g is not None:
                g.zero_()
        return (*grads, None)
    d_y = None if d_y is None else d_y.contiguous()
    d_normed = None if d_normed is None else d_normed.contiguous()
    nbytes = 0
    if d_post is not None or d_pre is not None or (d_gate is not None and c.gate_mode == _CHANNEL):
        nbytes = int(lib().bgmoe_gated_residual_norm_backward_workspace_bytes(c.rows, c.h))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=c.device) if nbytes else None
    ck.launch(c.device, lib().bgmoe_gated_residual_norm_backward, ptr(block), ptr(residual), c.code, ptr(post),
              ptr(gate), c.gate_mode, c.scale, ptr(pre), c.param_fp32, c.rows, c.h, ptr(inv), ptr(inv) + 4 * c.rows,
              ptr(d_y), ptr(d_normed), ptr(d_block), ptr(d_residual), ptr(d_post), ptr(d_gate), ptr(d_pre), ptr(ws),
              nbytes)
    return (*grads, None)


def _tied_to_sources(saved, d_y, d_normed, grads):
    """The gradients of (block, residual, post, gate, pre) with what each of them depends on."""
    block, residual, post, gate, pre, _ = saved
    if d_normed is not None:                              # through the second norm: on everything, but linearly on pre
        every = (block, residual, post, gate, d_y, d_normed)
        sources = ((*every, pre),) * 4 + (every,)
    else:                                                 # y is linear in residual, post_weight and gate
        sources = ((d_y, post, gate) + ((block,) if post is not None else ()), (d_y,), (d_y, block, gate), (d_y, block, post), ())
    return [no_second_gradient("gated_residual_rmsnorm", g, *s) for g, s in zip(grads, sources)]


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, block, residual, post, gate, pre, call):
        ctx.set_materialize_grads(False)
        y = torch.empty_like(block)
        normed = torch.empty_like(block) if pre is not None else None
        inv = torch.empty((2, call.rows), dtype=torch.float32, device=call.device)
        _forward(call, block, residual, post, gate, pre, y, normed, None, None, inv.data_ptr(),
                 inv.data_ptr() + 4 * call.rows)
        ctx.call = call
        ctx.save_for_backward(block, residual, post, gate, pre, inv)
        return y, normed

    @staticmethod
    def backward(ctx, d_y, d_normed):
        saved = ctx.saved_tensors                         # once: checkpointing recomputes them at the first access
        if not torch.is_grad_enabled():
            return _backward(ctx, saved, d_y, d_normed)
        with torch.no_grad():                             # a graph of the backward pass is being recorded
            grads = _backward(ctx, saved, d_y, d_normed)
        return (*_tied_to_sources(saved, d_y, d_normed, grads[:5]), None)


def _contiguous(*tensors):
    return tuple(t if t is None or t.is_contiguous() else t.contiguous() for t in tensors)


def gated_residual_rmsnorm(block: torch.Tensor, residual: torch.Tensor, *, post_weight: Optional[torch.Tensor] = None,
                           gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                           pre_weight: Optional[torch.Tensor] = None, eps: float = 1e-5
                           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``block``, ``residual`` ``[..., H]`` (bf16, fp16 or fp32, H <= 16384) -> ``(y, normed)``; ``normed`` is None
    without ``pre_weight``.  ``gate``: ``[H]`` (per channel), ``[..., 1]`` (per token) or ``[..., H]``.  Weights and gate
    have block's type or fp32.  Gradients reach all five tensors, each in its tensor's type; they have no gradient of their
    own and there is no forward-mode derivative (asking for either raises)."""
    c = _Call(block, residual, post_weight, gate, pre_weight, residual_scale, eps)
    ck.no_tangent("gated_residual_rmsnorm", block, residual, post_weight, gate, pre_weight)
    block, residual, post_weight, gate, pre_weight = _contiguous(block, residual, post_weight, gate, pre_weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (block, residual, post_weight, gate, pre_weight)):
        return _GatedNorm.apply(block, residual, post_weight, gate, pre_weight, c)
    y = torch.empty_like(block)
    normed = torch.empty_like(block) if pre_weight is not None else None
    _forward(c, block, residual, post_weight, gate, pre_weight, y, normed, None, None, None, None)
    return y, normed


def gated_residual_rmsnorm_int8_quant(block: torch.Tensor, residual: torch.Tensor, *,
                                      post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                                      residual_scale: float = 1.0, pre_weight: torch.Tensor = None, eps: float = 1e-5,
                                      out: Optional[torch.Tensor] = None
                                      ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The serving form: ``(y, normed, q, scale)`` with ``(q, scale)`` the bits of ``int8_quant_rows(normed)`` from the
    same pass.  ``out`` takes ``y`` and may be ``residual`` itself (the running residual updated in place), ``block`` or a
    full ``gate``, but shares no part of their memory otherwise."""
    if pre_weight is None:
        ck.fail("gated_residual_rmsnorm_int8_quant needs pre_weight: the int8 rows are those of the second norm")
    no_grad_needed("gated_residual_rmsnorm_int8_quant", block, residual, post_weight, gate, pre_weight)
    c = _Call(block, residual, post_weight, gate, pre_weight, residual_scale, eps)
    if out is not None:
        ck.cuda_tensor(block, out, block.dtype, "out")
        if out.shape != block.shape:
            ck.fail(f"out must have the shape {tuple(block.shape)}, got {tuple(out.shape)}")
        ck.writable("gated_residual_rmsnorm_int8_quant", out)
    block, residual, post_weight, gate, pre_weight = _contiguous(block, residual, post_weight, gate, pre_weight)
    if out is not None:                                   # a thread reads its elements of these before it writes y there
        ck.apart("gated_residual_rmsnorm_int8_quant", out, post_weight, pre_weight, same_ok=(block, residual, gate))
    y = torch.empty_like(block) if out is None else out
    normed = torch.empty_like(block)
    q = torch.empty(block.shape, dtype=torch.int8, device=c.device)
    scale = torch.empty(block.shape[:-1], dtype=torch.float32, device=c.device)
    _forward(c, block, residual, post_weight, gate, pre_weight, y, normed, q, scale, None, None)
    if out is not None:
        ck.written(out)
    return y, normed, q, scale
