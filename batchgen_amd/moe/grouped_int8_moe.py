"""The experts' products in 8-bit integers, next to the FP8 (``grouped_fp8_blockwise_moe``) and MXFP4 forms: rows
grouped by expert (``token_sort`` or the ragged dispatch) times one int8 ``[N, K]`` matrix per expert, with one scale
per row and one per output channel.  No counterpart in the reference.

* ``int8_grouped_gemm``: the down projection, or any grouped product;
* ``int8_fused_s1``: gate and up with ``silu(gate) * up`` in the epilogue (fp32 in between, one rounding).

Rows of expert g are ``[cu_seqlens[g], cu_seqlens[g] + seqlens[g])``; rows of no expert are neither read nor written.
Counts and offsets stay on the device.  Inference only: no gradient.
"""
from __future__ import annotations

from typing import Optional

import torch

from .._lib import lib, ptr
from ..kernels import _checks as ck
from ..quantization.int8 import no_grad_needed


def _rows(x, x_scale, seqlens, cu_seqlens, e):
    ck.cuda_tensor(None, x, torch.int8, "x")
    if x.dim() != 2:
        ck.fail(f"x must be int8 [rows, K], got {tuple(x.shape)}")
    m, k = x.shape
    ck.int32(k, "K")
    ck.int32(e, "E")
    ck.cuda_tensor(x, x_scale, torch.float32, "x_scale")
    if x_scale.numel() != m:
        ck.fail(f"x_scale must hold one element per row ({m}), got {x_scale.numel()}")
    ck.cuda_tensor(x, seqlens, torch.int32, "seqlens")
    ck.cuda_tensor(x, cu_seqlens, torch.int32, "cu_seqlens")
    if seqlens.numel() != e or cu_seqlens.numel() < e:
        ck.fail(f"seqlens must hold {e} and cu_seqlens at least {e} elements, got {seqlens.numel()} and "
                f"{cu_seqlens.numel()}")
    return m, k


def _weight(x, w, s, k, name):
    """Checks ``w [E, N, K]`` / ``s [E, N]`` (experts may be strided, e.g. halves of a stacked ``[E, 2N, K]``)."""
    if w.dtype is torch.int8 and s.dtype is torch.float32 and w.is_contiguous() and s.is_contiguous() and w.dim() == 3 and \
            w.size(2) == k and s.shape == w.shape[:2] and w.get_device() == s.get_device() == x.get_device():
        return
    ck.gpu(w, name)
    ck.same_device(x, w, name)
    ck.dtype(w, torch.int8, name)
    if w.dim() != 3 or w.size(2) != k or (w.numel() and (w.stride(2) != 1 or w.stride(1) != k)):
        ck.fail(f"{name} must be int8 [E, N, K = {k}] with contiguous matrices, got {tuple(w.shape)} strides {w.stride()}")
    ck.gpu(s, name + "_scale")
    ck.same_device(x, s, name + "_scale")
    ck.dtype(s, torch.float32, name + "_scale")
    if tuple(s.shape) != tuple(w.shape[:2]) or (s.numel() and s.stride(1) != 1):
        ck.fail(f"{name}_scale must be fp32 {tuple(w.shape[:2])} with contiguous rows, got {tuple(s.shape)}")


def _out(name, x, out, out_dtype, m, n):
    ck.int32(n, "N")
    dt = out.dtype if out is not None else (out_dtype or torch.bfloat16)
    code = ck.DTYPE_CODE.get(dt)
    if code is None or (out is not None and out_dtype not in (None, out.dtype)):
        ck.fail(f"output type must be bfloat16, float16 or float32 (and out's own), got {out_dtype or dt}")
    if out is None:
        return torch.empty((m, n), dtype=dt, device=x.device), code
    ck.cuda_tensor(x, out, dt, "out")
    if tuple(out.shape) != (m, n):
        ck.fail(f"out must have the shape {(m, n)}, got {tuple(out.shape)}")
    ck.writable(name, out)
    return out, code


def int8_grouped_gemm(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                      seqlens: torch.Tensor, cu_seqlens: torch.Tensor, out: Optional[torch.Tensor] = None,
                      out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x`` int8 ``[rows, K]``, ``x_scale`` fp32 ``[rows]``, ``weight`` int8 ``[E, N, K]``, ``weight_scale`` fp32
    ``[E, N]``, ``seqlens`` int32 ``[E]``, ``cu_seqlens`` int32 ``[E (+ 1)]`` -> ``[rows, N]`` (bf16 unless ``out_dtype``
    or ``out`` says otherwise; rows of no expert keep what ``out`` held, which shares no memory with the operands)."""
    no_grad_needed("int8_grouped_gemm", x_scale, weight_scale)
    held = out
    e = weight.size(0) if isinstance(weight, torch.Tensor) and weight.dim() == 3 else 0
    m, k = _rows(x, x_scale, seqlens, cu_seqlens, e)
    _weight(x, weight, weight_scale, k, "weight")
    n = weight.size(1)
    out, code = _out("int8_grouped_gemm", x, out, out_dtype, m, n)
    if m and n:
        if held is not None:
            ck.apart("int8_grouped_gemm", out, x, x_scale, weight, weight_scale, seqlens, cu_seqlens)
        ck.launch(x.device, lib().bgmoe_int8_grouped_gemm, ptr(x), ptr(x_scale), ptr(weight), weight.stride(0),
                  ptr(weight_scale), weight_scale.stride(0), ptr(seqlens), ptr(cu_seqlens), e, m, n, k, ptr(out),
                  code)
        if held is not None:
            ck.written(held)
    return out


def int8_fused_s1(x: torch.Tensor, x_scale: torch.Tensor, gate_weight: torch.Tensor, gate_scale: torch.Tensor,
                  up_weight: torch.Tensor, up_scale: torch.Tensor, seqlens: torch.Tensor, cu_seqlens: torch.Tensor,
                  out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``silu(x @ gate^T) * (x @ up^T)`` per expert; operands as ``int8_grouped_gemm`` with ``gate_weight`` and
    ``up_weight`` int8 ``[E, N, K]``."""
    no_grad_needed("int8_fused_s1", x_scale, gate_scale, up_scale)
    held = out
    e = gate_weight.size(0) if isinstance(gate_weight, torch.Tensor) and gate_weight.dim() == 3 else 0
    m, k = _rows(x, x_scale, seqlens, cu_seqlens, e)
    _weight(x, gate_weight, gate_scale, k, "gate_weight")
    _weight(x, up_weight, up_scale, k, "up_weight")
    if up_weight.shape != gate_weight.shape:
        ck.fail(f"gate_weight {tuple(gate_weight.shape)} and up_weight {tuple(up_weight.shape)} must have one shape")
    n = gate_weight.size(1)
    out, code = _out("int8_fused_s1", x, out, out_dtype, m, n)
    if m and n:
        if held is not None:
            ck.apart("int8_fused_s1", out, x, x_scale, gate_weight, gate_scale, up_weight, up_scale, seqlens, cu_seqlens)
        ck.launch(x.device, lib().bgmoe_int8_fused_s1, ptr(x), ptr(x_scale), ptr(gate_weight), gate_weight.stride(0),
                  ptr(gate_scale), gate_scale.stride(0), ptr(up_weight), up_weight.stride(0), ptr(up_scale),
                  up_scale.stride(0), ptr(seqlens), ptr(cu_seqlens), e, m, n, k, ptr(out), code)
        if held is not None:
            ck.written(held)
    return out
