"""8-bit integers with one scale per token and one per output channel (W8A8): the row quantiser and the dense product.
The product over rows grouped by expert is ``batchgen_amd.moe.grouped_int8_moe``.

``q[t, k] = rint(x[t, k] / s[t])`` with ``s[t] = max_k |x[t, k]| / 127``;
``out[t, j] = (sum_k q[t, k] * w[j, k]) * s[t] * c[j] (+ bias[j])``: the sum is an exact 32-bit integer, the rest fp32
with one rounding to the output type.  A token that holds an infinity or a NaN gives NaN outputs.  Both ops belong to
inference: they have no derivative and refuse operands that require a gradient while grad mode is on, or that carry
a forward-mode tangent.  They have no counterpart
in the reference, whose quantised products are FP8 and MXFP4.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .._lib import lib, ptr
from ..kernels import _checks as ck


def no_grad_needed(name: str, *tensors):
    ck.no_tangent(name, *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                ck.fail(f"{name} has no gradient: call it under torch.no_grad() or detach its operands")


def int8_quant_rows(x: torch.Tensor, out: Optional[torch.Tensor] = None,
                    scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [..., K]`` (bf16, fp16 or fp32) -> ``(q int8 [..., K], scale fp32 [...])``; ``out`` / ``scale`` take them
    and share no memory with ``x``."""
    ck.gpu(x, "x")
    no_grad_needed("int8_quant_rows", x)
    held = (out, scale)                                   # the caller's tensors
    code = ck.dtype_code(x, "x")
    if x.dim():
        ck.int32(x.size(-1), "K")
    x2 = ck.rows_of(x, "x")
    rows, k = x2.shape
    if out is None:
        out = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    else:
        ck.cuda_tensor(x, out, torch.int8, "out")
        if out.shape != x.shape:
            ck.fail(f"out must have the shape of x, {tuple(x.shape)}, got {tuple(out.shape)}")
    if scale is None:
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    else:
        ck.cuda_tensor(x, scale, torch.float32, "scale")
        if scale.shape != x.shape[:-1]:
            ck.fail(f"scale must have the shape {tuple(x.shape[:-1])}, got {tuple(scale.shape)}")
    ck.writable("int8_quant_rows", *held)
    if rows and k == 0:
        ck.fail("int8_quant_rows: rows without elements have no scale")
    if rows:
        if held[0] is not None:
            ck.apart("int8_quant_rows", out, x2, scale)
        if held[1] is not None:
            ck.apart("int8_quant_rows", scale, x2, out)
        ck.launch(x.device, lib().bgmoe_int8_quant_rows, ptr(x2), code, x2.stride(0), rows, k, ptr(out), ptr(scale))
        ck.written(*(t for t in held if t is not None))
    return out, scale


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                x_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [..., K] -> [..., N]`` with ``weight`` int8 ``[N, K]`` and ``weight_scale`` fp32 ``[N]``.

    ``x`` bf16, fp16 or fp32: quantised per token here (the bits of ``int8_quant_rows``), the output has its type unless
    ``out_dtype`` says otherwise.  ``x`` int8 with ``x_scale`` fp32 ``[...]``: used as it is, the output is bf16 unless
    ``out_dtype`` says otherwise.  ``bias``: fp32 ``[N]``.  ``out``: contiguous ``[..., N]``, apart from the
    operands' memory (only an ``x`` that is quantised here may be ``out``).  K is a multiple of 16, at
    most 131071 (beyond it a sum could leave 32 bits)."""
    ck.gpu(x, "x")
    no_grad_needed("int8_linear", x, x_scale, weight_scale, bias)
    held = out
    ck.cuda_tensor(x, weight, torch.int8, "weight")
    if weight.dim() != 2 or x.dim() < 1 or x.size(-1) != weight.size(1):
        ck.fail(f"int8_linear: x [..., K] and weight [N, K] do not fit: {tuple(x.shape)}, {tuple(weight.shape)}")
    n, k = weight.shape
    ck.int32(n, "N")
    ck.int32(k, "K")
    ck.cuda_tensor(x, weight_scale, torch.float32, "weight_scale")
    if weight_scale.numel() != n:
        ck.fail(f"weight_scale must hold N = {n} elements, got {weight_scale.numel()}")
    if bias is not None:
        ck.cuda_tensor(x, bias, torch.float32, "bias")
        if bias.numel() != n:
            ck.fail(f"bias must hold N = {n} elements, got {bias.numel()}")
    quantised = x.dtype == torch.int8
    if quantised != (x_scale is not None):
        ck.fail("int8_linear: x_scale goes with an int8 x, and only with it")
    if quantised:
        ck.cuda_tensor(x, x_scale, torch.float32, "x_scale")
        if x_scale.shape != x.shape[:-1] and x_scale.numel() != x.numel() // max(k, 1):
            ck.fail(f"x_scale must hold one element per row of x {tuple(x.shape)}, got {tuple(x_scale.shape)}")
    x2 = ck.rows_of(x, "x")
    m = x2.size(0)
    dt = out.dtype if out is not None else (out_dtype or (torch.bfloat16 if quantised else x.dtype))
    code = ck.DTYPE_CODE.get(dt)
    if code is None or (out is not None and out_dtype not in (None, out.dtype)):
        ck.fail(f"int8_linear: output type must be bfloat16, float16 or float32 (and out's own), got {out_dtype or dt}")
    shape = x.shape[:-1] + (n,)
    if out is None:
        out = torch.empty(shape, dtype=dt, device=x.device)
    else:
        ck.cuda_tensor(x, out, dt, "out")
        if out.shape != shape:
            ck.fail(f"out must have the shape {tuple(shape)}, got {tuple(out.shape)}")
        ck.writable("int8_linear", out)
    if m == 0 or n == 0:
        return out
    if quantised:
        row_stride = x2.stride(0) if m > 1 else k
        if x2.data_ptr() % 16 or row_stride % 16 or row_stride >= 1 << 24:  # what the kernels' loads take
            x2, row_stride = x2.clone(memory_format=torch.contiguous_format), k
        if held is not None:
            ck.apart("int8_linear", out, x2, x_scale, weight, weight_scale, bias)
        ck.launch(x.device, lib().bgmoe_int8_gemm, ptr(x2), row_stride, ptr(x_scale), ptr(weight),
                  ptr(weight_scale), ptr(bias), m, n, k, ptr(out), code, n)
    else:
        x_code = ck.dtype_code(x, "x")
        if held is not None:                              # (x itself is only read before the product: it may be out)
            ck.apart("int8_linear", out, weight, weight_scale, bias)
        # scratch of one call from torch's allocator: it follows the stream it is used on, and under graph capture it
        # belongs to the graph, so two captured graphs never share it
        ws = torch.empty(lib().bgmoe_int8_linear_workspace_bytes(m, n, k), dtype=torch.uint8, device=x.device)
        ck.launch(x.device, lib().bgmoe_int8_linear, ptr(x2), x_code, x2.stride(0), ptr(weight), ptr(weight_scale),
                  ptr(bias), m, n, k, ptr(out), code, n, ptr(ws), ws.numel())
    if held is not None:
        ck.written(held)
    return out
