"""Argument checks shared by the op modules (the reference's TORCH_CHECKs:
a violation raises RuntimeError before anything is launched)."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version as _increment_version

from .._lib import check

_current_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def fail(msg: str):
    raise RuntimeError(msg)


def gpu(t: torch.Tensor, name: str):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        fail(f"{name} must be a CUDA tensor")


def same_device(ref: torch.Tensor, t: torch.Tensor, name: str):
    if t.device != ref.device:
        fail(f"{name} must be on {ref.device}, got {t.device}")


def contiguous(t: torch.Tensor, name: str):
    if not t.is_contiguous():
        fail(f"{name} must be contiguous")


def dtype(t: torch.Tensor, dt, name: str):
    dts = dt if isinstance(dt, (tuple, list)) else (dt,)
    if t.dtype not in dts:
        fail(f"{name} must be {' or '.join(str(d) for d in dts)}, got {t.dtype}")


def cuda_tensor(ref, t, dt, name):
    # one expression for the common case; the checks below say what is wrong otherwise
    if isinstance(t, torch.Tensor) and t.dtype is dt and t.is_cuda and t.is_contiguous() and \
            (ref is None or t.get_device() == ref.get_device()):
        return
    gpu(t, name)
    if ref is not None:
        same_device(ref, t, name)
    contiguous(t, name)
    if dt is not None:
        dtype(t, dt, name)


def combine_args(expert_output, topk_pos, topk_weights, output, n, h, k, out_dtype):
    """The weighted combines read ``topk_pos`` / ``topk_weights`` [n*k] and ``expert_output`` [rows, h] and write
    ``output`` [n, h]: dtype, device, contiguity and minimum sizes, so that no wrong-typed or short tensor is
    ever handed to the kernel as a raw pointer."""
    if n < 0 or h <= 0:
        fail(f"N must be >= 0 and H positive, got N={n} H={h}")
    cuda_tensor(None, expert_output, torch.bfloat16, "expert_output")
    cuda_tensor(expert_output, topk_pos, torch.int32, "topk_pos")
    cuda_tensor(expert_output, topk_weights, torch.float32, "topk_weights")
    cuda_tensor(expert_output, output, out_dtype, "output")
    if topk_pos.numel() < n * k or topk_weights.numel() < n * k:
        fail(f"topk_pos / topk_weights must hold N*K = {n * k} elements")
    if output.numel() < n * h:
        fail(f"output must hold N*H = {n * h} elements")
    if expert_output.dim() < 2 or expert_output.size(-1) != h:      # [rows, H] or the masked [E_local, max_tokens, H]
        fail(f"expert_output must have rows of H={h} elements")


FP8_BYTES = (torch.uint8, torch.float8_e4m3fn)


def no_tangent(name: str, *tensors):
    """Refuses tensors that carry a forward-mode tangent: the kernels see only the values, and a result without a
    tangent would stand for a derivative of zero."""
    if forward_ad._current_level < 0:                   # outside of torch.autograd.forward_ad.dual_level()
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            fail(f"{name} has no forward-mode derivative: its operands must not carry a tangent")


def writable(name: str, *outs):
    """A caller's tensors that an op without a gradient is about to write: refused where autograd would go on with what
    they were (they require a gradient in grad mode, or carry a forward-mode tangent)."""
    if forward_ad._current_level >= 0:
        no_tangent(name, *outs)
    for t in outs:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            fail(f"{name} writes its output without a gradient: the tensor it writes must not require one in grad mode")


def _span(t: torch.Tensor) -> int:
    """Bytes from the first to the last element of a tensor that is not contiguous (and so not empty)."""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def apart(name: str, out: torch.Tensor, *operands, same_ok=()):
    """Refuses an output whose memory (first to last element) reaches into an operand's: blocks of one launch write the
    one while others still read the other.  An operand of ``same_ok`` may be the output's memory, element by element."""
    start = out.data_ptr()
    end = start + out.nbytes                            # (outputs are contiguous)
    for t in operands:
        if t is not None:
            p = t.data_ptr()
            if p < end and p + (t.nbytes if t.is_contiguous() else _span(t)) > start:
                fail(f"{name}: the output must not share memory with an operand")
    for t in same_ok:
        if t is not None:
            p = t.data_ptr()
            if p < end and p + (t.nbytes if t.is_contiguous() else _span(t)) > start and \
                    not (p == start and t.is_contiguous() and t.nbytes == out.nbytes and t.dtype == out.dtype):
                fail(f"{name}: the output must be an operand's whole memory or none of it")


def written(*outs):
    """Tells autograd that these tensors have been written, as torch's own in-place operations do: the backward pass of
    an earlier graph that saved one of them then raises instead of using the new values.  (Inference tensors, which
    have no version and cannot be saved, are passed over.)"""
    _increment_version(outs)


def launch(device: torch.device, fn, *args):
    """``fn(*args, stream)`` with ``device`` current, on its current stream.  The context manager and the stream object of
    torch.cuda take 4 us, as much as a short kernel; where the device is the current one already neither is needed."""
    index = device.index
    if index == _current_device():
        check(fn(*args, _raw_stream(index)))
    else:
        with torch.cuda.device(device):
            check(fn(*args, _raw_stream(index)))


# BGMOE_DT_*: element types of the operators that take all three
DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def dtype_code(t: torch.Tensor, name: str) -> int:
    code = DTYPE_CODE.get(t.dtype)
    if code is None:
        fail(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    return code


def int32(value: int, name: str) -> int:
    """``value`` where the C ABI takes an ``int``: ctypes would cut a larger one without a word."""
    if not -0x80000000 <= value <= 0x7fffffff:
        fail(f"{name} = {value} does not fit 32 bits")
    return value


def rows_of(t: torch.Tensor, name: str) -> torch.Tensor:
    """``t [..., K]`` as ``[rows, K]`` whose rows are contiguous (a 2-D tensor may keep a stride between its rows)."""
    if t.dim() == 2 and t.is_contiguous():
        return t
    if t.dim() == 0:
        fail(f"{name} must have at least one axis")
    if t.dim() == 2 and (t.stride(1) == 1 or t.size(1) <= 1) and (t.stride(0) >= t.size(1) or t.size(0) <= 1):
        return t
    t2 = t.reshape(-1, t.size(-1)) if t.size(-1) else t.reshape(t.numel(), 0)
    return t2 if t2.stride(1) == 1 and t2.stride(0) >= t2.size(1) else t2.contiguous()
