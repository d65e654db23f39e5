"""Root-mean-square norm over the last dimension, with the residual's addition.

``rms_norm(x, w)``                        y = x / sqrt(mean(x^2) + eps) * w
``add_rms_norm(x, residual, w)``          (y, h): h = x + residual in x's dtype, y = the norm of h
``rms_norm_quantized(x, w, residual=...)`` the same, y as an ``MXTensor`` (8- or 4-bit with block scales)

CUDA (bf16, fp16, fp32; rows of up to 16384 elements; weight in the input's dtype or fp32): one
kernel, fp32 statistics, every element read once; the first two are differentiable (the residual
and x share one gradient tensor; the weight's gradient is summed in a fixed order).  The quantised
form rounds the fp32 result once, to the format, and has no gradient.  CPU: the plain fp32
definition (the oracle).  No counterpart in the reference, whose norms are all LayerNorms.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._ext import kernels
from .microscale import MXTensor, _check_scalar, _no_grad_here, format_id, quantize_reference

__all__ = ["rms_norm", "add_rms_norm", "rms_norm_quantized"]


MAX_DIM = 16384      # elements of a row


def _check(x, weight, residual):      # what the kernels' wrappers refuse, for CPU tensors
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("rms_norm: needs a last dimension of at least one element")
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"rms_norm: bf16, fp16 or fp32 expected, got {x.dtype}")
    if x.shape[-1] > MAX_DIM:
        raise ValueError(f"rms_norm: rows of at most {MAX_DIM} elements")
    if weight.device != x.device or weight.shape != x.shape[-1:] or weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"rms_norm: weight must be [{x.shape[-1]}] of the input's dtype or fp32, on its device")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("rms_norm: residual must match the input's shape, dtype and device")


def _reference(x, weight, residual, eps):
    """(fp32 y, h) of the definition."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    return hf * torch.rsqrt(hf.square().mean(-1, keepdim=True) + eps) * weight.float(), h


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """RMS norm over the last dimension, in x's dtype; differentiable."""
    if x.is_cuda:
        return kernels().rms_norm(x, weight, None, eps)[0]
    _check(x, weight, None)
    return _reference(x, weight, None, eps)[0].to(x.dtype)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(RMS norm of h, h) with h = x + residual: the branch's output joins the residual stream and is normalised
    for the next branch in one pass.  The norm reads h as it is stored (rounded to x's dtype); differentiable."""
    if x.is_cuda:
        y, h = kernels().rms_norm(x, weight, residual, eps)
        return y, h
    _check(x, weight, residual)
    y, h = _reference(x, weight, residual, eps)
    return y.to(x.dtype), h


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                       residual: Optional[torch.Tensor] = None, fmt: str = "mxfp8",
                       global_scale: Optional[torch.Tensor] = None) -> Tuple[MXTensor, torch.Tensor]:
    """(quantised RMS norm of h, h), h = x (+ residual): the input of ``mx_linear``, without a 16-bit copy.
    ``fmt``: "mxfp8", "mxfp4" or "nvfp4" (with its tensor scale, fp32 [1]; default 1: blocks with maxima from 0.094 to
    2688 keep full precision, see ``mx_linear``).  No gradient."""
    f = format_id(fmt)
    if x.is_cuda:
        codes, scales, h = kernels().rms_norm_quantized(x, weight, residual, eps, f, global_scale)
        return MXTensor(codes, scales, fmt, x.shape, global_scale), x if residual is None else h
    _check(x, weight, residual)
    _no_grad_here("rms_norm_quantized", x, weight, residual)
    if global_scale is not None and fmt != "nvfp4":
        raise ValueError("rms_norm_quantized: only nvfp4 has a tensor scale")
    _check_scalar(global_scale, x, "rms_norm_quantized")
    y, h = _reference(x, weight, residual, eps)
    codes, scales = quantize_reference(y.reshape(-1, x.shape[-1]), fmt, global_scale)
    return MXTensor(codes, scales, fmt, x.shape, global_scale), h
