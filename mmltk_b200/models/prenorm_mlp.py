"""A pre-norm MLP block on the RMS norm, and its low-precision serving form.

``PreNormMlp``            h = x + residual; y = fc2(GELU(fc1(rms_norm(h)))); returns (y, h) -- y is the next
                          block's x, h its residual.  Trainable.
``PreNormMlp.quantize``   the same block with 8- or 4-bit weights: three kernels for norm + fc1 + fc2 in mxfp8
                          (the norm and fc1 write the next product's 8-bit input), no gradient.

No counterpart in the reference, whose blocks use LayerNorm and 16-bit linears.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from .. import ops

__all__ = ["PreNormMlp", "QuantizedPreNormMlp"]


class PreNormMlp(nn.Module):
    def __init__(self, dim: int, hidden: int, eps: float = 1e-6):
        super().__init__()
        self.norm_weight = nn.Parameter(torch.ones(dim))
        self.fc1, self.fc2 = nn.Linear(dim, hidden), nn.Linear(hidden, dim)
        self.eps = eps

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        if residual is None:
            n, h = ops.rms_norm(x, self.norm_weight, self.eps), x
        else:
            n, h = ops.add_rms_norm(x, residual, self.norm_weight, self.eps)
        n = ops.linear(n, self.fc1.weight, self.fc1.bias, act="gelu")
        return ops.linear(n, self.fc2.weight, self.fc2.bias), h

    @torch.no_grad()
    def quantize(self, fmt: str = "mxfp8") -> "QuantizedPreNormMlp":
        """The serving form of the present parameters: a copy, which later updates of this module do not reach."""
        copy = lambda t: None if t is None else t.detach().clone()  # noqa: E731
        return QuantizedPreNormMlp(copy(self.norm_weight), ops.mx_quantize(self.fc1.weight, fmt), copy(self.fc1.bias),
                                   ops.mx_quantize(self.fc2.weight, fmt), copy(self.fc2.bias), self.eps)


class QuantizedPreNormMlp:
    """Weights as ``MXTensor``; ``block(x, residual)`` as ``PreNormMlp``, from one token to long batches.

    nvfp4's tensor scales of the two inner activations follow from the weights, not from the data: a normalised row
    has a length of at most sqrt(dim), so |n_j| <= sqrt(dim) |w_j| for the norm's output and |z_j| <= sqrt(dim) |W1_j w| +
    |b_j| before the GELU, which only shrinks.  With these bounds at the top of the grid nothing saturates (but for what
    the rounding of n adds), a token's result does not depend on its batch, and blocks whose maximum is at least
    1 / 28672 of the bound keep full precision."""

    def __init__(self, norm_weight, w1: ops.MXTensor, b1, w2: ops.MXTensor, b2, eps: float = 1e-6):
        if w1.fmt != w2.fmt or w1.shape[0] != w2.shape[1]:
            raise ValueError(f"weights {w1} and {w2} do not make an MLP")
        self.norm_weight, self.w1, self.w2, self.eps = norm_weight, w1, w2, eps
        self.b1, self.b2 = (None if b is None else b.detach() for b in (b1, b2))
        self.scale1, self.scale2 = self._act_scales() if w1.fmt == "nvfp4" else (None, None)

    @torch.no_grad()
    def _act_scales(self):
        w = self.norm_weight.double()
        z = (self.w1.dequantize(torch.float32) * w).square().sum(-1).sqrt() * len(w) ** 0.5
        if self.b1 is not None:
            z = z + self.b1.double().abs()

        def scale(bounds):      # rows that are not finite answer for themselves
            top = torch.where(torch.isfinite(bounds), bounds, 0.0).amax()
            return torch.where(top > 0, (top / 2688).clamp(min=2.0 ** -100), 1.0).float().reshape(1)
        return scale(w.abs() * len(w) ** 0.5), scale(z)

    @torch.no_grad()
    def __call__(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        fmt = self.w1.fmt
        n, h = ops.rms_norm_quantized(x, self.norm_weight, self.eps, residual=residual, fmt=fmt,
                                      global_scale=self.scale1)
        if fmt == "mxfp8":      # the hidden activations leave the first product in the second one's format
            n = ops.mx_linear(n, self.w1, self.b1, act="gelu", out_fmt=fmt)
        else:
            n = ops.mx_linear(n, self.w1, self.b1, act="gelu", out_dtype=x.dtype)
        return ops.mx_linear(n, self.w2, self.b2, out_dtype=x.dtype, act_scale=self.scale2), h
