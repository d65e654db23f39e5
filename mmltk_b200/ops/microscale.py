"""Microscaled formats: 4- and 8-bit elements that share one scale per block of a row, and their products.

=======  ==================  =======================  =========================================
format   element (largest)   elements per scale       scale
=======  ==================  =======================  =========================================
mxfp4    e2m1 (6)            32                       power of two (e8m0)
nvfp4    e2m1 (6)            16                       e4m3, and one fp32 scale for the whole tensor
mxfp8    e4m3 (448)          32                       power of two (e8m0)
=======  ==================  =======================  =========================================

``mx_quantize(x, fmt)`` -> ``MXTensor``; ``t.dequantize(dtype)`` back; ``mx_linear(x, w, bias, act=...)``
multiplies by a quantised weight [n, k] on the block-scaled tensor cores.  A row's last block may be partial;
any sizes are allowed.

Rounding.  A power-of-two scale is the smallest one with which no element of its block saturates
(at least 2^-127).  An e4m3 scale is amax / 6 rounded to nearest, on the grid of the tensor scale
g: elements are x * (1 / (s g)).  Elements round to nearest, ties to even.  A block with an infinity
or a NaN gets a NaN scale: all its values, and what a product makes of them, are NaN; other blocks do not notice.
For nvfp4, g = (largest finite magnitude of x) * (1 / 2688, rounded to fp32) unless it is given.

Layout.  ``codes`` [rows, pitch]: rows padded to 16 bytes, 4-bit codes two to a byte, the even
element in the low half (uint8); 8-bit ones float8_e4m3fn.  ``scales`` uint8 [rows / 128, blocks / 4, 32, 4, 4]
(rounded up, zero padding): byte ``[r // 128, b // 4, r % 32, r // 32 % 4, b % 4]`` scales block b of
row r -- the tiles that the tensor cores read.

CUDA tensors run the framework's kernels; CPU tensors the plain definition (the oracle).  These are
serving operators and have no gradient.  No counterpart in the reference, which computes in 16 bits.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
import torch.nn.functional as F

from ._ext import kernels

__all__ = ["MXTensor", "mx_quantize", "mx_linear", "mx_status", "format_id", "quantize_reference",
           "dequantize_reference"]

_FORMATS = {"mxfp4": 0, "nvfp4": 1, "mxfp8": 2}
_BLOCK = {"mxfp4": 32, "nvfp4": 16, "mxfp8": 32}
_BITS = {"mxfp4": 4, "nvfp4": 4, "mxfp8": 8}
_ACTS = {None: 0, "none": 0, "gelu": 1, "relu": 2}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
WAIT_LIMIT = 1 << 22      # tries of a kernel's bounded wait (``kernels().mx_wait_limit``)
_OUT_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def format_id(fmt: str) -> int:
    try:
        return _FORMATS[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"unknown microscaled format {fmt!r} (one of {', '.join(_FORMATS)})") from None


class MXTensor:
    """A quantised tensor of logical ``shape`` [..., dim]; its blocks run along the last axis."""
    __slots__ = ("codes", "scales", "fmt", "shape", "global_scale")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, fmt: str, shape: Sequence[int],
                 global_scale: Optional[torch.Tensor] = None):
        format_id(fmt)
        if global_scale is not None and fmt != "nvfp4":
            raise ValueError(f"MXTensor: only nvfp4 has a tensor scale, not {fmt}")
        self.codes, self.scales, self.fmt, self.shape, self.global_scale = codes, scales, fmt, tuple(shape), global_scale

    @property
    def rows(self) -> int:
        n = 1
        for s in self.shape[:-1]:
            n *= s
        return n

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def to(self, device) -> "MXTensor":
        g = self.global_scale
        return MXTensor(self.codes.to(device), self.scales.to(device), self.fmt, self.shape,
                        None if g is None else g.to(device))

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values, rounded once to ``dtype`` (bf16, fp16 or fp32)."""
        if self.codes.is_cuda:
            y = kernels().mx_dequantize(self.codes, self.scales, self.global_scale, _FORMATS[self.fmt], self.rows,
                                         self.shape[-1], dtype)
        else:
            if dtype not in _OUT_DTYPES:
                raise TypeError(f"mx_dequantize: bf16, fp16 or fp32 expected, got {dtype}")
            _check_coded(self, "mx_dequantize")
            y = dequantize_reference(self).to(dtype)
        return y if len(self.shape) == 2 else y.view(self.shape)

    def __repr__(self) -> str:
        return f"MXTensor({self.fmt}, shape={self.shape}, device={self.device})"


# What the kernels' wrappers refuse, for CPU tensors.
def _check_coded(t: MXTensor, what: str) -> None:
    rows, dim, bits = t.rows, t.shape[-1], _BITS[t.fmt]
    pitch, tiles = -(-dim * bits // 128) * 16, -(-dim // (4 * _BLOCK[t.fmt]))
    if (t.codes.dtype != (torch.float8_e4m3fn if bits == 8 else torch.uint8) or tuple(t.codes.shape) != (rows, pitch)
            or not t.codes.is_contiguous()):
        raise ValueError(f"{what}: codes of {t} must be contiguous [{rows}, {pitch}]")
    if (t.scales.dtype != torch.uint8 or t.scales.device != t.codes.device or not t.scales.is_contiguous()
            or t.scales.numel() != -(-rows // 128) * tiles * 512):
        raise ValueError(f"{what}: scales of {t} must be contiguous uint8 [{-(-rows // 128)}, {tiles}, 32, 4, 4]")


def _check_scalar(g: Optional[torch.Tensor], like: torch.Tensor, what: str) -> None:
    if g is not None and (g.dtype != torch.float32 or g.numel() != 1 or g.device != like.device):
        raise ValueError(f"{what}: the tensor scale is one fp32 value on the same device")


def _no_grad_here(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what}: has no gradient (a serving operator); call it under torch.no_grad() or on "
                           "detached tensors")


def mx_quantize(x: torch.Tensor, fmt: str, global_scale: Optional[torch.Tensor] = None) -> MXTensor:
    """Quantise [..., dim] (bf16, fp16, fp32) along its last axis.  ``global_scale`` (nvfp4, fp32 [1]): the
    tensor scale to use; by default it is found from x (one more pass over it)."""
    f = format_id(fmt)
    if x.is_cuda:
        codes, scales, g = kernels().mx_quantize(x, f, global_scale)
        return MXTensor(codes, scales, fmt, x.shape, g)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("mx_quantize: needs a last dimension of at least one element")
    if x.dtype not in _OUT_DTYPES:
        raise TypeError(f"mx_quantize: bf16, fp16 or fp32 expected, got {x.dtype}")
    _no_grad_here("mx_quantize", x)
    if global_scale is not None and fmt != "nvfp4":
        raise ValueError("mx_quantize: only nvfp4 has a tensor scale")
    _check_scalar(global_scale, x, "mx_quantize")
    x2 = x.reshape(-1, x.shape[-1]).float()
    if fmt == "nvfp4" and global_scale is None:
        a = x2.abs()
        a = torch.where(torch.isfinite(a), a, torch.zeros_like(a)).amax() if x2.numel() else x2.new_zeros(())
        global_scale = torch.where(a > 0, (a * (1.0 / 2688.0)).clamp(min=2.0 ** -100), torch.ones_like(a)).reshape(1)
    codes, scales = quantize_reference(x2, fmt, global_scale)
    return MXTensor(codes, scales, fmt, x.shape, global_scale)


def mx_linear(x, weight: MXTensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
              out_dtype: Optional[torch.dtype] = None, out_fmt: Optional[str] = None,
              act_scale: Optional[torch.Tensor] = None):
    """act(x W^T + bias) with W an ``MXTensor`` [n, k]; fp32 accumulation, one rounding of the output.

    ``x``: [..., k] in bf16, fp16 or fp32, quantised to the weight's format in the call, or an ``MXTensor`` of that
    format.  ``act``: None, "gelu" (erf) or "relu".  The output is [..., n] in ``out_dtype`` (default: x's dtype, bf16
    for an ``MXTensor``) or, with ``out_fmt="mxfp8"``, an ``MXTensor``.

    ``act_scale`` (nvfp4 weight, fp32 [1]): the tensor scale g for quantising x, default 1.  Blocks of x whose maximum
    lies between 0.094 g and 2688 g keep full precision; below, their e4m3 scales are subnormal and lose bits, blocks
    under 0.0058 g are zeros (the product is then act(bias)), and values above 2688 g saturate.  For inputs
    outside that range give amax / 2688, or pass ``mx_quantize(x, "nvfp4")``, which finds it."""
    if act not in _ACTS:
        raise ValueError(f"mx_linear: unknown activation {act!r}")
    if out_fmt not in (None, "mxfp8"):
        raise ValueError(f"mx_linear: output format {out_fmt!r} (None or 'mxfp8')")
    if out_fmt is not None and out_dtype is not None:
        raise ValueError("mx_linear: out_dtype or out_fmt, not both")
    if len(weight.shape) != 2:
        raise ValueError(f"mx_linear: weight must be [n, k], got {weight.shape}")
    n, k = weight.shape
    fmt = weight.fmt
    quantised = isinstance(x, MXTensor)
    if quantised:
        if x.fmt != fmt or x.shape[-1] != k:
            raise ValueError(f"mx_linear: input {x.fmt} {x.shape} does not fit the weight {fmt} {weight.shape}")
        if act_scale is not None:
            raise ValueError("mx_linear: act_scale quantises an unquantised input")
    elif act_scale is not None and fmt != "nvfp4":
        raise ValueError("mx_linear: only nvfp4 has a tensor scale")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if quantised else x.dtype
    if out_dtype not in _OUT_DTYPES:
        raise TypeError(f"mx_linear: output in bf16, fp16 or fp32, got {out_dtype}")
    shape = (*x.shape[:-1], n)
    if weight.codes.is_cuda:
        if quantised:
            out = kernels().mx_linear(None, x.codes, x.scales, x.global_scale, x.rows, weight.codes, weight.scales,
                                       weight.global_scale, _FORMATS[fmt], n, k, bias, _ACTS[act], out_dtype,
                                       out_fmt is not None)
        else:
            out = kernels().mx_linear(x, None, None, act_scale, 0, weight.codes, weight.scales, weight.global_scale,
                                       _FORMATS[fmt], n, k, bias, _ACTS[act], out_dtype, out_fmt is not None)
        if out_fmt is not None:
            return MXTensor(out[0], out[1], out_fmt, shape)
        return out[0] if len(shape) == 2 else out[0].view(shape)
    _check_coded(weight, "mx_linear: weight")
    _check_scalar(weight.global_scale, weight.codes, "mx_linear: weight")
    if x.device != weight.device:
        raise ValueError("mx_linear: input and weight on different devices")
    if bias is not None:
        if bias.device != weight.device or bias.shape != (n,):
            raise ValueError(f"mx_linear: bias must be [{n}] on the weight's device")
        if bias.dtype not in _OUT_DTYPES:
            raise TypeError(f"mx_linear: bias in bf16, fp16 or fp32, got {bias.dtype}")
        _no_grad_here("mx_linear", bias)
    if quantised:
        _check_coded(x, "mx_linear: input")
        _check_scalar(x.global_scale, x.codes, "mx_linear: input")
    else:
        if x.shape[-1] != k:
            raise ValueError(f"mx_linear: input [..., {k}] expected, got {tuple(x.shape)}")
        one = torch.ones(1) if fmt == "nvfp4" else None
        x = mx_quantize(x, fmt, act_scale if act_scale is not None else one)
    y = dequantize_reference(x) @ dequantize_reference(weight).t()
    if bias is not None:
        y = y + bias.float()
    y = F.gelu(y) if _ACTS[act] == 1 else F.relu(y) if _ACTS[act] == 2 else y
    if out_fmt is None:
        return y.to(out_dtype).view(shape)
    return MXTensor(*quantize_reference(y, out_fmt), out_fmt, shape)


def mx_status(device=None) -> int:
    """Non-zero when a product, or a norm's backward, on ``device`` gave up a bounded wait since the last call: outputs
    since then may be invalid.  Nothing else reports it, so a program asks where it waits for results anyway (the call
    waits for all streams of the device; not under graph capture)."""
    dev = torch.device("cuda" if device is None else device)
    return kernels().mx_status(torch.cuda.current_device() if dev.index is None else dev.index)


# ---------------------------------------------------------------- the plain definition
def quantize_reference(x: torch.Tensor, fmt: str, g: Optional[torch.Tensor] = None):
    """fp32 [rows, dim] -> (codes, tiled scales)."""
    size, bits = _BLOCK[fmt], _BITS[fmt]
    rows, dim = x.shape
    nb = -(-dim // size)
    xb = F.pad(x.float(), (0, nb * size - dim)).view(rows, nb, size)
    amax = xb.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    if fmt == "nvfp4":
        g = torch.ones(1, device=x.device) if g is None else g
        s8 = (amax / (6.0 * g)).clamp(max=448.0).to(torch.float8_e4m3fn)
        s = s8.float()
        byte = torch.where(bad, 0x7F, s8.view(torch.uint8).int()).to(torch.uint8)
        inv = torch.where(s > 0, 1.0 / (s * g), torch.zeros_like(s))
    else:
        m, e = torch.frexp(torch.where(bad, torch.zeros_like(amax), amax))
        over = m > (0.75 if bits == 4 else 0.875)
        p = (e - (3 if bits == 4 else 9) + over.int()).clamp(-127, 127)
        p = torch.where(amax > 0, p, torch.full_like(p, -127))
        byte = torch.where(bad, 255, p + 127).to(torch.uint8)
        inv = ((127 - p) << 23).view(torch.float32)
    q = xb * inv[..., None]
    q = torch.where(bad[..., None], torch.zeros_like(q), q).reshape(rows, -1)[:, :dim]
    if bits == 8:
        codes = F.pad(q.clamp(-448, 448), (0, -dim % 16)).to(torch.float8_e4m3fn)
    else:
        mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
        a = q.abs()
        up = torch.bucketize(a, mid, right=True)       # a tie goes up here ...
        down = torch.bucketize(a, mid)                 # ... and down here: take the even code of the two
        code = torch.where(up % 2 == 0, up, down) | (torch.signbit(q).int() << 3)
        code = F.pad(code.to(torch.uint8), (0, -dim % 32))
        codes = code[:, 0::2] | (code[:, 1::2] << 4)
    rt, kt = -(-rows // 128), -(-nb // 4)
    tiled = F.pad(byte, (0, kt * 4 - nb, 0, rt * 128 - rows)).view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4)
    return codes.contiguous(), tiled.contiguous()


def dequantize_reference(t: MXTensor) -> torch.Tensor:
    """fp32 values [rows, dim]."""
    size, bits, rows, dim = _BLOCK[t.fmt], _BITS[t.fmt], t.rows, t.shape[-1]
    if bits == 8:
        q = t.codes[:, :dim].float()
    else:
        grid = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=t.codes.device)
        q = grid[torch.stack((t.codes & 15, t.codes >> 4), -1).view(rows, -1)[:, :dim].long()]
    nb = -(-dim // size)
    rt, kt = t.scales.shape[:2]
    byte = t.scales.permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :nb].contiguous()
    s = byte.view(torch.float8_e4m3fn if t.fmt == "nvfp4" else torch.float8_e8m0fnu).float()
    v = q * s.repeat_interleave(size, 1)[:, :dim]
    return v if t.global_scale is None else v * t.global_scale
