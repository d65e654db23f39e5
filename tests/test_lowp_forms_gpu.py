"""Forms of the low-precision kernels that sizes and strides select, each against the 64-bit definition: CTA pairs and
slices of the products, every group of threads of the quantised norm."""
import pytest
import torch

from mmltk_b200 import ops

from microscale_oracle import BLOCK, FORMATS, unpack
from test_microscale_gpu import DTYPES, TINY, UNIT, _operands, _product64

pytestmark = pytest.mark.gpu


def _bytes_of(amax, fmt, g=1.0):
    """Scale bytes of blocks with these largest magnitudes (finite, 64-bit)."""
    if fmt == "nvfp4":
        t = (amax.float() / (torch.tensor(6.0) * torch.tensor(g)).item()).clamp(max=448.0)
        return t.to(torch.float8_e4m3fn).view(torch.uint8).long()
    m, e = torch.frexp(amax)
    p = e - (3 if fmt == "mxfp4" else 9) + (m > (0.75 if fmt == "mxfp4" else 0.875)).int()
    return torch.where(amax > 0, p.clamp(-127, 127) + 127, 0).long()


def _check_quantised(t, y, err, g=1.0):
    """Every scale is one that a value within err of y's block maximum has; every element is the nearest one, on the scale
    that was stored, of a value within err of y."""
    fmt, dim = t.fmt, y.shape[1]
    size, nb = BLOCK[fmt], -(-dim // BLOCK[fmt])

    def blocks(v):
        return torch.nn.functional.pad(v, (0, nb * size - dim)).view(len(v), nb, size)
    byte = torch.from_numpy(unpack(t)[1]).to(y.device)
    lo = _bytes_of((blocks(y.abs()) - blocks(err)).clamp(min=0).amax(-1) * (1 - 2.0 ** -22), fmt, g)
    hi = _bytes_of((blocks(y.abs()) + blocks(err)).amax(-1) * (1 + 2.0 ** -22), fmt, g)
    assert ((lo <= byte) & (byte <= hi)).all()
    if fmt == "nvfp4":
        s = byte.to(torch.uint8).view(torch.float8_e4m3fn).double() * g
    else:
        s = torch.exp2(byte.double() - 127)
    s = s.repeat_interleave(size, 1)[:, :dim]
    v = t.dequantize(torch.float32).double()
    top = 448.0 if fmt == "mxfp8" else 6.0
    # half a step: 2^-4 of the value (e4m3), a quarter of it (e2m1), at least half of the smallest step; past the top, the top
    half = torch.maximum(y.abs() * (2.0 ** -4 if fmt == "mxfp8" else 0.25), s * (2.0 ** -10 if fmt == "mxfp8" else 0.25))
    half = torch.maximum(half, y.abs() - top * s)
    assert ((v - y).abs() <= half + 2 * err + 2.0 ** -22 * y.abs()).all()
    assert (v[s == 0] == 0).all()


# ---------------------------------------------------------------- products
# A pair of CTAs takes 256 x 256 tiles where the reduction has 8 stages (2048 4-bit or 1024 8-bit elements) and there
# are as many tiles as SMs: 13 x 14 here, the last rows in the even CTA only, the last column alone in its tile.
# Two slices of a reduction from 24 stages on, for tiles that fill an SM twice but not four times: 10 x 5.
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(3190, 3329, 2100), (3300, 3504, 2048), (3270, 3600, 2333), (1200, 600, 6200),
                                   (1153, 513, 6145)])
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, None), (torch.float16, "gelu"), (torch.float32, "relu")])
def test_pairs_and_slices(cuda_device, fmt, m, n, k, dtype, act):
    x, w, b = _operands(m, n, k, fmt, dtype, seed=21)
    wq = ops.mx_quantize(w.to(cuda_device), fmt)
    xq = ops.mx_quantize(x.to(cuda_device), fmt, torch.ones(1, device=cuda_device) if fmt == "nvfp4" else None)
    xv, wv = xq.dequantize(torch.float32).double(), wq.dequantize(torch.float32).double()
    bd = b.to(cuda_device)
    y, e = _product64(xv, wv, bd.double(), act)
    e = e + 2.0 ** -22 * y.abs()                  # nvfp4 values are rounded once to fp32 above
    for inp in (x.to(cuda_device), xq):
        got = ops.mx_linear(inp, wq, bd, act=act, out_dtype=dtype)
        assert got.dtype == dtype and ((got.double() - y).abs() <= e + UNIT[dtype] * y.abs() + TINY[dtype]).all()
    _check_quantised(ops.mx_linear(xq, wq, bd, act=act, out_fmt="mxfp8"), y, e)
    again = ops.mx_linear(xq, wq, bd, act=act, out_dtype=dtype)
    assert torch.equal(again, got) and ops.mx_status(cuda_device) == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_pairs_keep_non_finite_values_in_place(cuda_device, fmt):
    x, w, _ = _operands(3190, 3329, 2100, fmt, torch.float32, seed=22)
    x[1, 2099], x[3189, 5], w[7, 130], w[3328, 0] = float("nan"), float("inf"), float("nan"), float("-inf")
    y = ops.mx_linear(x.to(cuda_device), ops.mx_quantize(w.to(cuda_device), fmt))
    nan = torch.zeros(3190, 3329, dtype=torch.bool, device=cuda_device)
    nan[[1, 3189]], nan[:, [7, 3328]] = True, True
    assert torch.equal(torch.isnan(y), nan)


# ---------------------------------------------------------------- quantised norm
# Rows of dense tensors whose widths are no multiple of 16 bytes: a warp, then groups of 128, 192, 256, 384, 512 and (fp32)
# 768 threads; and the longest ones.
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dim", [3, 333, 1111, 1537, 2047, 4097, 5001, 8190, 9215, 12287, 16383])
def test_quantised_norm_of_rows_that_start_anywhere(cuda_device, fmt, dtype, residual, dim):
    gen = torch.Generator(device=cuda_device).manual_seed(dim)

    def normal(*shape):
        return torch.randn(*shape, device=cuda_device, generator=gen)
    x, r = (normal(11, dim) * 2).to(dtype), normal(11, dim).to(dtype)
    w = (1 + 0.2 * normal(dim)).to(dtype)
    g = 0.01 if fmt == "nvfp4" and residual else 1.0
    t, h = ops.rms_norm_quantized(x, w, 1e-6, residual=r if residual else None, fmt=fmt,
                                  global_scale=torch.full((1,), g, device=cuda_device) if g != 1.0 else None)
    want = (x.float() + r.float()).to(dtype) if residual else x
    assert torch.equal(h, want)
    hd = h.double()
    y = hd * (hd.square().mean(-1, keepdim=True) + 1e-6) ** -0.5 * w.double()
    # a sum of dim squares in fp32 is off by at most dim 2^-24, its root by half of that; a few more roundings
    _check_quantised(t, y, (dim / 2 + 8) * 2.0 ** -24 * y.abs(), torch.tensor(g).item())
