"""Quantisation, products and quantised norms on the GPU against 64-bit definitions."""
import numpy as np
import pytest
import torch

from mmltk_b200 import ops

from microscale_oracle import FORMATS, hard_rows, quantize, tensor_scale, unpack

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
# one rounding to the type (half a unit of its last place), relative; and half its smallest subnormal
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _same(t, x, fmt, g):
    codes, byte, val = quantize(x.double().numpy(), fmt, g)
    c, s = unpack(t)
    np.testing.assert_array_equal(s, byte)
    ok = ~np.isnan(val)
    np.testing.assert_array_equal(c[ok], codes[ok])
    return val


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 31, 64, 111, 200, 513])
def test_quantize_bits(cuda_device, fmt, dtype, dim):
    x = hard_rows(dim).to(dtype)
    g = None if fmt != "nvfp4" else torch.tensor([0.037])
    t = ops.mx_quantize(x.to(cuda_device), fmt, None if g is None else g.to(cuda_device))
    val = _same(t, x, fmt, None if g is None else g.item())
    for out in DTYPES:
        got = t.dequantize(out).double().cpu().numpy()
        fin = np.abs(val) < torch.finfo(out).max
        # q s g: at most one fp32 rounding before the stored type's
        np.testing.assert_allclose(got[fin], val[fin], rtol=UNIT[out] + 2.0 ** -23, atol=TINY[out] * 2)
        assert np.isnan(got[np.isnan(val)]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 40), (129, 100), (260, 1000), (1000, 24)])
def test_tensor_scale(cuda_device, dtype, rows, dim):
    x = (torch.randn(rows, dim, generator=torch.Generator().manual_seed(3)) * 5).to(dtype)
    t = ops.mx_quantize(x.to(cuda_device), "nvfp4")
    g = tensor_scale(x.float().numpy())
    assert t.global_scale.item() == g
    _same(t, x, "nvfp4", g)
    for bad in (torch.zeros_like(x), torch.full_like(x, float("inf"))):
        assert ops.mx_quantize(bad.to(cuda_device), "nvfp4").global_scale.item() == 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(3, 40), (129, 101), (260, 1000), (1300, 8192)])
def test_tensor_scale_of_the_finite_values(cuda_device, dtype, rows, dim):
    """One infinity and one NaN: their blocks are NaN, every other block as without them."""
    gen = torch.Generator(device=cuda_device).manual_seed(12)
    x = (torch.randn(rows, dim, device=cuda_device, generator=gen) * 1e-3).to(dtype)
    x[rows // 2, :16] = 0
    x[rows - 1, 16:32] = 0
    bad = x.clone()
    bad[rows // 2, 5], bad[rows - 1, 16] = float("inf"), float("nan")
    want, got = ops.mx_quantize(x, "nvfp4"), ops.mx_quantize(bad, "nvfp4")
    g = (x.float().abs().max().cpu() * (1.0 / 2688.0)).clamp(min=2.0 ** -100)
    assert got.global_scale.item() == want.global_scale.item() == g.item()
    a, b = want.dequantize(torch.float32), got.dequantize(torch.float32)
    a[rows // 2, :16] = a[rows - 1, 16:32] = float("nan")
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())
    wide = torch.full((rows, dim + 3), float("nan"), dtype=dtype, device=cuda_device)      # rows of a view
    wide[:, 1:1 + dim] = bad
    assert ops.mx_quantize(wide[:, 1:1 + dim], "nvfp4").global_scale.item() == g.item()


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_views_and_empty(cuda_device, fmt):
    x = torch.randn(6, 70, 96, generator=torch.Generator().manual_seed(4)).bfloat16().to(cuda_device)
    g = torch.ones(1, device=cuda_device) if fmt == "nvfp4" else None
    for v in (x[:, ::2], x[..., 8:72], x[..., 3:70], x.transpose(0, 1), x.transpose(1, 2), x[:1].expand(3, 70, 96),
              x[:, :, ::2], x.flatten()[5:5 + 64].view(2, 32)):
        t = ops.mx_quantize(v, fmt, g)
        assert t.shape == tuple(v.shape)
        _same(t, v.cpu().reshape(-1, v.shape[-1]), fmt, 1.0)
    e = ops.mx_quantize(x[:0], fmt, g)
    assert e.dequantize().shape == (0, 70, 96)
    assert ops.mx_linear(x[:0], ops.mx_quantize(x[0], fmt)).shape == (0, 70, 70)


# ---------------------------------------------------------------- products
def _operands(m, n, k, fmt, dtype, seed=5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(m, k, generator=gen) * (1 + 9 * (torch.rand(k, generator=gen) < 0.05))).to(dtype)
    w = torch.randn(n, k, generator=gen) * k ** -0.5
    return x, w, torch.randn(n, generator=gen).to(dtype)


def _product64(xv, wv, b, act):
    """(y, bound of the fp32 accumulation): each of the k + 2 additions is off by at most 2^-23 of the sum of
    magnitudes (a tensor core may truncate); |gelu'| <= 1.13, and its erf is good to 1.5e-7."""
    y = xv @ wv.t() + b
    mag = xv.abs() @ wv.abs().t() + b.abs()
    e = (xv.shape[1] + 2) * 2.0 ** -23 * mag
    if act == "relu":
        return y.clamp(min=0), e
    if act == "gelu":
        z = torch.nn.functional.gelu(y)
        return z, 1.13 * e + 2e-7 * y.abs() + 2.0 ** -23 * z.abs()
    return y, e


SIZES = [(1, 1, 1), (1, 64, 64), (2, 130, 32), (7, 128, 111), (17, 2050, 100), (33, 96, 257), (64, 300, 512),
         (65, 129, 300), (128, 128, 1024), (200, 520, 384), (300, 256, 2000), (2500, 1300, 200),
         (70, 200, 6200), (300, 131, 6500), (40, 1000, 9000)]      # the last three: reductions in slices


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, None), (torch.float16, "gelu"), (torch.float32, "relu")])
def test_linear(cuda_device, fmt, m, n, k, dtype, act):
    x, w, b = _operands(m, n, k, fmt, dtype)
    wq = ops.mx_quantize(w.to(cuda_device), fmt)
    one = torch.ones(1, device=cuda_device) if fmt == "nvfp4" else None
    xq = ops.mx_quantize(x.to(cuda_device), fmt, one)      # checked bit by bit above
    xv, wv = xq.dequantize(torch.float32).double(), wq.dequantize(torch.float32).double()
    bd = b.to(cuda_device)
    y, e = _product64(xv, wv, bd.double(), act)
    for inp in (x.to(cuda_device), xq):
        got = ops.mx_linear(inp, wq, bd, act=act, out_dtype=dtype)
        assert got.dtype == dtype and got.is_contiguous()
        # nvfp4 values are rounded once to fp32 above (the factor g)
        assert ((got.double() - y).abs() <= e + (UNIT[dtype] + 2.0 ** -22) * y.abs() + TINY[dtype]).all()
        # 8-bit output: where the scales agree, within half a step of the element type (2^-4 of the value, or half
        # of the smallest step 2^-9 s); they may differ only where the block maximum is within e of an edge
        t = ops.mx_linear(inp, wq, bd, act=act, out_fmt="mxfp8")
        unpack(t)                                           # zero padding
        v = t.dequantize(torch.float32).double()
        _, byte, _ = quantize(y.cpu().numpy(), "mxfp8")
        mine = unpack(t)[1]
        differ = np.abs(mine - byte)
        s = torch.from_numpy(2.0 ** (np.maximum(mine, byte) - 127.0)).to(cuda_device).repeat_interleave(32, 1)[:, :n]
        assert ((v - y).abs() <= e + 2.0 ** -4 * (y.abs() + e) + 2.0 ** -10 * s).all()
        blocks = torch.nn.functional.pad(y.abs(), (0, -n % 32)).view(m, -1, 32).amax(-1).cpu().numpy()
        emax = torch.nn.functional.pad(e, (0, -n % 32)).view(m, -1, 32).amax(-1).cpu().numpy()
        edge = 448.0 * 2.0 ** (np.minimum(mine, byte) - 127.0)
        assert ((differ == 0) | ((differ == 1) & (np.abs(blocks - edge) <= emax + 2.0 ** -22 * edge))).all()
    assert ops.mx_status(cuda_device) == 0


@pytest.mark.parametrize("sx,sw", [(1e30, 1e20), (1e-25, 1e-10), (1e-18, 1e-18), (1e-6, 1e-27), (1e30, 1e-30)])
@pytest.mark.parametrize("m,n,k", [(3, 40, 64), (40, 300, 200), (70, 200, 6200), (2500, 1300, 200)])
def test_tensor_scales_far_apart_from_one(cuda_device, sx, sw, m, n, k):
    """Two scales whose product is no normal fp32 number, but the product of a sum and both is."""
    x, w, _ = _operands(m, n, k, "nvfp4", torch.float32, seed=15)
    x, w = x * sx, w * sw
    x[1] = 0
    w[5] = w[5] * 2.0 ** -12
    xq, wq = (ops.mx_quantize(t.to(cuda_device), "nvfp4") for t in (x, w))
    xv, wv = xq.dequantize(torch.float32).double(), wq.dequantize(torch.float32).double()
    b = torch.zeros(n, device=cuda_device)
    y, e = _product64(xv, wv, b.double(), None)
    got = ops.mx_linear(xq, wq, b, out_dtype=torch.float32).double()
    fits = y.abs() < torch.finfo(torch.float32).max / 2
    assert fits[1].all() and fits[:, 5].all() == (sx * sw < 1e40)
    # nvfp4 values are rounded once to fp32 above; half the smallest subnormal
    assert ((got - y).abs() <= e + 2.0 ** -22 * y.abs() + 2.0 ** -149)[fits].all() and (got[1] == 0).all()
    assert torch.isinf(got[y.abs() > e + 2.0 * torch.finfo(torch.float32).max]).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 5, 48, 150, 600])
def test_linear_without_bias_repeats_bitwise(cuda_device, fmt, m):
    x, w, _ = _operands(m, 384, 3000, fmt, torch.bfloat16)
    wq = ops.mx_quantize(w.to(cuda_device), fmt)
    xd = x.to(cuda_device)
    a, b = ops.mx_linear(xd, wq), ops.mx_linear(xd, wq)
    assert torch.equal(a, b)
    # a token's result does not depend on what else is in the batch of the same kernel
    for i in {0, m - 1}:
        c = ops.mx_linear(xd[i:i + 1].expand(m, -1), wq)
        assert torch.equal(c[0], c[-1]) and torch.equal(c[0], a[i])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [3, 200])
def test_non_finite_values_stay_in_their_row_and_column(cuda_device, fmt, m):
    x, w, _ = _operands(m, 260, 300, fmt, torch.float32)
    x[1, 299], x[2, 5], w[7, 130] = float("nan"), float("inf"), float("nan")
    wq = ops.mx_quantize(w.to(cuda_device), fmt, torch.full((1,), 0.01, device=cuda_device) if fmt == "nvfp4" else None)
    y = ops.mx_linear(x.to(cuda_device), wq)
    nan = torch.zeros(m, 260, dtype=torch.bool, device=cuda_device)
    nan[1:3], nan[:, 7] = True, True
    assert torch.equal(torch.isnan(y), nan)
    t = ops.mx_linear(x.to(cuda_device), wq, out_fmt="mxfp8").dequantize()
    assert torch.isnan(t[1:3]).all() and torch.isnan(t[0, :32]).all() and torch.isfinite(t[0, 32:]).all()


@pytest.mark.parametrize("m", [4, 300])
def test_linear_strides_streams_and_graph(cuda_device, m):
    x, w, b = _operands(m, 500, 640, "mxfp8", torch.bfloat16)
    wq = ops.mx_quantize(w.to(cuda_device), "mxfp8")
    bd, xd = b.to(cuda_device), x.to(cuda_device)
    want = ops.mx_linear(xd, wq, bd)
    wide = torch.zeros(m, 700, dtype=torch.bfloat16, device=cuda_device)
    for off in (0, 3, 8):
        wide[:, off:off + 640] = xd
        assert torch.equal(ops.mx_linear(wide[:, off:off + 640], wq, bd), want)
    assert torch.equal(ops.mx_linear(xd.t().contiguous().t(), wq, bd), want)
    assert torch.equal(ops.mx_linear(xd, wq, bd[None].expand(2, -1).t()[:, 0]), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.mx_linear(xd, wq, bd)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    buf = torch.zeros_like(xd)
    with torch.cuda.graph(graph):
        out = ops.mx_linear(buf, wq, bd)
    buf.copy_(xd)
    graph.replay()
    assert torch.equal(out, want)


def test_offsets_past_32_bits(cuda_device):
    rows, dim = 70000, 32768                     # 2.3e9 elements
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device=cuda_device)
    x.copy_(torch.randn(1, dim, device=cuda_device))
    x[-300:] = torch.randn(300, dim, device=cuda_device)
    t = ops.mx_quantize(x, "mxfp4")
    tail = ops.mx_quantize(x[-112:], "mxfp4")     # 70000 = 546 * 128 + 112: the last scale tile's rows
    assert torch.equal(t.codes[-112:], tail.codes) and torch.equal(t.scales[-1], tail.scales[0])
    d = t.dequantize()
    assert torch.equal(d[-112:], tail.dequantize())
    del x, d
    w = ops.mx_quantize(torch.randn(dim, 64, device=cuda_device), "mxfp4")
    a = torch.randn(rows, 64, device=cuda_device).bfloat16()
    y = ops.mx_linear(a, w)
    assert torch.equal(y[-112:], ops.mx_linear(a[-240:], w)[-112:])


# ---------------------------------------------------------------- the pre-norm MLP in low precision
@pytest.mark.parametrize("rows", [1, 40, 333])
def test_norm_feeds_the_product(cuda_device, rows):
    gen = torch.Generator().manual_seed(8)
    x, r = (torch.randn(rows, 384, generator=gen).bfloat16().to(cuda_device) for _ in range(2))
    w = (1 + 0.1 * torch.randn(384, generator=gen)).bfloat16().to(cuda_device)
    w1 = ops.mx_quantize(torch.randn(200, 384, generator=gen).to(cuda_device) * 0.05, "mxfp8")
    t, h = ops.rms_norm_quantized(x, w, residual=r)
    assert torch.equal(h, ops.add_rms_norm(x, r, w)[1])
    got = ops.mx_linear(t, w1)
    assert torch.equal(got, ops.mx_linear(t.dequantize(torch.float32), w1, out_dtype=torch.bfloat16))
