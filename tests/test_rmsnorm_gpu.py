"""RMS norm, its residual form and its gradients against the 64-bit formulas."""
import numpy as np
import pytest
import torch

from mmltk_b200 import ops

from microscale_oracle import FORMATS, quantize, unpack

DTYPES = (torch.bfloat16, torch.float16, torch.float32)
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}
EPS = 1e-6
SHAPES = [(1, 1), (1, 64), (3, 7), (9, 128), (5, 111), (130, 384), (17, 1000), (33, 1024), (6, 2048), (11, 1111),
          (3, 4096), (2, 5001), (3, 8192), (2, 16384), (2, 16383), (2500, 96), (1500, 518), (700, 2047), (301, 8190)]


def _inputs(rows, dim, dtype, wdtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    mk = lambda: (torch.randn(rows, dim, generator=gen) * 2).to(dtype)  # noqa: E731
    return mk(), mk(), (1 + 0.2 * torch.randn(dim, generator=gen)).to(wdtype), mk(), mk()


def _formulas(h, w, gy, gh):
    """y, gx, gw in 64 bits, and the magnitudes that their fp32 roundings are relative to."""
    h, w, gy = h.double(), w.double(), gy.double()
    rstd = (h.square().mean(-1, keepdim=True) + EPS) ** -0.5
    xh = h * rstd
    c = (xh * w * gy).mean(-1, keepdim=True)
    gx = rstd * (w * gy - xh * c)
    mag = rstd * ((w * gy).abs() + xh.abs() * (xh * w * gy).abs().mean(-1, keepdim=True))
    if gh is not None:
        gx, mag = gx + gh.double(), mag + gh.double().abs()
    return xh * w, gx, (gy * xh).sum(0), mag, (gy * xh).abs().sum(0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_and_gradients(cuda_device, rows, dim, dtype, residual):
    wdtype = torch.float32 if residual else dtype
    x, r, w, gy, gh = _inputs(rows, dim, dtype, wdtype)
    xd, rd, wd = (t.to(cuda_device).requires_grad_() for t in (x, r, w))
    if residual:
        y, h = ops.add_rms_norm(xd, rd, wd, EPS)
        assert torch.equal(h.detach().cpu(), (x.float() + r.float()).to(dtype))
        g = torch.autograd.grad([y, h], [xd, rd, wd], [gy.to(cuda_device), gh.to(cuda_device)])
        assert torch.equal(g[0], g[1])
        gx, gw = g[0], g[2]
        h = h.detach().cpu()
    else:
        y, h = ops.rms_norm(xd, wd, EPS), x
        gx, gw = torch.autograd.grad(y, [xd, wd], gy.to(cuda_device))
    assert y.dtype == dtype and gx.dtype == dtype and gw.dtype == wdtype
    y64, gx64, gw64, mag, gmag = _formulas(h, w, gy, gh if residual else None)
    # a sum of dim squares in fp32 is off by at most dim 2^-24, its root by half of that; a few more roundings
    u = (dim / 2 + 8) * 2.0 ** -24
    assert ((y.detach().cpu().double() - y64).abs() <= (u + UNIT[dtype]) * y64.abs() + TINY[dtype]).all()
    assert ((gx.cpu().double() - gx64).abs() <= (2.5 * dim + 24) * 2.0 ** -24 * mag + UNIT[dtype] * gx64.abs() + TINY[dtype]).all()
    assert ((gw.cpu().double() - gw64).abs() <= (rows + dim / 2 + 16) * 2.0 ** -24 * gmag + UNIT[wdtype] * gw64.abs() + TINY[wdtype]).all()
    with torch.no_grad():                                     # the same bits without the graph
        again = ops.add_rms_norm(xd, rd, wd, EPS)[0] if residual else ops.rms_norm(xd, wd, EPS)
    assert torch.equal(again, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [48, 333])
def test_gradient_against_differences(cuda_device, dim):
    x, r, w, gy, gh = (t.to(cuda_device) for t in _inputs(6, dim, torch.float32, torch.float32, seed=3))
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = ops.add_rms_norm(*leaves, EPS)
    grads = torch.autograd.grad([y, h], leaves, [gy, gh])
    gen = torch.Generator(device=cuda_device).manual_seed(1)

    def loss(args):
        a, b = ops.add_rms_norm(*args, EPS)
        return (a.double() * gy.double()).sum().item() + (b.double() * gh.double()).sum().item()

    size = (y.double() * gy.double()).abs().sum().item() + (h.double() * gh.double()).abs().sum().item()
    for i in range(3):
        d = torch.randn(leaves[i].shape, device=cuda_device, generator=gen)
        d = d / d.norm()

        def diff(step):
            p, m = ([t if j != i else t + s * step * d for j, t in enumerate((x, r, w))] for s in (1, -1))
            return (loss(p) - loss(m)) / (2 * step)
        step = 2.0 ** -6
        one, two = diff(step), diff(2 * step)
        # the step's error is a third of the change from twice the step; each loss is off by roundings of its terms
        tol = abs(two - one) + (dim / 2 + 16) * 2.0 ** -24 * size / step
        assert abs((grads[i].double() * d.double()).sum().item() - one) <= tol


@pytest.mark.gpu
def test_partial_and_missing_gradients(cuda_device):
    x, r, w, gy, gh = (t.to(cuda_device) for t in _inputs(10, 200, torch.float32, torch.float32))
    xs, rs, ws = (t.clone().requires_grad_() for t in (x, r, w))
    y, h = ops.add_rms_norm(xs, rs, ws, EPS)
    full = torch.autograd.grad([y, h], [xs, rs, ws], [gy, gh], retain_graph=True)
    only_y = torch.autograd.grad(y, [xs, rs, ws], gy, retain_graph=True)
    only_h = torch.autograd.grad(h, [xs, rs], gh, retain_graph=True)
    assert torch.equal(only_h[0], gh) and torch.equal(only_h[1], gh) and torch.equal(only_y[2], full[2])
    assert ((only_y[0] + gh - full[0]).abs() <= 2.0 ** -22 * (full[0].abs() + gh.abs() + only_y[0].abs())).all()
    expanded = torch.autograd.grad(y, xs, gy[:1].expand(10, 200), retain_graph=True)[0]
    assert torch.equal(expanded, torch.autograd.grad(y, xs, gy[:1].repeat(10, 1), retain_graph=True)[0])
    ops.rms_norm(xs, ws.detach(), EPS).backward(gy)          # weight frozen
    ops.rms_norm(x, ws, EPS).backward(gy)                    # input frozen
    assert xs.grad is not None and ws.grad is not None
    with pytest.raises(RuntimeError):
        torch.autograd.grad(ops.rms_norm(xs, ws, EPS).sum(), xs, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim", [(3000, 384), (700, 4096), (5000, 100)])
def test_weight_gradient_repeats_bitwise(cuda_device, rows, dim):
    x, _, w, gy, _ = (t.to(cuda_device) for t in _inputs(rows, dim, torch.bfloat16, torch.float32))
    ws = w.requires_grad_()
    a, b = (torch.autograd.grad(ops.rms_norm(x, ws, EPS), ws, gy)[0] for _ in range(2))
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_extreme_rows(cuda_device):
    x = torch.zeros(6, 256)
    x[1] = 1e-30
    x[2] = 1e18
    x[3, 7] = float("inf")
    x[4, 9] = float("nan")
    x[5, 0] = 3.0
    w = torch.ones(256)
    y = ops.rms_norm(x.to(cuda_device), w.to(cuda_device), EPS).cpu()
    assert (y[0] == 0).all() and torch.isfinite(y[:3]).all() and torch.isnan(y[4]).all()
    assert torch.isnan(y[3, 7]) and (y[3, :7] == 0).all()
    assert torch.allclose(y[2], torch.ones(256), rtol=2.0 ** -20) and torch.allclose(y[1], x[1] * 1e3, rtol=2.0 ** -20)
    assert ops.rms_norm(x[:0].to(cuda_device), w.to(cuda_device)).shape == (0, 256)
    e = x[:0].to(cuda_device).requires_grad_()
    we = w.to(cuda_device).requires_grad_()
    ge, gwe = torch.autograd.grad(ops.rms_norm(e, we).sum(), [e, we])
    assert ge.shape == (0, 256) and (gwe == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_views(cuda_device, dtype):
    x, r, w, _, _ = (t.to(cuda_device) for t in _inputs(60, 96, dtype, dtype))
    x, r = x.view(6, 10, 96), r.view(6, 10, 96)
    for pick in (lambda t: t[:, ::2], lambda t: t[..., 8:72], lambda t: t[..., 3:70], lambda t: t.transpose(0, 1),
                 lambda t: t[:1].expand(4, 10, 96), lambda t: t[..., ::2]):
        a, b = pick(x), pick(r)
        wv = w[:a.shape[-1]]
        for wi in (wv, torch.cat((wv[:1], wv))[1:]):          # the second starts off a 16-byte boundary
            y, h = ops.add_rms_norm(a, b, wi, EPS)
            y2, h2 = ops.add_rms_norm(a.contiguous(), b.contiguous(), wv.clone(), EPS)
            assert y.shape == a.shape and torch.equal(h, h2)
            # scalar and vector loads sum in another order: the root's error, and one step of the type
            assert ((y.double() - y2.double()).abs() <= (2 * UNIT[dtype] + 100 * 2.0 ** -24) * y2.double().abs() + TINY[dtype]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 16), (1, 2048), (5, 111), (140, 384), (3, 1000), (4, 4096), (2, 8192), (2, 16380)])
def test_quantised_norm(cuda_device, fmt, dtype, rows, dim):
    x, r, w, _, _ = _inputs(rows, dim, dtype, dtype)
    t, h = ops.rms_norm_quantized(x.to(cuda_device), w.to(cuda_device), EPS, residual=r.to(cuda_device), fmt=fmt)
    assert torch.equal(h.cpu(), (x.float() + r.float()).to(dtype))
    hd = h.cpu().double()
    y = (hd * (hd.square().mean(-1, keepdim=True) + EPS) ** -0.5 * w.double()).numpy()
    _, byte, val = quantize(y, fmt, 1.0)
    _, s = unpack(t)
    v = t.dequantize(torch.float32).double().cpu().numpy()
    # y is off by u; a scale or an element differs from the definition's only where u reaches across an edge
    u = (dim / 2 + 8) * 2.0 ** -24
    same = (s == byte).repeat(16 if fmt == "nvfp4" else 32, 1)[:, :dim]
    assert same.mean() > 0.99
    step = np.where(same, np.abs(val), np.abs(y))
    lost = np.abs(v - val) > 1e-12
    half = {"mxfp8": 2.0 ** -3, "mxfp4": 0.5, "nvfp4": 0.5}[fmt]       # one element step, relative to the value
    smin = 2.0 ** (byte - 127.0) if fmt != "nvfp4" else None
    assert lost.mean() <= 64 * u + 2.0 / lost.size + (~same).mean()
    if smin is not None:
        smallest = (smin * (2.0 ** -9 if fmt == "mxfp8" else 0.5)).repeat(32, 1)[:, :dim]
        assert (np.abs(v - val) <= half * step + smallest)[same].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(5, 3), (40, 333), (33, 1111), (19, 8191)])
def test_rows_at_different_offsets(cuda_device, dtype, rows, dim):
    """Inputs whose rows are not equally far past a 16-byte boundary."""
    x, r, w, gy, gh = _inputs(rows, dim, dtype, dtype, seed=7)

    def shifted(t, k, pad):
        big = torch.full((rows, dim + pad), float("nan"), dtype=dtype, device=cuda_device)
        big[:, k:k + dim] = t.to(cuda_device)
        return big[:, k:k + dim]
    xd, rd = shifted(x, 1, 5).requires_grad_(), shifted(r, 2, 2).requires_grad_()
    wd = w.to(cuda_device).requires_grad_()
    y, h = ops.add_rms_norm(xd, rd, wd, EPS)
    assert torch.equal(h.detach().cpu(), (x.float() + r.float()).to(dtype))
    gx, _, gw = torch.autograd.grad([y, h], [xd, rd, wd], [shifted(gy, 3, 4), shifted(gh, 0, 1)])
    y64, gx64, gw64, mag, gmag = _formulas(h.detach().cpu(), w, gy, gh)
    u = (dim / 2 + 8) * 2.0 ** -24
    assert ((y.detach().cpu().double() - y64).abs() <= (u + UNIT[dtype]) * y64.abs() + TINY[dtype]).all()
    assert ((gx.cpu().double() - gx64).abs() <= (2.5 * dim + 24) * 2.0 ** -24 * mag + UNIT[dtype] * gx64.abs() + TINY[dtype]).all()
    assert ((gw.cpu().double() - gw64).abs() <= (rows + dim / 2 + 16) * 2.0 ** -24 * gmag + UNIT[dtype] * gw64.abs() + TINY[dtype]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [5, 333, 1111, 4097, 9215])
def test_a_bad_row_leaves_its_neighbours(cuda_device, dtype, dim):
    """NaN and infinity in a row that shares 16-byte granules with the rows around it."""
    x, r, w, gy, gh = (t.to(cuda_device) for t in _inputs(9, dim, dtype, dtype, seed=8))
    good = [0, 1, 2, 4, 5, 7, 8]

    def results(xx, gg):
        xs, rs = xx.clone().requires_grad_(), r.clone().requires_grad_()
        y, h = ops.add_rms_norm(xs, rs, w, EPS)
        g = torch.autograd.grad([y, h], xs, [gg, gh])[0]
        with torch.no_grad():
            t, h8 = ops.rms_norm_quantized(xx, w, residual=r)
            y1 = ops.rms_norm(xx, w, EPS)
        return y, h, g, y1, h8, t.dequantize()
    want = results(x, gy)
    bad, bad_gy = x.clone(), gy.clone()
    bad[3], bad[6] = float("nan"), float("inf")
    bad_gy[3], bad_gy[6] = float("-inf"), float("nan")
    for a, b in zip(results(bad, bad_gy), want):
        assert torch.equal(a[good], b[good]) and not a[3].isfinite().all() and not a[6].isfinite().all()


def test_norm_cpu_definition():
    x, r, w, gy, gh = _inputs(5, 40, torch.float32, torch.float32)
    xs, rs, ws = (t.clone().requires_grad_() for t in (x, r, w))
    y, h = ops.add_rms_norm(xs, rs, ws, EPS)
    y64, gx64, gw64, _, _ = _formulas(h.detach(), w, gy, gh)
    g = torch.autograd.grad([y, h], [xs, rs, ws], [gy, gh])
    for a, b in zip((y, g[0], g[1], g[2]), (y64, gx64, gx64, gw64)):
        assert (a.double() - b).abs().max() <= 64 * 2.0 ** -24 * b.abs().max()
    assert torch.equal(ops.rms_norm(h.detach(), w, EPS), y.detach())
