"""The microscaled formats' plain definition (CPU) against a 64-bit one, their layout, and what the operators refuse."""
import numpy as np
import pytest
import torch

from mmltk_b200 import ops
from mmltk_b200.ops import MXTensor

from microscale_oracle import BLOCK, FORMATS, hard_rows, quantize, tensor_scale, unpack


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [1, 15, 32, 100, 257])
def test_quantize_matches_64_bit_definition(fmt, dim):
    x = hard_rows(dim)
    g = None if fmt != "nvfp4" else torch.tensor([0.037])
    t = ops.mx_quantize(x, fmt, g)
    codes, byte, val = quantize(x.double().numpy(), fmt, None if g is None else g.item())
    c, s = unpack(t)
    np.testing.assert_array_equal(s, byte)
    np.testing.assert_array_equal(np.where(np.isnan(val), 0, c), np.where(np.isnan(val), 0, codes))
    # a value is code x scale (x g): products of few-bit factors, so one fp32 rounding at most (below its normals,
    # half a step of 2^-149; 4 x 2^126, which a number just below 2^128 rounds to, is an infinity in fp32)
    with np.errstate(over="ignore"):
        want = val.astype(np.float32)
    np.testing.assert_allclose(t.dequantize(torch.float32).numpy(), want, rtol=2.0 ** -23, atol=2.0 ** -149)


def test_tensor_scale_is_found():
    x = torch.randn(7, 65, generator=torch.Generator().manual_seed(1))
    assert ops.mx_quantize(x, "nvfp4").global_scale.item() == tensor_scale(x.numpy())
    for bad in (torch.zeros(2, 16), torch.full((2, 16), float("inf"))):
        assert ops.mx_quantize(bad, "nvfp4").global_scale.item() == 1.0


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("std", [1e-4, 1.0, 1e4])
def test_tensor_scale_of_the_finite_values(bad, std):
    x = torch.randn(6, 80, generator=torch.Generator().manual_seed(11)) * std
    x[0, :16] = 0
    want = ops.mx_quantize(x, "nvfp4")
    y = x.clone()
    y[0, 3] = bad
    got = ops.mx_quantize(y, "nvfp4")
    assert got.global_scale.item() == want.global_scale.item() == tensor_scale(x.numpy())
    a, b = want.dequantize(torch.float32), got.dequantize(torch.float32)
    assert torch.isnan(b[0, :16]).all() and torch.equal(a[1:], b[1:]) and torch.equal(a[0, 16:], b[0, 16:])


@pytest.mark.parametrize("g", [1.0, 2.0 ** -20, 3e4])
def test_range_of_a_tensor_scale(g):
    """What the products' and norms' documentation says of block maxima on the grid of a given scale."""
    x = torch.randn(500, 16, generator=torch.Generator().manual_seed(13))
    x = x / x.abs().amax(1, keepdim=True)

    def worst(top):
        v = (x * top * g).float()
        return ((ops.mx_quantize(v, "nvfp4", torch.tensor([g])).dequantize(torch.float32) - v).abs() / (top * g)).max().item()
    # a normal e4m3 scale is off by 1 / 16 at most, an element by half its largest step: 17 / 16 / 6, and fp32's roundings
    assert all(worst(top) <= 17 / 96 + 1e-5 for top in (0.094, 0.1, 0.3, 1.0, 40.0, 2688.0))
    assert worst(0.0175) > 0.25 and worst(0.0058) == 1.0 and worst(4000.0) > 0.32
    v = x * 1e-6 * g      # the scale that is found fits
    assert ((ops.mx_quantize(v, "nvfp4").dequantize(torch.float32) - v).abs() <= (17 / 96 + 1e-5) * 1e-6 * g).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_layout_sizes(fmt):
    t = ops.mx_quantize(torch.randn(2, 65, 130), fmt)
    nb = -(-130 // BLOCK[fmt])
    assert t.shape == (2, 65, 130) and t.rows == 130
    assert t.codes.shape == (130, 144 if fmt == "mxfp8" else 80)
    assert t.scales.shape == (2, -(-nb // 4), 32, 4, 4)
    assert t.dequantize().shape == (2, 65, 130) and t.dequantize().dtype == torch.bfloat16


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("act", [None, "relu", "gelu"])
def test_linear_definition(fmt, act):
    gen = torch.Generator().manual_seed(2)
    x, w, b = torch.randn(3, 5, 70, generator=gen), torch.randn(9, 70, generator=gen), torch.randn(9, generator=gen)
    wq = ops.mx_quantize(w, fmt)
    g = 1.0 if fmt == "nvfp4" else None
    xv = quantize(x.view(-1, 70).double().numpy(), fmt, g)[2]
    wv = wq.dequantize(torch.float32).double()
    y = torch.from_numpy(xv) @ wv.t() + b.double()
    y = {None: lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu}[act](y).view(3, 5, 9)
    got = ops.mx_linear(x, wq, b, act=act)
    assert got.shape == (3, 5, 9) and got.dtype == torch.float32
    # 70 products summed in fp32, none larger than the sum of magnitudes
    bound = 72 * 2.0 ** -24 * (torch.from_numpy(np.abs(xv)) @ wv.abs().t() + b.abs()).max().item()
    assert (got.double() - y).abs().max().item() <= 1.13 * bound      # |gelu'| <= 1.13
    q = ops.mx_linear(x, wq, b, act=act, out_fmt="mxfp8")
    assert isinstance(q, MXTensor) and q.shape == (3, 5, 9)
    again = ops.mx_quantize(got, "mxfp8")
    assert torch.equal(q.codes.view(torch.uint8), again.codes.view(torch.uint8)) and torch.equal(q.scales, again.scales)


def _refusals(dev):
    x = torch.randn(4, 64, device=dev)
    w = ops.mx_quantize(torch.randn(8, 64, device=dev), "mxfp4")
    wn = ops.mx_quantize(torch.randn(8, 64, device=dev), "nvfp4")
    one = torch.ones(1, device=dev)
    calls = [
        lambda: ops.mx_quantize(x, "int4"),
        lambda: ops.mx_quantize(x.double(), "mxfp4"),
        lambda: ops.mx_quantize(x.long(), "mxfp4"),
        lambda: ops.mx_quantize(x[0, 0], "mxfp4"),
        lambda: ops.mx_quantize(x[:, :0], "mxfp4"),
        lambda: ops.mx_quantize(x, "mxfp4", one),
        lambda: ops.mx_quantize(x.clone().requires_grad_(), "mxfp8"),
        lambda: ops.mx_linear(x[:, :32], w),
        lambda: ops.mx_linear(x, w, act="tanh"),
        lambda: ops.mx_linear(x, w, out_fmt="mxfp4"),
        lambda: ops.mx_linear(x, w, out_fmt="mxfp8", out_dtype=torch.bfloat16),
        lambda: ops.mx_linear(x, w, out_dtype=torch.float64),
        lambda: ops.mx_linear(x, w, act_scale=one),
        lambda: ops.mx_linear(wn, wn, act_scale=one),
        lambda: ops.mx_linear(ops.mx_quantize(x, "mxfp8"), w),
        lambda: ops.mx_linear(ops.mx_quantize(x[:, :32], "mxfp4"), w),
        lambda: ops.rms_norm(x, torch.ones(32, device=dev)),
        lambda: ops.rms_norm(x.double(), torch.ones(64, device=dev).double()),
        lambda: ops.rms_norm(x[0, 0], torch.ones(1, device=dev)),
        lambda: ops.add_rms_norm(x, x[:2], torch.ones(64, device=dev)),
        lambda: ops.add_rms_norm(x, x.half(), torch.ones(64, device=dev)),
        lambda: ops.rms_norm_quantized(x.clone().requires_grad_(), torch.ones(64, device=dev)),
        lambda: ops.rms_norm_quantized(x, torch.ones(64, device=dev), fmt="fp4"),
        lambda: ops.rms_norm_quantized(x, torch.ones(64, device=dev), global_scale=one),
    ]
    for i, call in enumerate(calls):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was accepted")


def test_refusals_cpu():
    _refusals("cpu")


@pytest.mark.gpu
def test_refusals_gpu(cuda_device):
    _refusals(cuda_device)
    x = torch.randn(4, 64, device=cuda_device)
    w = ops.mx_quantize(torch.randn(8, 64, device=cuda_device), "mxfp4")
    for call in (
        lambda: ops.rms_norm(torch.zeros(2, 16385, device=cuda_device), torch.ones(16385, device=cuda_device)),
        lambda: ops.rms_norm(x, torch.ones(64)),
        lambda: ops.mx_linear(x.cpu(), w),
        lambda: ops.mx_linear(x, w, torch.ones(8)),
        lambda: ops.mx_linear(x, w, torch.ones(9, device=cuda_device)),
        lambda: ops.mx_linear(x, MXTensor(w.codes[:4], w.scales, "mxfp4", (8, 64))),
        lambda: ops.mx_linear(x, MXTensor(w.codes, w.scales[..., :2], "mxfp4", (8, 64))),
        lambda: ops.mx_linear(x, MXTensor(w.codes.float(), w.scales, "mxfp4", (8, 64))),
        lambda: MXTensor(w.codes, w.scales, "mxfp4", (9, 64)).dequantize(),
        lambda: ops.mx_quantize(x, "nvfp4", torch.ones(1)),
        lambda: ops.mx_quantize(x, "nvfp4", torch.ones(2, device=cuda_device)),
    ):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_a_tensor_scale_belongs_to_nvfp4(fmt):
    # (the plain definition and the product applied one to the other formats too, the kernel that reads values back did not)
    t = ops.mx_quantize(torch.randn(3, 40), fmt)
    with pytest.raises(ValueError, match="only nvfp4"):
        MXTensor(t.codes, t.scales, fmt, t.shape, torch.full((1,), 2.0))


def _more_refusals(dev):
    """What the kernels' wrappers refuse, on any device."""
    x, w = torch.randn(4, 64, device=dev), ops.mx_quantize(torch.randn(8, 64, device=dev), "mxfp4")
    wn = ops.mx_quantize(torch.randn(8, 64, device=dev), "nvfp4")
    ones = torch.ones(64, device=dev)
    two = torch.ones(2, device=dev)
    calls = [
        lambda: ops.mx_linear(x, w, torch.ones(1, device=dev)),
        lambda: ops.mx_linear(x, w, torch.ones(9, device=dev)),
        lambda: ops.mx_linear(x, w, torch.ones(4, 8, device=dev)),
        lambda: ops.mx_linear(x, w, torch.ones(8, device=dev).double()),
        lambda: ops.mx_linear(x, w, torch.ones(8, device=dev, requires_grad=True)),
        lambda: ops.mx_linear(x.clone().requires_grad_(), w),
        lambda: ops.mx_linear(x, wn, act_scale=two),
        lambda: ops.mx_linear(x, wn, act_scale=two[:1].double()),
        lambda: ops.mx_linear(x, MXTensor(w.codes[:4], w.scales, "mxfp4", (8, 64))),
        lambda: ops.mx_linear(x, MXTensor(w.codes, w.scales[..., :2], "mxfp4", (8, 64))),
        lambda: ops.mx_linear(x, MXTensor(w.codes.float(), w.scales, "mxfp4", (8, 64))),
        lambda: ops.mx_linear(x, MXTensor(w.codes, w.scales.int(), "mxfp4", (8, 64))),
        lambda: ops.mx_linear(x, MXTensor(wn.codes, wn.scales, "nvfp4", (8, 64), two)),
        lambda: ops.mx_linear(MXTensor(w.codes[:4], w.scales, "mxfp4", (8, 64)), w),
        lambda: MXTensor(w.codes, w.scales, "mxfp4", (9, 64)).dequantize(),
        lambda: w.dequantize(torch.float64),
        lambda: ops.mx_quantize(x, "nvfp4", two),
        lambda: ops.mx_quantize(x, "nvfp4", two[:1].double()),
        lambda: ops.rms_norm(x, ones.double()),
        lambda: ops.rms_norm(x, ones.bfloat16()),
        lambda: ops.rms_norm(x, ones.long()),
        lambda: ops.rms_norm(x.to(torch.float8_e4m3fn), ones),
        lambda: ops.rms_norm(torch.zeros(2, 16385, device=dev), torch.ones(16385, device=dev)),
        lambda: ops.rms_norm_quantized(x, ones, fmt="nvfp4", global_scale=two),
        lambda: ops.rms_norm_quantized(x, ones.clone().requires_grad_()),
    ]
    for i, call in enumerate(calls):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was accepted")
    with torch.no_grad():
        ops.mx_linear(x, w, torch.ones(8, device=dev, requires_grad=True))


def test_more_refusals_cpu():
    _more_refusals("cpu")


@pytest.mark.gpu
def test_more_refusals_gpu(cuda_device):
    _more_refusals(cuda_device)
    x, w = torch.randn(4, 64), ops.mx_quantize(torch.randn(8, 64), "mxfp4")
    for call in (lambda: ops.mx_linear(x.to(cuda_device), w), lambda: ops.mx_linear(x, w, torch.ones(8, device=cuda_device)),
                 lambda: ops.rms_norm(x, torch.ones(64, device=cuda_device))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()


def test_debug_switch_is_looked_up_at_every_call(monkeypatch):
    from mmltk_b200.ops import _ext

    class Fake:
        def __init__(self, name):
            self.name = name

        def __getattr__(self, op):
            raise LookupError(f"{self.name}.{op}")

    class OnGpu:      # stands for a CUDA tensor, as far as the call looks before it reaches the extension
        is_cuda, shape, dtype = True, (1, 64), torch.float32

        def __getattr__(self, name):
            raise AssertionError(name)
    monkeypatch.setattr(_ext, "_cache", {})
    monkeypatch.setattr(_ext, "_load", lambda name: _ext._cache.setdefault(name, (Fake(name), None)))
    x = OnGpu()
    calls = {"mx_quantize": lambda: ops.mx_quantize(x, "mxfp4"), "rms_norm": lambda: ops.rms_norm(x, x),
             "rms_norm_quantized": lambda: ops.rms_norm_quantized(x, x), "mx_status": lambda: ops.mx_status(torch.device("cuda", 0))}
    for value, name in (("0", "_kernels"), ("1", "_kernels_dbg"), (None, "_kernels"), ("1", "_kernels_dbg")):
        if value is None:
            monkeypatch.delenv("MMLTK_DEBUG_BOUNDS", raising=False)
        else:
            monkeypatch.setenv("MMLTK_DEBUG_BOUNDS", value)
        assert _ext.kernel_module_name() == name
        for op, call in calls.items():
            with pytest.raises(LookupError, match=f"^{name}.{op}$"):
                call()


def test_an_error_message_with_a_number_reaches_python():
    # formatted by the extension itself: needs the process's libstdc++ (it crashed on a private copy)
    c = torch.zeros(2, 16, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="unknown format 9"):
        ops.kernels().mx_dequantize(c, c, None, 9, 2, 16, torch.float32)
