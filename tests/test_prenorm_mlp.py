"""The pre-norm MLP block: training form, and its 8- and 4-bit serving forms."""
import pytest
import torch

from mmltk_b200.models.prenorm_mlp import PreNormMlp, QuantizedPreNormMlp

from microscale_oracle import FORMATS


def _block(dim=96, hidden=160, seed=0):
    torch.manual_seed(seed)
    m = PreNormMlp(dim, hidden)
    with torch.no_grad():
        m.norm_weight.add_(0.1 * torch.randn(dim))
    return m


def _plain(m, x, r):
    h = (x + r).double()
    n = h * (h.square().mean(-1, keepdim=True) + m.eps) ** -0.5 * m.norm_weight.double()
    n = torch.nn.functional.gelu(n @ m.fc1.weight.double().t() + m.fc1.bias.double())
    return n @ m.fc2.weight.double().t() + m.fc2.bias.double(), h


def test_training_form_cpu():
    m = _block()
    x, r = torch.randn(2, 7, 96, requires_grad=True), torch.randn(2, 7, 96)
    y, h = m(x, r)
    y64, h64 = _plain(m, x, r)
    assert (y.double() - y64).abs().max() < 1e-5 * y64.abs().max() and torch.equal(h, x + r)
    (y.sum() + h.sum()).backward()
    assert all(p.grad is not None for p in m.parameters()) and x.grad is not None


@pytest.mark.parametrize("fmt", FORMATS)
def test_serving_form_cpu(fmt):
    m = _block()
    x, r = torch.randn(9, 96), torch.randn(9, 96)
    y, h = m.quantize(fmt)(x, r)
    y64, _ = _plain(m, x, r)
    # three operands rounded in a row, each to half a step at most: 2^-4 of a value (e4m3), 1/4 (e2m1); the sums average
    # the errors out, so the whole stays below one operand's worst case
    assert torch.equal(h, x + r) and (y.double() - y64).norm() < (2.0 ** -4 if fmt == "mxfp8" else 0.25) * y64.norm()
    with pytest.raises(ValueError):
        q = m.quantize(fmt)
        QuantizedPreNormMlp(q.norm_weight, q.w1, q.b1, q.w1, q.b2)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e-5, 1e-2, 1e3])
def test_serving_form_of_small_and_large_activations(fmt, size):
    """Inner activations far below and above one keep the format's precision."""
    m = _block()
    with torch.no_grad():
        m.norm_weight.mul_(size)
        m.fc1.bias.mul_(size)
        m.fc2.bias.zero_()
    x, r = torch.randn(9, 96), torch.randn(9, 96)
    y, _ = m.quantize(fmt)(x, r)
    y64, _ = _plain(m, x, r)
    # as above: three operands' roundings in a row, below one operand's worst case
    assert (y.double() - y64).norm() < (2.0 ** -4 if fmt == "mxfp8" else 0.25) * y64.norm()


@pytest.mark.parametrize("fmt", FORMATS)
def test_serving_form_is_a_copy(fmt):
    m = _block()
    x, r = torch.randn(9, 96), torch.randn(9, 96)
    q = m.quantize(fmt)
    y, h = q(x, r)
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(-3).add_(1)
    y2, h2 = q(x, r)
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_serving_form_gpu(cuda_device, fmt, rows):
    m = _block(384, 1000)
    x, r = torch.randn(rows, 384).bfloat16(), torch.randn(rows, 384).bfloat16()
    with torch.no_grad():
        want, hw = m.quantize(fmt)(x, r)
        got, h = m.to(cuda_device).quantize(fmt)(x.to(cuda_device), r.to(cuda_device))
    # the same roundings but where a sum's last bits decide one: half a step of bf16, twice
    assert torch.equal(h.cpu(), hw) and (got.cpu().double() - want.double()).norm() <= 2.0 ** -7 * want.double().norm()


@pytest.mark.gpu
def test_training_form_gpu(cuda_device):
    m = _block(384, 1536).to(cuda_device, torch.bfloat16)
    x = torch.randn(50, 384, device=cuda_device).bfloat16().requires_grad_()
    r = torch.randn(50, 384, device=cuda_device).bfloat16()
    y, h = m(x, r)
    (y.float().square().sum() + h.float().sum()).backward()
    ref = _block(384, 1536).to(cuda_device).double()
    for a, b in zip(ref.parameters(), m.parameters()):
        a.data.copy_(b.data)
    xd = x.detach().double().requires_grad_()
    yd, hd = _plain(ref, xd, r.double())
    (yd.square().sum() + hd.sum()).backward()
    # five bf16 roundings in the forward and backward chain of a value, 2^-9 each
    for a, b in ((y, yd), (x.grad, xd.grad), (m.norm_weight.grad, ref.norm_weight.grad)):
        assert (a.double() - b).norm() <= 5 * 2.0 ** -8 * b.norm()
