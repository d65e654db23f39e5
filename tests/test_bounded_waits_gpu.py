"""A bounded wait that runs out: the call returns, the status word says so, and the GPU goes on."""
import os
import subprocess
import sys

import pytest
import torch

from mmltk_b200 import ops
from mmltk_b200.ops import kernels

pytestmark = pytest.mark.gpu


def _linear(m, n, k, fmt, dev, **kw):
    gen = torch.Generator(device=dev).manual_seed(m)
    x = torch.randn(m, k, device=dev, generator=gen).bfloat16()
    w = ops.mx_quantize(torch.randn(n, k, device=dev, generator=gen) * k ** -0.5, fmt)
    return lambda: ops.mx_linear(x, w, **kw)


def _backward(rows, dim, dtype, dev):
    gen = torch.Generator(device=dev).manual_seed(rows)
    x, gy = (torch.randn(rows, dim, device=dev, generator=gen).to(dtype) for _ in range(2))
    w = torch.ones(dim, device=dev, dtype=dtype)

    def run():
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.cat([t.flatten() for t in torch.autograd.grad(ops.rms_norm(xs, ws), [xs, ws], gy)])
    return run


CASES = {
    "few tokens, one slice": lambda d: _linear(3, 200, 200, "mxfp4", d),
    "few tokens, slices": lambda d: _linear(9, 1500, 5000, "nvfp4", d),
    "one tile a CTA": lambda d: _linear(300, 600, 700, "mxfp8", d, act="gelu"),
    "wide tiles, many a CTA": lambda d: _linear(9000, 2000, 520, "nvfp4", d),
    "slices over a cluster": lambda d: _linear(200, 300, 9000, "mxfp4", d, out_fmt="mxfp8"),
    "pairs": lambda d: _linear(3300, 3500, 2600, "mxfp8", d),
    "norm backward": lambda d: _backward(2000, 4096, torch.bfloat16, d),
    "norm backward, rows that start anywhere": lambda d: _backward(2000, 4097, torch.float32, d),
}


@pytest.fixture
def no_wait():
    was = kernels().mx_wait_limit(0)
    yield
    kernels().mx_wait_limit(was)


def _bits(t):
    return t.codes.view(torch.uint8) if isinstance(t, ops.MXTensor) else t


@pytest.mark.parametrize("name", CASES)
def test_a_wait_that_runs_out(cuda_device, name, no_wait):
    run = CASES[name](cuda_device)
    k = kernels()
    k.mx_wait_limit(ops.microscale.WAIT_LIMIT)
    want = _bits(run()).clone()
    assert ops.mx_status(cuda_device) == 0
    for _ in range(3):
        k.mx_wait_limit(0)
        run()                                     # its output is invalid
        assert ops.mx_status(cuda_device) != 0
        assert ops.mx_status(cuda_device) == 0    # the read cleared it
        k.mx_wait_limit(ops.microscale.WAIT_LIMIT)
        assert torch.equal(_bits(run()), want) and ops.mx_status(cuda_device) == 0


FIRST_CALL_CAPTURED = """
import torch
from mmltk_b200 import ops
from mmltk_b200.ops import kernels
x = torch.randn(64, 700, device="cuda").bfloat16()
w = ops.mx_quantize(torch.randn(200, 700, device="cuda"), "mxfp8")
good, bad = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
with torch.cuda.graph(good):                 # the process's first product
    a = ops.mx_linear(x, w)
was = kernels().mx_wait_limit(0)
with torch.cuda.graph(bad):
    b = ops.mx_linear(x, w)
kernels().mx_wait_limit(was)
assert ops.mx_status() == 0                  # nothing has run
bad.replay()
good.replay()                                # does not erase what the other one recorded
assert ops.mx_status() != 0 and ops.mx_status() == 0
want = ops.mx_linear(x, w)
good.replay()
assert torch.equal(a, want) and ops.mx_status() == 0
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
kernels().mx_wait_limit(0)
with torch.cuda.stream(side):
    for _ in range(20):
        big = torch.randn(4096, 4096, device="cuda") @ torch.randn(4096, 4096, device="cuda")
    ops.mx_linear(x, w)
kernels().mx_wait_limit(was)
assert ops.mx_status() != 0                  # of another stream, still running
print("checked")
"""


def test_status_of_a_captured_first_call_and_of_other_streams():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=root, capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and r.stdout.strip() == "checked", r.stdout + r.stderr


def test_wait_limit_is_checked():
    for bad in (-1, 1 << 23):
        with pytest.raises(RuntimeError):
            kernels().mx_wait_limit(bad)
