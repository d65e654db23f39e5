"""Tensor memory is never held by a CTA that waits for its cluster while it has to share an SM."""
import os

import pytest
import torch

from mmltk_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_few_tokens_give_tensor_memory_back_before_the_cluster_meets():
    text = open(os.path.join(ROOT, "csrc", "kernels", "mx_few.cu")).read()
    body = text[text.index("mx_few_kernel("):text.index("FewPlan few_plan")]
    assert body.count("tcgen05.alloc") == body.count("tcgen05.dealloc") == 1
    assert body.index("tcgen05.alloc") < body.index("tcgen05.dealloc") < body.index("cluster_sync_all()")


@pytest.mark.gpu
def test_few_tokens_beside_a_16_bit_product(cuda_device):
    """Small products of few tokens in clusters on one stream, pairs of CTAs of a 16-bit product on another: both
    want tensor memory of the same SMs."""
    gen = torch.Generator(device=cuda_device).manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, device=cuda_device, generator=gen).bfloat16()
    x, w = normal(4, 500), ops.mx_quantize(normal(20000, 500), "mxfp4")
    a, b = normal(4000, 1536), normal(1920, 1536)
    with torch.no_grad():
        want = ops.mx_linear(x, w), ops.linear(a, b, None)
        torch.cuda.synchronize()
        one, two = torch.cuda.Stream(), torch.cuda.Stream()
        few, wide = [], []
        for _ in range(50):
            with torch.cuda.stream(one):
                few.append(ops.mx_linear(x, w))
            with torch.cuda.stream(two):
                wide.append(ops.linear(a, b, None))
        torch.cuda.synchronize()
    assert all(torch.equal(t, want[0]) for t in few) and all(torch.equal(t, want[1]) for t in wide)
    assert ops.mx_status(cuda_device) == 0
