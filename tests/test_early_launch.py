"""Kernels that start under the end of the one before them wait for it before they touch memory (read from the sources)."""
import glob
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _kernels():
    """(name, body) of every __global__ function of a file that launches kernels early."""
    for path in sorted(glob.glob(os.path.join(ROOT, "csrc", "kernels", "*.cu"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        if "wait_previous" not in text:
            continue
        for m in re.finditer(r"__global__[^;{]*?(\w+_kernel)\(", text):
            start = end = text.index("{", m.end())
            depth = 0
            while True:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
                if depth == 0:
                    break
            yield f"{os.path.basename(path)}:{m.group(1)}", text[start + 1:end - 1]


KERNELS = dict(_kernels())
EARLY = [n for n, b in KERNELS.items() if "allow_next" in b or "wait_previous" in b]


def test_the_early_kernels_are_found():
    assert {"microscale.cu:mx_amax_kernel", "microscale.cu:mx_quantize_kernel", "rmsnorm.cu:rms_fwd_kernel",
            "mx_gemm.cu:mx_gemm_kernel", "mx_few.cu:mx_few_kernel"} <= set(EARLY)


@pytest.mark.parametrize("name", EARLY)
def test_waits_once_before_any_access(name):
    body = KERNELS[name]
    assert body.count("wait_previous();") == 1
    before = body[:body.index("wait_previous();")]
    assert before.count("{") == before.count("}")                      # not in a branch ...
    assert not before.rstrip().endswith((")", "else"))                 # ... nor the statement of one
    # no load and no store of global memory in front of it
    for access in (r"\.load\(", r"\bload_\w+", r"\bld_\w+", r"\bst_\w+", r"\*\s*reinterpret_cast", r"\*\s*static_cast",
                   r"\*g_", r"\bamax\[", r"cp\.async", r"atomic"):
        assert not re.search(access, before), access
