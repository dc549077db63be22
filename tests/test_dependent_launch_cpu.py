"""CPU: kernels launched with a programmatic dependency run beside the end of the kernel before them, whose results they read.  The
read-only load path (`__ldg`, `ld.global.nc`, and what the compiler makes of `const __restrict__` parameters) is for memory that nobody
writes during a kernel's life, so the sources of such kernels do not use it."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfyui-featherops_b200", "csrc")


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("name", ["mxfp4.cu", "mxfp4.cuh", "mxfp4_mm.cu", "norm.cu", "small_m.cu", "scaled_mm.cu"])
def test_no_read_only_loads(name):
    code = _code(name)
    if name.endswith(".cu"):
        assert ("launch_dependent(" in code or "ProgrammaticStreamSerialization" in code) and "pdl_wait_for_previous_kernel" in code
    assert not re.findall(r"__ldg|\.nc\b|__restrict__", code)
