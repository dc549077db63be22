"""GPU: a norm whose wait for a row runs out.  The limit is set to zero for a process of its own, so a row that has not arrived at the first look
counts as lost: the call reports it, what it stores of such a row is NaN and never anything that was not read, and the context stays usable."""

import importlib
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# rows, cols, has y, coefficients, norm of y, what is asked for
CASES = [(3000, 5120, True, False, False, "rh"), (3000, 5120, True, True, False, "rh"), (3000, 5120, True, False, True, "rh"), (3000, 5120, True, True, True, "r"),
         (3000, 5120, False, False, False, "h"), (20000, 64, True, False, False, "rh"), (20000, 256, True, True, True, "rh"), (9000, 512, True, False, True, "rh"),
         (2000, 16384, True, True, True, "rh"), (3000, 8192, True, True, False, "packed")]

SCRIPT = """
import ctypes, importlib, sys
sys.path.insert(0, %r)
import torch, __graft_entry__
__graft_entry__.load_package()
native = importlib.import_module("feather_b200.kernel.b200.native")
from tests.test_norm_wait_gpu import CASES, call
status = torch.zeros(1, dtype=torch.int32, device="cuda")
seen = []
for case in CASES:
    outs = call(native, case, status)
    torch.cuda.synchronize()
    seen.append((int(status.item()), [o.cpu() for o in outs]))
    status.zero_()
torch.save(seen, sys.argv[1])
few = call(native, (100, 512, True, True, True, "rh"), status)              # the form for few rows has no such wait
torch.cuda.synchronize()
assert int(status.item()) == 0 and all((o != 7).any() for o in few)
"""


def call(native, case, status):
    """The C entry with outputs that are full of sevens beforehand."""
    import ctypes

    rows, cols, has_y, coefficients, post, want = case
    g = torch.Generator(device="cuda").manual_seed(cols)

    def t(*shape, dtype=torch.bfloat16):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    x, y = t(rows, cols), t(rows, cols)
    gate, shift = t(cols, dtype=torch.float32), t(cols, dtype=torch.float32)
    r, h = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    a = native.NormArgs(x=x.data_ptr(), rows=rows, cols=cols, ldx=cols, ldy=cols, ldr=cols, ldh=cols, residual_scale=1.0, eps=1e-6, post_norm=int(post), x_dtype=1, y_dtype=1, h_dtype=1,
                        status_dev=status.data_ptr())
    outs = []
    if has_y:
        a.y = y.data_ptr()
        if "r" in want:
            a.r = r.data_ptr()
            outs.append(r)
    if want == "packed":
        h = torch.full((rows, cols // 2), 7, dtype=torch.uint8, device="cuda")
        scales = torch.full(((rows + 127) // 128 * ((cols + 127) // 128) * 512,), 7, dtype=torch.uint8, device="cuda")
        a.h_scales = scales.data_ptr()
        outs.append(scales)
    if want != "r":
        a.h = h.data_ptr()
        outs.append(h)
    if coefficients and has_y:
        a.gate, a.gate_rows, a.gate_ld = gate.data_ptr(), rows, cols
    if coefficients and want != "r":
        a.shift, a.shift_rows, a.shift_ld = shift.data_ptr(), rows, cols
    torch.cuda.synchronize()
    assert native.load_library().feather_gated_norm(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    return outs


@pytest.mark.parametrize("limit", ["", "soon", "5 s", "-1", "99999999999999999999"])
def test_a_limit_that_is_no_shorter_number_is_the_default(pkg, native, cuda_dev, tmp_path, limit):
    script, out = tmp_path / "wait.py", tmp_path / "seen.pt"
    script.write_text(SCRIPT % ROOT)
    res = subprocess.run([sys.executable, str(script), str(out)], env={**os.environ, "FEATHER_NORM_WAIT_NS": limit}, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=180, cwd=ROOT)
    assert res.returncode == 0, res.stdout[-3000:]
    assert all(code == 0 for code, _ in torch.load(out))


def test_a_wait_that_runs_out(pkg, native, cuda_dev, tmp_path):
    script, out = tmp_path / "wait.py", tmp_path / "seen.pt"
    script.write_text(SCRIPT % ROOT)
    res = subprocess.run([sys.executable, str(script), str(out)], env={**os.environ, "FEATHER_NORM_WAIT_NS": "0"}, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=180, cwd=ROOT)
    assert res.returncode == 0, res.stdout[-3000:]
    status = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    for case, (code, outs) in zip(CASES, torch.load(out)):
        ref = call(native, case, status)
        torch.cuda.synchronize()
        assert int(status.item()) == 0
        assert code == 0 or code & 0xFF == native.FEATHER_ERR_DEVICE_TIMEOUT, (case, code)
        _, cols, _, coefficients, _, _ = case
        missing = 0
        for got, want in zip(outs, (o.cpu() for o in ref)):
            # untouched or NaN (an MXFP4 block: scale code 255, zero elements)
            lost = (got == 7) | (torch.isnan(got) if got.is_floating_point() else (got == 255) | (got == 0))
            assert (lost | (got == want)).all(), case
            missing += int((lost & (want != got)).sum())
        assert (missing > 0) == (code != 0), case
        # Where nothing lies between the copies and the look (the other warps of a wide group do not issue any, tens of cycles against the hundreds
        # that a copy takes) rows are lost for certain.  A group of one warp (up to 512 columns) issues its ring first, and a block with
        # coefficients folds them first: that takes about as long as a copy, and either may be.
        assert code != 0 or coefficients or cols <= 512, case
