"""CPU: further refusals of the MXFP4 operators and of the fused norm.  As in test_mxfp4_cpu.py, calls that would reach the GPU are made with fake
CUDA tensors: the checks come before the first pointer."""

import importlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("feather_b200.kernel.mxfp4")


@pytest.fixture(scope="module")
def norm(pkg):
    return importlib.import_module("feather_b200.kernel.norm")


def test_product_into_a_given_output(native):
    with FakeTensorMode():
        def u8(*shape, device="cuda"):
            return torch.empty(shape, dtype=torch.uint8, device=device)

        def out(*shape, dtype=BF16, device="cuda"):
            return torch.empty(shape, dtype=dtype, device=device)

        a, sa, b, sb, bias = u8(4, 64), u8(1, 1, 512), u8(200, 64), u8(2, 1, 512), out(200)
        for args, match in (
            ((a, sa, b, sb, None, out(3, 200)), r"out must be \[4, 200\]"),                      # too few rows: would be written past its end
            ((a, sa, b, sb, None, out(4, 199)), r"out must be \[4, 200\]"),
            ((a, sa, b, sb, None, out(4 * 200)), r"out must be \[4, 200\]"),
            ((a, sa, b, sb, None, out(200, 4).t()), "contiguous columns"),
            ((a, sa, b, sb, None, out(1, 200).expand(4, 200)), "rows of out overlap"),
            ((a, sa, b, sb, None, out(4, 200, device="cuda:1")), "same device"),
            ((a, sa, b, sb, None, out(4, 200, device="cpu")), "same device"),
            ((a, sa, b, sb, None, out(4, 200, dtype=torch.float32)), "out_dtype must be"),
            ((a, sa, b, sb, bias, out(4, 200, dtype=torch.float16)), "bias must have the out dtype"),
            ((a, sa, b, sb, bias[:7], out(4, 200)), "N elements"),
            ((a, sa, u8(200, 96), u8(2, 2, 512), None, out(4, 200)), "same K"),
            ((a, sa, b, sa, None, out(4, 200)), "b_scales must be"),
            ((a, u8(1, 4, 128), b, sb, None, out(4, 200)), "a_scales must be"),
            ((u8(64, 4).t(), sa, b, sb, None, out(4, 200)), "contiguous"),
            ((a.float(), sa, b, sb, None, out(4, 200)), "uint8"),
        ):
            with pytest.raises(RuntimeError, match=match):
                native.mxfp4_mm_into(*args)
        with pytest.raises(RuntimeError, match="no backward"):
            native.mxfp4_mm_into(a, sa, b, sb, None, out(4, 200).requires_grad_())


def test_forward_mode_inputs_are_refused(mx, norm):
    """The tangent of a dual tensor would be dropped without a word; gradients being off does not turn forward mode off."""
    import torch.autograd.forward_ad as fwad

    x, bias = torch.ones((4, 64)), torch.ones(64)
    for no_grad in (False, True):
        with fwad.dual_level(), torch.set_grad_enabled(not no_grad):
            dual, dual_bias = fwad.make_dual(x, torch.ones_like(x)), fwad.make_dual(bias, torch.ones_like(bias))
            u8 = torch.zeros((4, 32), dtype=torch.uint8)
            for call in (
                lambda: mx.quantize_mxfp4(dual),
                lambda: mx.linear_mxfp4(dual, u8, u8),
                lambda: mx.linear_mxfp4(x, u8, u8, dual_bias),
                lambda: mx.scaled_mm_mxfp4(u8, u8, u8, u8, dual_bias),
                lambda: norm.gated_residual_norm(dual),
                lambda: norm.gated_residual_norm(x, dual),
                lambda: norm.gated_residual_norm(x, x, gate=dual_bias),
                lambda: norm.gated_residual_norm(x, x, shift=dual_bias),
            ):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
    with fwad.dual_level(), pytest.raises(RuntimeError, match="CUDA"):       # a tensor without a tangent goes on to the other checks
        mx.quantize_mxfp4(x)


def test_flags_that_have_no_truth_value(norm):
    """The error of the flag itself, not one of the interpreter's about an error that was left behind."""
    x = torch.zeros((2, 64))
    for name in ("post_norm", "want_norm", "packed"):
        with pytest.raises(RuntimeError, match="ambiguous"):
            norm.gated_residual_norm(x, **{name: torch.tensor([1, 2])})
    for name in ("residual_scale", "eps"):
        with pytest.raises(TypeError):
            norm.gated_residual_norm(x, **{name: "much"})
