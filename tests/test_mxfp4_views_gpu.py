"""GPU: tensors that carry their sign as a flag (torch's negative bit, as the imaginary part of a conjugate does) are read with it."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_negative_bit(pkg, cuda_dev):
    mx = importlib.import_module("feather_b200.kernel.mxfp4")
    norm = importlib.import_module("feather_b200.kernel.norm").gated_residual_norm
    g = torch.Generator().manual_seed(1)

    def pair(*shape, dtype=BF16):
        t = torch.randn(shape, generator=g).to(dtype).to(cuda_dev)
        flagged = torch._neg_view(t)
        assert flagged.is_neg()
        return flagged, flagged.resolve_neg()

    (x, x_ref), (y, y_ref), (c, c_ref) = pair(70, 128), pair(70, 128), pair(128, dtype=torch.float32)
    odd, odd_ref = pair(9, 33)
    w = mx.quantize_mxfp4(torch.randn((40, 128), generator=g).to(cuda_dev))
    for got, want in (
        (mx.quantize_mxfp4(x)[:1], mx.quantize_mxfp4(x_ref)[:1]),
        ([mx.linear_mxfp4(x, *w)], [mx.linear_mxfp4(x_ref, *w)]),
        (norm(x, y, gate=c, weight=c, bias=c, scale=c, shift=c), norm(x_ref, y_ref, gate=c_ref, weight=c_ref, bias=c_ref, scale=c_ref, shift=c_ref)),
        (norm(odd, odd, post_norm=True), norm(odd_ref, odd_ref, post_norm=True)),
    ):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    z = torch.randn((30, 64), generator=g, dtype=torch.cfloat).to(cuda_dev).conj()
    assert torch.equal(mx.quantize_mxfp4(z.imag)[0], mx.quantize_mxfp4(z.imag.clone().resolve_neg())[0])
    with pytest.raises(RuntimeError, match="resolve_neg"):
        mx.linear_mxfp4(x, *w, pair(40)[0])
    out = torch.empty((70, 40), dtype=BF16, device=cuda_dev)
    with pytest.raises(RuntimeError, match="resolve_neg"):
        importlib.import_module("feather_b200.kernel.b200.native").mxfp4_mm_into(*mx.quantize_mxfp4(x_ref), *w, None, torch._neg_view(out))
