"""GPU: chains of the MXFP4 operators and the fused norm, each of which may start beside the end of the one that writes its operands.  Buffers
are freed and used again from step to step, so a load that came too early, or from a stale line, would see the step before."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _steps(mx, norm, x, weights, gate, rounds, between):
    """A block over and over: packed norm, product, norm of the result with a modulation and a bias made on the way, quantise, dequantise."""
    b, sb, c, sc = weights
    y, outs = None, []
    for i in range(rounds):
        x, (data, scales) = norm(x, y, gate=None if y is None else gate, packed=True)
        between()
        up = mx.scaled_mm_mxfp4(data, scales, b, sb)
        between()
        bias = norm(up[:1], up[-1:], post_norm=True, kind="layer", want_norm=False)[0][0]
        between()
        y = mx.linear_mxfp4(up, c, sc, bias[: c.shape[0]].contiguous())
        between()
        y = mx.dequantize_mxfp4(*mx.quantize_mxfp4(y), BF16)
        between()
        _, y = norm(x, y, gate=y, scale=y[0], shift=y[-1], kind="layer")
        between()
        outs.append((x, y))
        x = x * 0.5                                                         # a kernel of torch in between
    return outs


@pytest.mark.parametrize("tokens", [1, 7, 64, 300, 3000])
@pytest.mark.parametrize("hidden,wide", [(256, 512), (1024, 1280)])
def test_a_chain_gives_what_its_steps_give_alone(pkg, native, cuda_dev, tokens, hidden, wide):
    mx = importlib.import_module("feather_b200.kernel.mxfp4")
    norm = importlib.import_module("feather_b200.kernel.norm").gated_residual_norm
    g = torch.Generator().manual_seed(tokens)

    def t(*shape, scale=1.0):
        return (torch.randn(shape, generator=g) * scale).to(cuda_dev)

    x, gate = t(tokens, hidden).to(BF16), t(hidden, scale=0.3)
    weights = (*mx.quantize_mxfp4(t(wide, hidden, scale=hidden ** -0.5)), *mx.quantize_mxfp4(t(hidden, wide, scale=wide ** -0.5)))
    ref = _steps(mx, norm, x, weights, gate, 6, torch.cuda.synchronize)
    for _ in range(10):
        got = _steps(mx, norm, x, weights, gate, 6, lambda: None)
        torch.cuda.synchronize()
        for a, b in zip(got, ref):
            assert all(torch.equal(p.view(torch.int16), q.view(torch.int16)) for p, q in zip(a, b))
    native.check_device_status(cuda_dev)
    assert torch.isfinite(ref[-1][0]).all()


@pytest.mark.parametrize("rows,cols", [(1, 5120), (4, 1027), (300, 5120), (2000, 512), (3000, 1024)])
def test_operands_rewritten_before_each_call(pkg, cuda_dev, rows, cols):
    """The same buffers hold other values at each call, written by the call before: x, y, and every vector of the norm."""
    norm = importlib.import_module("feather_b200.kernel.norm").gated_residual_norm
    g = torch.Generator().manual_seed(cols)
    a, b = (torch.randn((rows, cols), generator=g).to(BF16).to(cuda_dev) for _ in range(2))

    def run(between):
        x, y, outs = a, b, []
        for i in range(20):
            x, h = norm(x, y, gate=y[0], weight=x[0], bias=x[-1], scale=y[-1], shift=y[0], post_norm=i % 2 == 1, post_weight=x[0] if i % 2 else None, kind=("rms", "layer")[i % 2])
            between()
            x, y = norm(h, None, weight=y[0])[1], h
            between()
            outs.append((x, y))
            outs = outs[-3:]
        return outs

    ref = run(torch.cuda.synchronize)
    for _ in range(10):
        got = run(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(p.view(torch.int16), q.view(torch.int16)) for s, r in zip(got, ref) for p, q in zip(s, r))
