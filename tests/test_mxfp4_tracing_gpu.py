"""GPU: a traced call of the MXFP4 operators and the fused norm gives other inputs their own results; what a functorch transform cannot do is
refused."""

import importlib

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def fns(pkg):
    mx = importlib.import_module("feather_b200.kernel.mxfp4")
    return mx, importlib.import_module("feather_b200.kernel.norm").gated_residual_norm


def _block(mx, norm, b, sb):
    def run(x, gate):
        r, (data, scales) = norm(x, None, packed=True)
        y = mx.scaled_mm_mxfp4(data, scales, b, sb)
        r, h = norm(x, y, gate=gate)
        z = mx.linear_mxfp4(h, b, sb, gate.to(BF16))
        z = mx.dequantize_mxfp4(*mx.quantize_mxfp4(z), torch.float16)
        return norm(r, z, gate=gate, want_norm=False)[0], h

    return run


@pytest.mark.parametrize("how", ["jit", "fx", "fx_pre_dispatch", "fx_symbolic", "compile_eager", "compile_aot_eager"])
def test_traced(fns, cuda_dev, how):
    mx, norm = fns
    g = torch.Generator().manual_seed(1)

    def inputs(rows):
        return torch.randn((rows, 128), generator=g).to(BF16).to(cuda_dev), torch.randn(128, generator=g).to(cuda_dev)

    run = _block(mx, norm, *mx.quantize_mxfp4(torch.randn((128, 128), generator=g).to(cuda_dev)))
    first, second = inputs(70), inputs(70)
    if how == "jit":
        traced = torch.jit.trace(run, first)
    elif how.startswith("compile"):
        torch._dynamo.reset()
        traced = torch.compile(run, backend=how[len("compile_"):], fullgraph=True)
    else:
        traced = make_fx(run, pre_dispatch=how == "fx_pre_dispatch", tracing_mode="symbolic" if how == "fx_symbolic" else "real", _allow_non_fake_inputs=True)(*first)
    for args in (first, second) + ((inputs(9),) if how == "fx_symbolic" or how.startswith("compile") else ()):
        for got, want in zip(traced(*args), run(*args)):
            assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_functorch(fns, cuda_dev):
    mx, norm = fns
    b, sb = mx.quantize_mxfp4(torch.randn((96, 64), device=cuda_dev))
    x = torch.randn((5, 3, 64), device=cuda_dev, dtype=BF16)

    def linear(v):
        return mx.linear_mxfp4(v, b, sb)

    with pytest.raises(RuntimeError, match="no backward"):
        torch.func.grad(lambda v: linear(v).float().sum())(x)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(linear, (x,), (torch.ones_like(x),))
    # rows and samples do not mix, so a mapped call is the call on all of them, where torch maps it at all
    for fn in (linear, lambda v: norm(v, v)[1]):
        try:
            mapped = torch.func.vmap(fn)(x)
        except RuntimeError:
            continue
        assert torch.equal(mapped.view(torch.int16), fn(x).view(torch.int16))
