"""CPU: the MXFP4 operators and the fused norm under whatever watches torch's dispatcher, with fake CUDA tensors.  Nobody may take the result of
one run for a constant."""

import importlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def block(pkg):
    """Every operator once; a function of x, weights and a modulation."""
    mx = importlib.import_module("feather_b200.kernel.mxfp4")
    norm = importlib.import_module("feather_b200.kernel.norm").gated_residual_norm

    def run(x, b, sb, gate):
        x, (data, scales) = norm(x, None, packed=True)
        y = mx.scaled_mm_mxfp4(data, scales, b, sb)
        x, h = norm(x, y.view(x.shape), gate=gate)
        z = mx.linear_mxfp4(h, b, sb, gate.to(BF16))
        z = mx.dequantize_mxfp4(*mx.quantize_mxfp4(z.view(-1, z.shape[-1])), torch.float16)
        return norm(x, z.view(x.shape), gate=gate, want_norm=False)[0], h

    return run


def _inputs(device="cuda"):
    return (torch.empty((2, 40, 128), dtype=BF16, device=device), torch.empty((128, 64), dtype=torch.uint8, device=device), torch.empty((1, 1, 512), dtype=torch.uint8, device=device),
            torch.empty(128, device=device))


NAMES = {"quantize_mxfp4": 1, "dequantize_mxfp4": 1, "scaled_mm_mxfp4": 1, "linear_mxfp4": 1, "gated_residual_norm": 3}


def _count(targets):
    seen = [t.name().split("::")[1] for t in targets if getattr(t, "namespace", "") == "feather_ops_internal"]
    return {n: seen.count(n) for n in set(seen)}


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_make_fx_sees_every_call(block, mode, pre_dispatch):
    if mode == "real":                                                      # "real" tracing of fake inputs: the fakes are all there is
        with FakeTensorMode():
            graph = make_fx(block, pre_dispatch=pre_dispatch)(*_inputs())
    elif mode == "fake":
        with FakeTensorMode():
            args = _inputs()
        graph = make_fx(block, tracing_mode="fake", pre_dispatch=pre_dispatch)(*args)
    else:                                                                   # sizes that are symbols are not looked at, nor is the device
        graph = make_fx(block, tracing_mode="symbolic", pre_dispatch=pre_dispatch)(*_inputs("cpu"))
    assert _count([n.target for n in graph.graph.nodes if n.op == "call_function"]) == NAMES
    assert not [n for n in graph.graph.nodes if n.op == "get_attr"]          # no result of the traced run in it


def test_fake_tensors_in_eager_calls(block):
    with FakeTensorMode():
        args = _inputs()
        r, h = block(*args)
    assert r.shape == h.shape == (2, 40, 128) and r.dtype == h.dtype == BF16 and r.device.type == "cuda"


def test_a_dispatch_mode_sees_every_call(block):
    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    with FakeTensorMode():
        args = _inputs()
        with Log():
            block(*args)
    assert _count(seen) == NAMES


def test_export(block):
    class Module(torch.nn.Module):
        def forward(self, x, b, sb, gate):
            return block(x, b, sb, gate)

    with FakeTensorMode():
        args = _inputs()
    program = torch.export.export(Module(), args, strict=False)
    assert _count([n.target for n in program.graph.nodes if n.op == "call_function"]) == NAMES


def test_compile_takes_the_whole_block(block):
    """One graph without a break; it is only looked at here, not run."""
    graphs = []

    class Seen(Exception):
        pass

    def backend(gm, example_inputs):
        graphs.append(gm)
        raise Seen

    torch._dynamo.reset()
    with pytest.raises(Exception, match="Seen"):
        torch.compile(block, backend=backend, fullgraph=True)(*_inputs("cpu"))
    assert _count([getattr(n.target, "_opoverload", n.target) for n in graphs[0].graph.nodes if n.op == "call_function"]) == NAMES
    torch._dynamo.reset()
