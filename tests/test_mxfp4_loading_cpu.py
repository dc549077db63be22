"""CPU: what the MXFP4 Linear makes of a checkpoint's weight and scale where no kernel is needed."""

import importlib
import importlib.util

import pytest
import torch
import torch.nn.functional as F

FP8 = (torch.float8_e5m2, torch.float8_e4m3fn)


@pytest.fixture(scope="module")
def ops_mod(pkg):
    return importlib.import_module("feather_b200.comfy_feather.ops")


def _linear(ops_mod, k, n, state, excluded=(), out_dtype=torch.bfloat16):
    lin = ops_mod.feather_ops(out_dtype=out_dtype, excluded_names=excluded, weight_format="mxfp4").Linear(k, n, bias=False)
    lin._load_from_state_dict({"blocks.0.ffn." + key: v for key, v in state.items()}, "blocks.0.ffn.", {}, True, [], [], [])
    return lin


@pytest.mark.parametrize("key", ["weight_scale", "scale_weight"])
@pytest.mark.parametrize("dtype", FP8)
@pytest.mark.parametrize("k,excluded", [(48, ()), (16, ()), (64, ("ffn",)), (72, ())])
def test_a_plain_layer_keeps_its_scale(ops_mod, k, excluded, dtype, key):
    """Layers that stay un-quantised (K not a multiple of 32, or excluded by name) hold the values the checkpoint stands for."""
    g = torch.Generator().manual_seed(k)
    codes, scale = torch.randn((40, k), generator=g).to(dtype), torch.tensor(0.3)
    lin = _linear(ops_mod, k, 40, {"weight": codes, key: scale}, excluded)
    want = (codes.float() * scale).to(torch.bfloat16)
    assert not lin.is_quantized and lin.weight.dtype == torch.bfloat16 and torch.equal(lin.weight, want)
    x = torch.randn((3, k), generator=g)
    assert torch.equal(lin(x), F.linear(x, want.float()))


def test_a_plain_layer_without_a_scale_is_left_alone(ops_mod):
    for weight in (torch.randn(40, 48), torch.randn(40, 48).to(torch.float8_e5m2)):
        lin = _linear(ops_mod, 48, 40, {"weight": weight})
        assert lin.weight.dtype == weight.dtype and torch.equal(lin.weight.float(), weight.float())


def _unscaled(monkeypatch, layout):
    """The fp32 weight that would be quantised, instead of quantising it."""
    seen = []

    def quantize(x):
        seen.append(x)
        return torch.zeros((x.shape[0], x.shape[1] // 2), dtype=torch.uint8), torch.zeros((1, 1, 512), dtype=torch.uint8)

    monkeypatch.setattr(layout, "_quantize", quantize)
    return seen


def test_which_axis_a_scale_belongs_to(ops_mod, monkeypatch):
    """One scale, or one for each output row as a column; anything else would be spread along K or over a wrong axis."""
    layout = importlib.import_module("feather_b200.comfy_feather.mxfp4")
    seen = _unscaled(monkeypatch, layout)
    w = torch.randn((64, 64)).to(torch.float8_e4m3fn)
    for scale in (torch.tensor(0.5), torch.tensor([0.5]), torch.rand(64, 1)):
        layout.make_mxfp4_weight(w, scale, torch.bfloat16)
        assert torch.equal(seen.pop(), w.float() * scale.reshape(-1, 1))
    for scale in (torch.rand(64), torch.rand(1, 64), torch.rand(64, 64), torch.rand(64, 2), torch.rand(1, 64, 1)):
        with pytest.raises(ValueError, match="scale"):
            layout.make_mxfp4_weight(w, scale, torch.bfloat16)
        with pytest.raises(ValueError, match="scale"):
            _linear(ops_mod, 64, 64, {"weight": w, "weight_scale": scale}, ("ffn",))
    vector = _linear(ops_mod, 1, 8, {"weight": torch.ones(8).to(torch.float8_e5m2), "weight_scale": torch.tensor([2.0])})
    assert torch.equal(vector.weight, torch.full((8,), 2.0, dtype=torch.bfloat16))


def test_packed_scales_are_e8m0(pkg):
    """Bytes of another format are no exponents: 0x38 is 1.0 as e4m3 and 2^-71 as E8M0."""
    layout = importlib.import_module("feather_b200.comfy_feather.mxfp4")
    mx = importlib.import_module("feather_b200.kernel.mxfp4")
    data, ones = torch.zeros((8, 32), dtype=torch.uint8), torch.ones((8, 2))
    for scale in (torch.full((8, 2), 127, dtype=torch.uint8), ones.to(torch.float8_e8m0fnu)):
        assert layout.make_mxfp4_weight(data, scale, torch.bfloat16)._params.scale.view(-1)[0] == 127
    for dtype in (torch.float8_e4m3fn, torch.float8_e5m2, torch.int8, torch.bool):
        with pytest.raises(ValueError, match="scale bytes"):
            layout.make_mxfp4_weight(data, ones.to(dtype), torch.bfloat16)
        with pytest.raises(RuntimeError, match="bytes"):
            mx.prepack_mxfp4_scales(ones.to(dtype))


def test_a_packed_weight_that_lies_unaligned_is_copied(pkg):
    """A loader may hand out views of one buffer at any offset; the kernels read 16 bytes at a time."""
    layout = importlib.import_module("feather_b200.comfy_feather.mxfp4")
    n, k = 40, 96
    scale = torch.full((n, k // 32), 127, dtype=torch.uint8)
    buffer = torch.randint(0, 256, (n * k // 2 + 64,), generator=torch.Generator().manual_seed(1)).to(torch.uint8)
    first = (-buffer.data_ptr()) % 16
    for offset in range(17):
        view = buffer[first + offset:first + offset + n * k // 2].view(n, k // 2)
        weight = layout.make_mxfp4_weight(view, scale, torch.bfloat16)
        assert weight._qdata.data_ptr() % 16 == 0 and weight._qdata.is_contiguous() and torch.equal(weight._qdata, view)
        assert (weight._qdata.data_ptr() == view.data_ptr()) == (offset % 16 == 0)       # no copy where none is needed


def test_a_torch_without_the_e8m0_type_still_imports(pkg, monkeypatch):
    """The fp8 operators import this module too."""
    mx = importlib.import_module("feather_b200.kernel.mxfp4")
    monkeypatch.delattr(torch, "float8_e8m0fnu")
    spec = importlib.util.spec_from_file_location("feather_b200.kernel.mxfp4_again", mx.__file__)
    source = open(mx.__file__).read().split("# ---", 1)[0]                   # up to the operators, which register once
    space = {"__name__": spec.name, "__package__": "feather_b200.kernel"}
    exec(compile(source, mx.__file__, "exec"), space)
    assert space["SCALE_DTYPES"] == (torch.uint8,)
