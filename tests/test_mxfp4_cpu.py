"""CPU: refusals of the MXFP4 operators and of the fused norm, the scale layout, and the C entry points' argument checks.  Calls
that would reach the GPU are made with fake CUDA tensors (shapes and types, no memory): every check comes before the first pointer."""

import ctypes
import importlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tests import mx_ref


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("feather_b200.kernel.mxfp4")


@pytest.fixture(scope="module")
def norm(pkg):
    return importlib.import_module("feather_b200.kernel.norm")


def test_reference_quantiser_by_hand():
    """The 64-bit form of the tests against values worked out by hand."""
    x = torch.zeros((1, 64))
    x[0, :8] = torch.tensor([4.0, 0.25, 0.75, 1.25, 2.5, 3.5, -5.0, 7.9])
    x[0, 32:36] = torch.tensor([1.0, 0.0625, -0.1875, 0.25])
    codes, scales = mx_ref.quantize(x)
    assert scales.tolist() == [[127, 125]]
    assert codes[0, :8].tolist() == [6, 0, 2, 2, 4, 6, 8 + 6, 7]
    assert codes[0, 32:36].tolist() == [6, 0, 8 + 2, 2]
    v = mx_ref.values(codes, scales)
    assert v[0, :8].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 4.0, -4.0, 6.0] and v[0, 32:36].tolist() == [1.0, 0.0, -0.25, 0.25]
    assert torch.equal(mx_ref.unpack(mx_ref.pack(codes)), codes)


@pytest.mark.parametrize("rows,blocks", [(1, 1), (3, 4), (127, 5), (128, 8), (300, 33)])
def test_scale_tiles(mx, rows, blocks):
    plain = torch.randint(0, 256, (rows, blocks), generator=torch.Generator().manual_seed(rows)).to(torch.uint8)
    tiles = mx.prepack_mxfp4_scales(plain)
    assert tuple(tiles.shape) == ((rows + 127) // 128, (blocks + 3) // 4, 512)
    for r, b in {(0, 0), (rows - 1, blocks - 1), (rows // 2, blocks // 3), (min(rows - 1, 70), blocks // 2)}:
        assert tiles[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4] == plain[r, b]
    assert torch.equal(mx.unprepack_mxfp4_scales(tiles, rows, blocks * 32), plain)
    assert int(tiles.sum(dtype=torch.int64)) == int(plain.sum(dtype=torch.int64))      # the padding is zero


def test_scale_bytes(native):
    lib = native.load_library()
    for rows, k in ((1, 32), (128, 128), (129, 160), (5120, 13824)):
        assert lib.feather_mxfp4_scale_bytes(rows, k) == (rows + 127) // 128 * ((k + 127) // 128) * 512
    assert lib.feather_mxfp4_scale_bytes(0, 32) == 0


def test_mxfp4_refusals(mx):
    with pytest.raises(RuntimeError, match="CUDA"):
        mx.quantize_mxfp4(torch.zeros((2, 64)))
    with pytest.raises(RuntimeError, match="CUDA"):
        mx.dequantize_mxfp4(torch.zeros((2, 32), dtype=torch.uint8), torch.zeros((1, 1, 512), dtype=torch.uint8), torch.float32)
    with pytest.raises(RuntimeError, match="tiles of"):
        mx.unprepack_mxfp4_scales(torch.zeros((1, 1, 512), dtype=torch.uint8), 200, 128)
    with pytest.raises(RuntimeError, match="bytes"):
        mx.prepack_mxfp4_scales(torch.zeros((4, 4)))
    with FakeTensorMode():
        def u8(*shape, device="cuda"):
            return torch.empty(shape, dtype=torch.uint8, device=device)

        x = torch.empty((4, 64), device="cuda")
        for bad, match in ((torch.empty((4, 48), device="cuda"), "multiple of 32"), (torch.empty((64,), device="cuda"), "2D"), (torch.empty((4, 0), device="cuda"), "multiple of 32"),
                           (torch.empty((4, 64), dtype=torch.float64, device="cuda"), "cannot quantise"), (u8(4, 64), "cannot quantise")):
            with pytest.raises(RuntimeError, match=match):
                mx.quantize_mxfp4(bad)
        x.requires_grad_()
        with pytest.raises(RuntimeError, match="no backward"):
            mx.quantize_mxfp4(x)
        with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
            mx.dequantize_mxfp4(u8(4, 32), u8(1, 1, 512), torch.int8)
        a, sa, b, sb = u8(4, 64), u8(1, 1, 512), u8(200, 64), u8(2, 1, 512)
        bias = torch.empty((200,), dtype=torch.bfloat16, device="cuda")
        for args, match in (
            ((a, sa, b, sb, None, torch.float32), "out_dtype"),
            ((a, sa, b, sb, bias, torch.float16), "bias must have the out dtype"),
            ((a, sa, b, sb, bias[:100], torch.bfloat16), "N elements"),
            ((a, sa, b, sa, None, torch.bfloat16), "b_scales must be"),
            ((a, u8(1, 4, 128), b, sb, None, torch.bfloat16), "a_scales must be"),
            ((a, sa, u8(200, 96), sb.view(2, 1, 512).repeat(1, 2, 1), None, torch.bfloat16), "same K"),
            ((u8(4, 24), sa, b, sb, None, torch.bfloat16), "multiple of 32"),
            ((a.float(), sa, b, sb, None, torch.bfloat16), "uint8"),
            ((u8(64, 4).t(), sa, b, sb, None, torch.bfloat16), "contiguous"),
            ((u8(4, 64, device="cpu"), sa, b, sb, None, torch.bfloat16), "CUDA tensors"),
            ((a, sa, u8(200, 64, device="cuda:1"), u8(2, 1, 512, device="cuda:1"), None, torch.bfloat16), "same device"),
            ((a, sa, u8(0, 64), u8(0, 1, 512), None, torch.bfloat16), "at least one row"),
        ):
            with pytest.raises(RuntimeError, match=match):
                mx.scaled_mm_mxfp4(*args)
        with pytest.raises(RuntimeError, match="no backward"):
            mx.scaled_mm_mxfp4(a, sa, b, sb, torch.empty((200,), dtype=torch.bfloat16, device="cuda", requires_grad=True))
        with pytest.raises(RuntimeError, match="dimension"):
            mx.linear_mxfp4(torch.empty((), device="cuda"), b, sb)


def test_norm_refusals(norm):
    f = norm.gated_residual_norm
    with pytest.raises(RuntimeError, match="CUDA"):
        f(torch.zeros((2, 64)))
    with FakeTensorMode():
        def t(*shape, dtype=torch.bfloat16, device="cuda"):
            return torch.empty(shape, dtype=dtype, device=device)

        x, y, c = t(2, 8, 64), t(2, 8, 64), t(64)
        for args, kw, match in (
            ((x.double(),), {}, "x must be"),
            ((x, y.double()), {}, "y must be"),
            ((x, t(2, 8, 32)), {}, "x's shape"),
            ((x, t(2, 8, 64, device="cuda:1")), {}, "same device"),
            ((x, y), {"kind": "batch"}, "kind"),
            ((x, y), {"eps": -1.0}, "eps"),
            ((x, y), {"eps": float("nan")}, "eps"),
            ((x,), {"gate": c}, "need y"),
            ((x,), {"post_norm": True}, "need y"),
            ((x,), {"want_norm": False}, "only the norm"),
            ((x, y), {"post_weight": c}, "needs post_norm"),
            ((x, y), {"want_norm": False, "weight": c}, "leaves out"),
            ((x, y), {"want_norm": False, "packed": True}, "leaves out"),
            ((x, y), {"weight": t(32)}, "64 elements"),
            ((x, y), {"weight": c.double()}, "weight must be"),
            ((x, y), {"bias": t(64, device="cuda:1")}, "same device"),
            ((x, y), {"gate": t(2, 64)}, "leading dimensions"),
            ((x, y), {"gate": t(1, 8, 64)}, "leading dimensions"),
            ((x, y), {"scale": t(32)}, "must end in 64"),
            ((x, y), {"shift": t(1, 2, 8, 64)}, "must end in 64"),
            ((x, y), {"shift": t(64, dtype=torch.float64)}, "shift must be"),
            ((x, y), {"out_dtype": torch.float64}, "out_dtype"),
            ((x, y), {"packed": True, "out_dtype": torch.float32}, "rounded to out_dtype first"),
            ((t(2, 40), t(2, 40)), {"packed": True}, "multiple of 32"),
            ((t(2, 16385),), {}, "at most 16384"),
            ((t(2, 0),), {}, "at least one element"),
            ((t(),), {}, "at least one element"),
        ):
            with pytest.raises(RuntimeError, match=match):
                f(*args, **kw)
        for name in ("gate", "weight"):
            with pytest.raises(RuntimeError, match="no backward"):
                f(x, y, **{name: torch.empty((64,), device="cuda", requires_grad=True)})


def test_c_entries_check_their_arguments(native):
    lib = native.load_library()
    null, one, odd = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(24)       # never dereferenced: the checks fail first

    def says(status, code, text):
        assert status == code, lib.feather_last_error_string()
        if text:
            assert text in lib.feather_last_error_string()

    q = lib.feather_mxfp4_quantize
    says(q(one, 0, 4, 48, 48, one, one, null), 1, b"divisible by 32")
    says(q(one, 0, -1, 32, 32, one, one, null), 1, b"negative")
    says(q(one, 7, 4, 32, 32, one, one, null), 1, b"src_dtype")
    says(q(null, 0, 4, 32, 32, one, one, null), 1, b"null")
    says(q(one, 0, 4, 64, 32, one, one, null), 1, b"ld")
    says(q(one, 0, 4, 32, 32, odd, one, null), 1, b"16-byte")
    says(q(ctypes.c_void_p(17), 1, 4, 32, 32, one, one, null), 1, b"element size")
    says(q(one, 0, 4, 1 << 31, 1 << 31, one, one, null), 1, b"30")
    says(q(null, 0, 0, 32, 32, null, null, null), 0, b"")
    d = lib.feather_mxfp4_dequantize
    says(d(one, one, 4, 32, 5, one, null), 1, b"dst_dtype")
    says(d(one, one, 4, 32, 0, odd, null), 1, b"16-byte")
    says(d(null, null, 0, 32, 0, null, null), 0, b"")
    m = lib.feather_mxfp4_mm
    says(m(one, one, one, one, null, one, 4, 8, 48, 8, 0, null, null), 1, b"divisible by 32")
    says(m(one, one, one, one, null, one, 4, 0, 32, 8, 0, null, null), 1, b"positive")
    says(m(one, one, one, one, null, one, 4, 8, 32, 4, 0, null, null), 1, b"ldc")
    says(m(one, one, one, one, null, one, 4, 8, 32, 8, 2, null, null), 1, b"output_dtype")
    says(m(one, null, one, one, null, one, 4, 8, 32, 8, 0, null, null), 1, b"null")
    says(m(one, odd, one, one, null, one, 4, 8, 32, 8, 0, null, null), 1, b"16-byte")
    says(m(one, one, one, one, ctypes.c_void_p(17), one, 4, 8, 32, 8, 0, null, null), 1, b"element size")
    says(m(null, null, null, null, null, null, 0, 8, 32, 8, 0, null, null), 0, b"")

    def args(**kw):
        base = dict(x=16, y=16, r=16, h=16, rows=4, cols=64, ldx=64, ldy=64, ldr=64, ldh=64, x_dtype=1, y_dtype=1, h_dtype=1, eps=1e-6, residual_scale=1.0)
        return native.NormArgs(**{**base, **kw})

    for kw, code, text in (
        ({"cols": 0}, 1, b"positive"), ({"cols": 16385}, 2, b"16384"), ({"rows": 1 << 31}, 1, b"31 bits"), ({"kind": 2}, 1, b"kind"), ({"x": 0}, 1, b"null"),
        ({"r": 0, "h": 0}, 1, b"null"), ({"y": 0}, 1, b"need y"), ({"post_weight": 16}, 1, b"post_norm"), ({"gate": 16}, 1, b"gate_rows"),
        ({"x_dtype": 3}, 1, b"unknown type"), ({"x": 17}, 1, b"misaligned"), ({"ldy": 63}, 1, b"row pitch"), ({"gate": 16, "gate_rows": 2, "gate_ld": 8}, 1, b"row pitch"),
        ({"h_scales": 16, "cols": 40}, 1, b"divisible by 32"), ({"h_scales": 16, "h_dtype": 0}, 1, b"h_dtype"), ({"h_scales": 24}, 1, b"16-byte"),
        ({"h_scales": 16, "ldx": 65}, 1, b"16-byte"), ({"rows": 0, "x": 0}, 0, b""),
    ):
        says(lib.feather_gated_norm(ctypes.byref(args(**kw)), null), code, text)
    says(lib.feather_gated_norm(None, null), 1, b"null")


def test_operations_and_loader_take_a_weight_format(pkg):
    ops_mod = importlib.import_module("feather_b200.comfy_feather.ops")
    loader = importlib.import_module("feather_b200.comfy_feather.loader")
    layout = importlib.import_module("feather_b200.comfy_feather.mxfp4")
    import comfy.sd

    with pytest.raises(ValueError, match="weight_format"):
        ops_mod.feather_ops(weight_format="nvfp4")
    assert loader.FeatherUNetLoader.INPUT_TYPES()["optional"]["weight_format"][0] == ["fp8e5m2", "mxfp4"]
    loader.FeatherUNetLoader().load_unet("model_a.safetensors", "wan", "mxfp4")
    ops = comfy.sd._last_call["model_options"]["custom_operations"]
    assert issubclass(ops.Linear, ops_mod._FeatherMXFP4Linear) and ops._out_dtype == torch.float16
    loader.FeatherUNetLoader().load_unet("model_a.safetensors", "wan")
    assert not issubclass(comfy.sd._last_call["model_options"]["custom_operations"].Linear, ops_mod._FeatherMXFP4Linear)

    # a packed checkpoint needs no GPU to load; its values come back as they were saved
    lin = ops_mod.feather_ops(weight_format="mxfp4").Linear(96, 40, bias=False)
    data = torch.randint(0, 256, (40, 48), generator=torch.Generator().manual_seed(1)).to(torch.uint8)
    scale = torch.randint(100, 140, (40, 3), generator=torch.Generator().manual_seed(2)).to(torch.uint8)
    lin._load_from_state_dict({"l.weight": data, "l.weight_scale": scale}, "l.", {}, True, [], [], [])
    assert lin.is_quantized and tuple(lin.weight.shape) == (40, 96)
    saved = layout.FeatherMXFP4Layout.state_dict_tensors(lin.weight._qdata, lin.weight._params)
    assert torch.equal(saved[""], data) and torch.equal(saved["_scale"], scale)
    with pytest.raises(ValueError, match="recalculate"):
        layout.FeatherMXFP4Layout.quantize(torch.zeros((4, 32)), scale=torch.tensor(1.0))
    with pytest.raises(ValueError, match="divisible by 32"):
        layout.quantize_mxfp4_weight(torch.zeros((4, 48)))
    with pytest.raises(TypeError, match="FeatherMXFP4Layout"):
        layout.get_mxfp4_plain_tensors(torch.zeros(4))
