"""GPU: MXFP4 weights in the ComfyUI operator (under the test double of `comfy`) and the MXFP4 forward of the DiT harness."""

import importlib

import pytest
import torch
import torch.nn.functional as F

from tests import mx_ref

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops_mod(pkg):
    return importlib.import_module("feather_b200.comfy_feather.ops")


@pytest.fixture(scope="module")
def layout(pkg):
    return importlib.import_module("feather_b200.comfy_feather.mxfp4")


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("feather_b200.kernel.mxfp4")


def _randn(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


def _linear(ops_mod, k, n, state, out_dtype=BF16, excluded=(), prefix="blocks.0.ffn."):
    lin = ops_mod.feather_ops(out_dtype=out_dtype, excluded_names=excluded, weight_format="mxfp4").Linear(k, n, bias="bias" in state)
    missing, sd = [], {prefix + key: v for key, v in state.items()}
    lin._load_from_state_dict(sd, prefix, {}, True, missing, [], [])
    assert not missing and not sd
    return lin


@pytest.mark.parametrize("src", [FP32, BF16, FP16])
@pytest.mark.parametrize("x_dtype", [FP32, BF16, FP16])
def test_load_and_forward(ops_mod, layout, cuda_dev, src, x_dtype):
    k, n = 256, 384
    w, bias, x = _randn((n, k), 1, 1 / 16).to(src), _randn((n,), 2), _randn((3, 33, k), 3).to(x_dtype)
    lin = _linear(ops_mod, k, n, {"weight": w, "bias": bias})
    assert lin.is_quantized and layout.is_mxfp4_weight(lin.weight) and lin.weight._qdata.device.type == "cpu"
    lin = lin.to(cuda_dev)
    y = lin(x.to(cuda_dev))
    assert y.shape == (3, 33, n) and y.dtype == x_dtype
    a, b = mx_ref.values(*mx_ref.quantize(x.view(-1, k))), mx_ref.values(*mx_ref.quantize(w))
    exact = a @ b.t() + bias.to(BF16).double()
    off = mx_ref.product_bound(a, b, exact, BF16)                           # rounded to bf16, then cast to x's dtype
    mx_ref.within(y.view(-1, n).cpu(), exact, off, "linear")
    assert lin(x.to(cuda_dev)[:0]).shape == (0, 33, n)


def test_what_stays_plain(ops_mod, cuda_dev):
    for k, excluded in ((48, ()), (64, ("ffn",))):
        w = _randn((40, k), 1)
        lin = _linear(ops_mod, k, 40, {"weight": w}, excluded=excluded)
        assert not lin.is_quantized and torch.equal(lin.weight, w)
        x = _randn((5, k), 2).to(cuda_dev)
        assert torch.equal(lin.to(cuda_dev)(x), F.linear(x, w.to(cuda_dev)))


def test_scaled_fp8_and_packed_checkpoints(ops_mod, layout, mx, cuda_dev):
    n, k = 96, 160
    codes8 = _randn((n, k), 1).to(torch.float8_e5m2)
    lin = _linear(ops_mod, k, n, {"weight": codes8, "weight_scale": torch.tensor(0.25)})
    ref_codes, ref_scales = mx_ref.quantize(codes8.float() * 0.25)
    assert torch.equal(lin.weight._qdata, mx_ref.pack(ref_codes))
    # what a checkpoint of these weights holds loads back bit for bit, from either type of scale bytes
    saved = layout.FeatherMXFP4Layout.state_dict_tensors(lin.weight._qdata, lin.weight._params)
    assert torch.equal(saved[""], mx_ref.pack(ref_codes)) and torch.equal(saved["_scale"], ref_scales)
    for scale in (saved["_scale"], saved["_scale"].view(torch.float8_e8m0fnu)):
        again = _linear(ops_mod, k, n, {"weight": saved[""], "weight_scale": scale})
        assert torch.equal(again.weight._qdata, lin.weight._qdata) and torch.equal(again.weight._params.scale, mx.prepack_mxfp4_scales(ref_scales))
        assert tuple(again.weight.shape) == (n, k)
    excluded = _linear(ops_mod, k, n, {"weight": saved[""], "weight_scale": saved["_scale"]}, excluded=("ffn",))
    assert not excluded.is_quantized and torch.equal(excluded.weight.double(), mx_ref.values(ref_codes, ref_scales))
    with pytest.raises(ValueError, match="scale bytes"):
        layout.make_mxfp4_weight(saved[""], saved["_scale"][:, :2], BF16)
    with pytest.raises(ValueError, match="scale bytes"):
        layout.make_mxfp4_weight(saved[""], None, BF16)


def test_lora_merge_and_unmerged_patches(ops_mod, layout, cuda_dev):
    n, k = 128, 192
    w = _randn((n, k), 1, 0.1)
    lin = _linear(ops_mod, k, n, {"weight": w}).to(cuda_dev)
    plain = lin.convert_weight(lin.weight).to(cuda_dev)                      # the test double leaves the packed data where it was loaded
    assert plain.dtype == BF16 and torch.equal(plain.cpu().double(), mx_ref.values(*mx_ref.quantize(w)))
    merged = plain + 0.01 * _randn((n, k), 2).to(BF16).to(cuda_dev)
    returned = lin.set_weight(merged, seed=7, return_weight=True)
    assert layout.is_mxfp4_weight(returned)
    lin.set_weight(merged, seed=7)
    codes, scales = mx_ref.quantize(merged.cpu())
    assert torch.equal(lin.weight._qdata.cpu(), mx_ref.pack(codes)) and torch.equal(returned._qdata, lin.weight._qdata)
    with pytest.raises(TypeError, match="MXFP4"):
        lin.convert_weight(plain)

    class Adapter:
        weights = (_randn((n, 8), 3, 0.1), _randn((8, k), 4, 0.1), None)

    class PatchFn:
        key = "w"
        patches = {"w": [(0.5, Adapter(), 1.0, None, None)]}

    x = _randn((9, k), 5).to(BF16).to(cuda_dev)
    base = lin(x)
    lin.weight_function = [PatchFn()]
    down = F.linear(x, Adapter.weights[1].to(x))
    assert torch.equal(lin(x), base + F.linear(down, Adapter.weights[0].to(x)) * 0.5)
    assert len(lin.weight_function) == 1


# ------------------------------------------------------------------------------------------------ DiT
def _dit(pkg, dev, **kw):
    dit = importlib.import_module("feather_b200.kernel.b200.dit")
    return dit.FeatherDiT(dit.DitConfig(hidden=512, heads=4, head_dim=128, ffn=1408, blocks=3), device=dev, seed=4, init_device=torch.device("cpu"), **kw)


@pytest.mark.parametrize("batch,tokens", [(0, 200), (2, 75), (2, 1), (1, 700)])
@pytest.mark.parametrize("modulated", [False, True])
def test_dit_forward_is_its_steps(pkg, native, mx, cuda_dev, batch, tokens, modulated):
    """The whole forward, run as it is used, equals the same steps one by one: gated residual and norm, quantisation, product.  Bit for
    bit, since the fused norm's MXFP4 result is the quantised 16-bit result.  Every linear is checked against its formula on the way."""
    norm = importlib.import_module("feather_b200.kernel.norm").gated_residual_norm
    model = _dit(pkg, cuda_dev, weight_format="mxfp4")
    cfg = model.cfg
    lead = (batch,) if batch else ()
    x = _randn((*lead, tokens, cfg.hidden), 5).to(BF16).to(cuda_dev)
    mod = None
    if modulated:
        mod = _randn((cfg.blocks, 6, batch, 1, cfg.hidden) if batch else (cfg.blocks, 6, cfg.hidden), 6, 0.3).to(cuda_dev)
    seen = []
    got = model(x, hook=lambda name, i, a, y: seen.append((name, i, a, y)), modulation=mod)
    native.check_device_status(cuda_dev)
    assert got.shape == x.shape and len(seen) == 6 * cfg.blocks

    for name, i, a, y in seen:
        lin = model.blocks[i][name]
        k = lin.data.shape[1] * 2
        data, scales = a if isinstance(a, tuple) else mx.quantize_mxfp4(a.reshape(-1, k))
        va = mx_ref.values(mx_ref.unpack(data), mx.unprepack_mxfp4_scales(scales, data.shape[0], k))
        vb = mx_ref.values(mx_ref.unpack(lin.data), mx.unprepack_mxfp4_scales(lin.scales, lin.data.shape[0], k))
        exact = va @ vb.t() + lin.bias.double()
        mx_ref.within(y, exact, mx_ref.product_bound(va, vb, exact, BF16), f"block {i} {name}")

    r, gate = x, None
    y = None
    for i, blk in enumerate(model.blocks):
        s1, c1, g1, s2, c2, g2 = (None,) * 6 if mod is None else mod[i]
        r, h = norm(r, y, gate=gate, weight=blk["norm1"], shift=s1, scale=c1)
        q, k, v = (blk[n](h).view(-1, tokens, cfg.hidden) for n in "qkv")
        attn = torch.cat([model._attention(q[b], k[b], v[b], blk) for b in range(q.shape[0])])
        r, h = norm(r, blk["o"](attn).view(x.shape), gate=g1, weight=blk["norm2"], shift=s2, scale=c2)
        y, gate = blk["down"](F.gelu(blk["up"](h), approximate="tanh")).view(x.shape), g2
    r, _ = norm(r, y, gate=gate, want_norm=False)
    assert torch.equal(got.view(torch.int16), r.view(torch.int16))
    assert torch.isfinite(got).all()


def test_dit_forward_captured(pkg, cuda_dev):
    model = _dit(pkg, cuda_dev, weight_format="mxfp4")
    x = _randn((96, 512), 5).to(BF16).to(cuda_dev)
    ref = model(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        model(x)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = model(x)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref)


def test_dit_refusals(pkg, cuda_dev):
    with pytest.raises(ValueError, match="weight_format"):
        _dit(pkg, cuda_dev, weight_format="int4")
    with pytest.raises(ValueError, match="one rank"):
        _dit(pkg, cuda_dev, weight_format="mxfp4", world=2)
    with pytest.raises(ValueError, match="modulation"):
        _dit(pkg, cuda_dev)(torch.zeros((4, 512), dtype=BF16, device=cuda_dev), modulation=torch.zeros((3, 6, 512), device=cuda_dev))
