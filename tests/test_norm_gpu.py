"""GPU: the fused gate, residual and norms against the plain 64-bit form (tests/mx_ref.py), element by element within the bound of
fp32 arithmetic and one rounding."""

import importlib

import pytest
import torch

from tests import mx_ref

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def norm(pkg):
    return importlib.import_module("feather_b200.kernel.norm")


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("feather_b200.kernel.mxfp4")


def _t(shape, seed, dev, dtype=FP32, spread=1.0, about=0.0):
    return (about + spread * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).to(dev)


def _check(norm, x, y, out_dtype=None, **kw):
    r, h = norm.gated_residual_norm(x, y, out_dtype=out_dtype, **kw)
    kw["residual_scale"] = float(torch.tensor(kw.get("residual_scale", 1.0), dtype=FP32))
    ref_r, ref_h, off_r, off_h = mx_ref.gated_norm(x, y, **kw)
    if y is None:
        assert r is x
    else:
        assert r.dtype == x.dtype and r.shape == x.shape
        mx_ref.within(r, ref_r, off_r, "r")
    assert h.shape == x.shape
    mx_ref.within(h, ref_h, off_h, "h")
    return r, h


WIDTHS = [1, 7, 8, 33, 64, 127, 256, 257, 512, 1000, 1024, 1027, 1032, 2048, 4097, 5120, 8192, 8200, 13824, 16383, 16384]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("cols", WIDTHS)
def test_widths(norm, cuda_dev, cols, kind):
    for rows in (1, 5):
        x, y = _t((rows, cols), cols, cuda_dev, BF16, about=0.3), _t((rows, cols), cols + 1, cuda_dev, BF16)
        w, b, pw, g = _t((cols,), 3, cuda_dev, BF16, 0.2, 1.0), _t((cols,), 4, cuda_dev), _t((cols,), 5, cuda_dev, FP16, 0.2, 1.0), _t((cols,), 6, cuda_dev, BF16)
        _check(norm, x, y, gate=g, residual_scale=0.5, post_norm=True, post_weight=pw, weight=w, bias=b, kind=kind)


def test_many_rows_take_the_wide_threads(norm, cuda_dev):
    """More rows than the one-vector-a-thread form takes."""
    for cols in (2048, 5120, 8192):
        x, y = _t((400, cols), 1, cuda_dev, BF16), _t((400, cols), 2, cuda_dev, BF16)
        for kind in ("rms", "layer"):
            _check(norm, x, y, gate=_t((cols,), 3, cuda_dev), post_norm=True, scale=_t((cols,), 4, cuda_dev, spread=0.2), shift=_t((cols,), 5, cuda_dev), kind=kind)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("cols", [8, 40, 64, 256, 264, 320, 512, 520, 1000, 1024, 1032, 2048, 2560, 4096, 5120, 5128, 6144, 8192, 8200, 13824, 16384])
def test_thousands_of_rows(norm, mx, cuda_dev, cols, kind):
    """The form for many rows: samples that end inside a wave of rows, whole and partial vectors, all three coefficients or none, h alone
    and r alone, and the MXFP4 result."""
    batch, length = 3, 1601 if cols <= 2560 else 901
    x, y = _t((batch, length, cols), 1, cuda_dev, BF16), _t((batch, length, cols), 2, cuda_dev, BF16)
    kw = dict(gate=_t((batch, 1, cols), 3, cuda_dev), scale=_t((batch, 1, cols), 4, cuda_dev, spread=0.2), shift=_t((batch, 1, cols), 5, cuda_dev), kind=kind)
    r, h = _check(norm, x, y, post_norm=True, post_weight=_t((cols,), 6, cuda_dev, BF16, 0.2, 1.0), **kw)
    _check(norm, x, y, kind=kind)
    _check(norm, x, None, kind=kind, weight=_t((cols,), 7, cuda_dev, FP16, 0.2, 1.0), bias=_t((cols,), 8, cuda_dev))
    alone, none = norm.gated_residual_norm(x, y, gate=kw["gate"], kind=kind, want_norm=False)
    both, _ = norm.gated_residual_norm(x, y, gate=kw["gate"], kind=kind)
    assert none is None and torch.equal(alone, both)
    if cols % 32 == 0:
        _, h = norm.gated_residual_norm(x, y, **kw)
        _, (data, scales) = norm.gated_residual_norm(x, y, packed=True, **kw)
        ref_data, ref_scales = mx.quantize_mxfp4(h.view(-1, cols))
        assert torch.equal(data, ref_data)
        assert torch.equal(mx.unprepack_mxfp4_scales(scales, batch * length, cols), mx.unprepack_mxfp4_scales(ref_scales, batch * length, cols))


@pytest.mark.parametrize("x_dtype,y_dtype", [(FP32, FP32), (FP32, FP16), (FP16, BF16), (BF16, FP32)])
def test_thousands_of_rows_of_other_types(norm, cuda_dev, x_dtype, y_dtype):
    for cols in (200, 1024, 5120, 12288):
        x, y = _t((5, 701, cols), 1, cuda_dev, x_dtype, about=3.0), _t((5, 701, cols), 2, cuda_dev, y_dtype)
        _check(norm, x, y, gate=_t((5, 1, cols), 3, cuda_dev, y_dtype), post_norm=True, shift=_t((cols,), 4, cuda_dev), kind="layer")
        wide = torch.zeros((3505, cols + 16), dtype=x_dtype, device=cuda_dev)
        wide[:, 8:-8] = x.view(-1, cols)
        _check(norm, wide[:, 8:-8], y.view(-1, cols), residual_scale=0.25)


@pytest.mark.parametrize("x_dtype,y_dtype", [(BF16, BF16), (FP16, FP16), (FP32, FP32), (FP32, BF16), (FP16, BF16)])
def test_thousands_of_rows_without_a_norm_of_y(norm, cuda_dev, x_dtype, y_dtype):
    """Nothing waits for y's statistics: both sides of the widths and of the shared memory where the form for it ends (12288 fp32 columns
    with coefficients are too many, without them they are not)."""
    for cols in (520, 1536, 5120, 6144, 12288, 12296):
        x, y = _t((3, 701, cols), 1, cuda_dev, x_dtype, about=0.5), _t((3, 701, cols), 2, cuda_dev, y_dtype)
        for kind in ("rms", "layer"):
            _check(norm, x, y, gate=_t((3, 1, cols), 3, cuda_dev), scale=_t((3, 1, cols), 4, cuda_dev, spread=0.2), shift=_t((cols,), 5, cuda_dev), kind=kind)
        _check(norm, x, y, residual_scale=0.25, weight=_t((cols,), 7, cuda_dev, FP16, 0.2, 1.0), kind="rms")
        _check(norm, x, y, kind="layer")
        _check(norm, x, None, bias=_t((cols,), 8, cuda_dev), kind="layer")


@pytest.mark.parametrize("cols", [1, 2, 31, 33, 255, 257, 513, 1027, 2047, 2049, 4099, 8191, 15873, 16383])
def test_odd_widths_beside_a_warp_and_a_block(norm, cuda_dev, cols):
    """Widths where a warp's part of a row is one element, whole, or short of whole by one, in rows that begin at every alignment; r alone and
    h alone."""
    x, y = _t((2, 5, cols), 1, cuda_dev, FP16, about=0.5), _t((2, 5, cols), 2, cuda_dev, BF16)
    for kind in ("rms", "layer"):
        r, h = _check(norm, x, y, gate=_t((2, 5, cols), 3, cuda_dev), post_norm=True, post_weight=_t((cols,), 6, cuda_dev, BF16, 0.2, 1.0),
                      scale=_t((2, 1, cols), 4, cuda_dev, FP16, 0.2), shift=_t((cols,), 5, cuda_dev, BF16), kind=kind)
        _check(norm, x, None, kind=kind, weight=_t((cols,), 7, cuda_dev, FP16, 0.2, 1.0), bias=_t((cols,), 8, cuda_dev))
    alone, none = norm.gated_residual_norm(x, y, gate=_t((cols,), 9, cuda_dev), want_norm=False)
    both, _ = norm.gated_residual_norm(x, y, gate=_t((cols,), 9, cuda_dev))
    assert none is None and torch.equal(alone, both)


@pytest.mark.parametrize("x_dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("y_dtype", [BF16, FP16, FP32])
def test_types(norm, cuda_dev, x_dtype, y_dtype):
    for cols in (96, 1027, 2560):
        x, y = _t((2, 9, cols), 1, cuda_dev, x_dtype), _t((2, 9, cols), 2, cuda_dev, y_dtype)
        for out in (BF16, FP16, FP32, None):
            _, h = _check(norm, x, y, out_dtype=out, gate=_t((2, 1, cols), 3, cuda_dev, y_dtype), scale=_t((2, 1, cols), 4, cuda_dev, x_dtype, 0.2), shift=_t((2, 9, cols), 5, cuda_dev))
            assert h.dtype == (out or (x_dtype if x_dtype != FP32 else y_dtype))


@pytest.mark.parametrize("cols", [40, 1027, 4096])
def test_modulation_shapes_and_strides(norm, cuda_dev, cols):
    x, y = _t((3, 4, 5, cols), 1, cuda_dev, BF16), _t((3, 4, 5, cols), 2, cuda_dev, BF16)
    chunks = _t((3, 1, 1, 6 * cols), 3, cuda_dev, spread=0.3).chunk(6, dim=-1)
    _check(norm, x, y, gate=chunks[2], scale=chunks[1], shift=chunks[5], kind="layer")
    _check(norm, x, y, gate=_t((3, 4, 1, cols), 4, cuda_dev), scale=_t((3, 4, 5, cols), 5, cuda_dev, spread=0.2), shift=_t((cols,), 6, cuda_dev))
    _check(norm, x, y, gate=_t((1, 1, 1, cols), 4, cuda_dev), scale=_t((1, cols), 5, cuda_dev, spread=0.2))
    wide = _t((12, cols + 24), 7, cuda_dev, BF16)
    _check(norm, wide[:, 8:8 + cols], wide[:, 16:16 + cols])                # aligned rows of a wider tensor
    _check(norm, wide[::2, 3:3 + cols], wide[1::2, 5:5 + cols], weight=_t((cols + 1,), 8, cuda_dev)[1:])
    _check(norm, _t((cols, 6), 9, cuda_dev, BF16).t(), _t((6, cols), 10, cuda_dev, BF16))
    _check(norm, _t((1, cols), 11, cuda_dev, BF16).expand(6, cols), _t((6, cols), 12, cuda_dev, BF16))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norm_alone_and_residual_alone(norm, cuda_dev, kind):
    x, y = _t((7, 640), 1, cuda_dev, FP16), _t((7, 640), 2, cuda_dev, FP16)
    _check(norm, x, None, kind=kind, weight=_t((640,), 3, cuda_dev, FP16))
    r, h = norm.gated_residual_norm(x, y, gate=_t((640,), 4, cuda_dev), kind=kind, post_norm=True, want_norm=False)
    full, _ = norm.gated_residual_norm(x, y, gate=_t((640,), 4, cuda_dev), kind=kind, post_norm=True)
    assert h is None and torch.equal(r, full)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("cols", [64, 1027, 5120])
def test_rows_of_zeros_infinities_and_far_means(norm, cuda_dev, cols, kind):
    x, y = _t((6, cols), 1, cuda_dev, BF16), _t((6, cols), 2, cuda_dev, BF16)
    x[0], y[0] = 0.0, 0.0                                                   # a padding row: its norm is zero
    x[1, cols // 2] = float("nan")
    x[2, 3] = float("inf")
    x[3] = 500.0 + x[3]                                                     # a mean far from zero
    x[4], y[4] = 2.0 ** -60, 0.0                                            # eps decides
    r, h = norm.gated_residual_norm(x, y, kind=kind)
    assert (h[0] == 0).all() and torch.isnan(h[1]).all() and torch.isnan(r[1]).sum() == 1 and torch.isnan(h[2]).any()
    keep = [0, 3, 4, 5]
    ref_r, ref_h, off_r, off_h = mx_ref.gated_norm(x[keep], y[keep], kind=kind)
    mx_ref.within(r[keep], ref_r, off_r, "r")
    mx_ref.within(h[keep], ref_h, off_h, "h")


@pytest.mark.parametrize("out", [BF16, FP16])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (130, 160), (5, 1024), (9, 1056), (2, 5120), (400, 2080), (1, 13824)])
def test_packed_result_is_the_quantised_result(norm, mx, cuda_dev, rows, cols, out):
    x, y = _t((rows, cols), 1, cuda_dev, BF16), _t((rows, cols), 2, cuda_dev, BF16)
    x[0, 0] = float("nan") if cols == 160 else 1.0
    kw = dict(gate=_t((cols,), 3, cuda_dev), scale=_t((cols,), 4, cuda_dev, spread=0.2), kind="layer", out_dtype=out)
    r, h = norm.gated_residual_norm(x, y, **kw)
    r2, (data, scales) = norm.gated_residual_norm(x, y, packed=True, **kw)
    ref_data, ref_scales = mx.quantize_mxfp4(h)
    assert torch.equal(r.view(torch.int16), r2.view(torch.int16)) and torch.equal(data, ref_data)
    assert torch.equal(mx.unprepack_mxfp4_scales(scales, rows, cols), mx.unprepack_mxfp4_scales(ref_scales, rows, cols))
    off = torch.zeros(rows * cols + 1, dtype=BF16, device=cuda_dev)         # rows that are not 16-byte aligned
    off[1:] = x.flatten()
    r3, (d3, _) = norm.gated_residual_norm(off[1:].view(rows, cols), y, packed=True, **kw)
    assert torch.equal(d3, data) and torch.equal(r3.view(torch.int16), r2.view(torch.int16))


def test_empty_and_graph(norm, cuda_dev):
    r, h = norm.gated_residual_norm(torch.empty((2, 0, 64), device=cuda_dev), torch.empty((2, 0, 64), device=cuda_dev), gate=torch.ones((2, 1, 64), device=cuda_dev))
    assert r.shape == h.shape == (2, 0, 64)
    x, y = _t((37, 640), 1, cuda_dev, BF16), _t((37, 640), 2, cuda_dev, BF16)
    ref = norm.gated_residual_norm(x, y, post_norm=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = norm.gated_residual_norm(x, y, post_norm=True)
    for t in got:
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = norm.gated_residual_norm(x, y, post_norm=True)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("cols", [256, 1000, 4104, 5120, 8192, 12288])
@pytest.mark.parametrize("x_dtype", [BF16, FP32])
def test_a_modulation_for_each_row(norm, mx, cuda_dev, cols, x_dtype):
    shape = (2, 210, cols)
    x, y = _t(shape, 1, cuda_dev, x_dtype), _t(shape, 2, cuda_dev, BF16)
    shift, scale, gate = (t for t in _t((2, 210, 3 * cols), 3, cuda_dev, spread=0.3).chunk(3, dim=-1))
    kw = dict(gate=gate, scale=scale, shift=shift, post_norm=True, post_weight=_t((cols,), 4, cuda_dev, BF16, 0.2, 1.0), weight=_t((cols,), 5, cuda_dev, FP16, 0.2, 1.0), bias=_t((cols,), 6, cuda_dev))
    for kind in ("rms", "layer"):
        _check(norm, x, y, kind=kind, **kw)
    if cols % 32 == 0:
        _, h = norm.gated_residual_norm(x, y, out_dtype=BF16, **kw)
        _, (data, scales) = norm.gated_residual_norm(x, y, out_dtype=BF16, packed=True, **kw)
        ref_data, ref_scales = mx.quantize_mxfp4(h.view(-1, cols))
        assert torch.equal(data, ref_data) and torch.equal(mx.unprepack_mxfp4_scales(scales, 420, cols), mx.unprepack_mxfp4_scales(ref_scales, 420, cols))
