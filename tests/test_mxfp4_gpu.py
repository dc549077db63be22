"""GPU: MXFP4 quantisation, dequantisation and the MXFP4 product against plain 64-bit forms (tests/mx_ref.py).

Quantising is exact arithmetic (a power-of-two scale, one rounding), so codes and scales are compared bit for bit.  The product is
compared element by element within the bound of fp32 accumulation and one rounding."""

import importlib

import pytest
import torch

from tests import mx_ref

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("feather_b200.kernel.mxfp4")


def _rows(rows, k, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, k), generator=g) * torch.exp2(torch.randint(-6, 7, (rows, k // 32), generator=g).float()).repeat_interleave(32, dim=1)
    return x.to(dtype).to(dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 64), (3, 96), (7, 160), (128, 128), (129, 1024), (300, 1056), (1, 5120), (33, 13824)])
def test_quantise_bit_for_bit(mx, cuda_dev, rows, k, dtype):
    x = _rows(rows, k, dtype, rows + k, cuda_dev)
    data, scales = mx.quantize_mxfp4(x)
    codes, ref_scales = mx_ref.quantize(x)
    assert torch.equal(mx.unprepack_mxfp4_scales(scales, rows, k), ref_scales)
    assert torch.equal(data, mx_ref.pack(codes))
    tail = scales.view(scales.shape[0], scales.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:rows, k // 32:]
    assert not tail.any()                                                   # a row's scale bytes past its last block are zero
    for out in DTYPES:
        y = mx.dequantize_mxfp4(data, scales, out)
        ref = mx_ref.values(codes, ref_scales)
        assert torch.equal(y.float(), ref.to(out).float())


def test_quantise_every_border(mx, cuda_dev):
    """Blocks whose scaled elements are every border between two codes, its two neighbours, and both signs, at the smallest, an ordinary
    and the largest scale; block maxima next to powers of two, where the scale changes."""
    grid = torch.tensor(mx_ref.GRID)
    border = (grid[1:] + grid[:-1]) / 2
    points = torch.cat([border, torch.nextafter(border, border + 1), torch.nextafter(border, border - 1), grid, torch.tensor([7.0, 7.5])])
    points = torch.cat([points, -points])
    points = torch.cat([points, torch.zeros((-len(points)) % 31)]).view(-1, 31)
    blocks = torch.cat([points, torch.full((len(points), 1), 4.0)], dim=1)  # the 4 pins the scale at 1 (largest element in [4, 8))
    for e in (-120, -3, 0, 9, 124):
        x = torch.ldexp(blocks, torch.tensor(e)).to(cuda_dev)
        data, scales = mx.quantize_mxfp4(x)
        codes, ref = mx_ref.quantize(x)
        assert torch.equal(mx.unprepack_mxfp4_scales(scales, len(x), 32), ref) and torch.equal(data, mx_ref.pack(codes))
        assert ref.unique().tolist() == [127 + e]
    powers = torch.ldexp(torch.ones(40), torch.arange(-150, 128, 7)[:40].int())
    tops = torch.cat([powers, torch.nextafter(powers, torch.full_like(powers, float("inf"))), torch.nextafter(powers, torch.zeros_like(powers))])
    x = torch.zeros((len(tops), 32))
    x[:, 5], x[:, 6], x[:, 31] = tops, -tops / 3, tops / 5
    x = x.to(cuda_dev)
    data, scales = mx.quantize_mxfp4(x)
    codes, ref = mx_ref.quantize(x)
    assert torch.equal(mx.unprepack_mxfp4_scales(scales, len(x), 32), ref) and torch.equal(data, mx_ref.pack(codes))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantise_nan_infinity_and_zero_blocks(mx, cuda_dev, dtype):
    x = torch.ones((6, 96), dtype=dtype)
    x[0, 40], x[1, 0], x[2, 95], x[3, 32:64] = float("nan"), float("inf"), float("-inf"), 0.0
    x[4, :32] = -0.0
    x = x.to(cuda_dev)
    data, scales = mx.quantize_mxfp4(x)
    codes, ref = mx_ref.quantize(x)
    assert torch.equal(mx.unprepack_mxfp4_scales(scales, 6, 96), ref) and torch.equal(data, mx_ref.pack(codes))
    assert ref[0, 1] == 255 and ref[1, 0] == 255 and ref[2, 2] == 255 and ref[3, 1] == 0
    y = mx.dequantize_mxfp4(data, scales, torch.float32)
    assert torch.isnan(y[0, 32:64]).all() and torch.isnan(y).sum() == 96 and (y[3, 32:64] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantise_strided_and_misaligned_rows(mx, cuda_dev, dtype):
    wide = _rows(9, 320, dtype, 3, cuda_dev)
    for view in (wide[:, 32:192], wide[:, 1:161], wide[::2, 64:128], wide.t()[:256, :8].t()[:, :256], wide[:1, 3:35], wide[4:5].expand(4, 320)):
        data, scales = mx.quantize_mxfp4(view)
        ref_data, ref_scales = mx.quantize_mxfp4(view.contiguous().clone())
        assert torch.equal(data, ref_data)
        assert torch.equal(mx.unprepack_mxfp4_scales(scales, *view.shape), mx.unprepack_mxfp4_scales(ref_scales, *view.shape))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1030, 5120), (4111, 96), (2100, 1312)])
def test_quantise_many_rows_of_every_alignment(mx, cuda_dev, rows, k, dtype):
    """Rows that begin on 32-byte, 16-byte and element boundaries only, each of them pitched and not: the loads differ, the bits do not."""
    x = _rows(rows, k, dtype, 5, cuda_dev)
    codes, ref_scales = mx_ref.quantize(x)
    packed = mx_ref.pack(codes)
    for first, pitch in ((0, k), (8, k), (3, k), (0, k + 16), (0, k + 8), (16, k + 32), (8, k + 24), (1, k + 1)):
        flat = torch.full((first + rows * pitch,), float("nan"), dtype=dtype, device=cuda_dev)
        view = flat[first:].view(rows, pitch)[:, :k]
        view.copy_(x)
        data, scales = mx.quantize_mxfp4(view)
        assert torch.equal(data, packed) and torch.equal(mx.unprepack_mxfp4_scales(scales, rows, k), ref_scales), (first, pitch)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantise_every_16_bit_value(mx, cuda_dev, dtype):
    """All 65 536 patterns, among neighbours of their own size and among far smaller and larger ones."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    shuffled = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(1))]
    x = torch.cat([bits, shuffled]).view(dtype).view(-1, 64).to(cuda_dev)
    data, scales = mx.quantize_mxfp4(x)
    codes, ref = mx_ref.quantize(x)
    assert torch.equal(mx.unprepack_mxfp4_scales(scales, len(x), 64), ref) and torch.equal(data, mx_ref.pack(codes))


def test_empty_calls(mx, cuda_dev):
    data, scales = mx.quantize_mxfp4(torch.empty((0, 64), device=cuda_dev))
    assert data.shape == (0, 32) and scales.shape == (0, 1, 512)
    assert mx.dequantize_mxfp4(data, scales, torch.bfloat16).shape == (0, 64)
    b, bs = mx.quantize_mxfp4(torch.ones((5, 64), device=cuda_dev))
    assert mx.scaled_mm_mxfp4(data, scales, b, bs).shape == (0, 5)
    assert mx.linear_mxfp4(torch.empty((2, 0, 64), device=cuda_dev), b, bs).shape == (2, 0, 5)


# ------------------------------------------------------------------------------------------------ product
def _operand(mx, rows, k, seed, dev, spread=3):
    """Random codes and scales (every code occurs, scales 2^-spread .. 2^spread), with their fp64 values."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (rows, k), generator=g).to(torch.uint8)
    scales = (127 + torch.randint(-spread, spread + 1, (rows, k // 32), generator=g)).to(torch.uint8)
    return mx_ref.pack(codes).to(dev), mx.prepack_mxfp4_scales(scales).to(dev), mx_ref.values(codes, scales).to(dev)


SHAPES = [(1, 1, 32), (1, 8, 64), (1, 128, 256), (2, 130, 96), (5, 257, 160), (16, 384, 512), (17, 129, 1056), (31, 640, 800), (33, 1000, 288), (64, 128, 2048), (65, 511, 320),
          (128, 256, 1024), (129, 384, 544), (200, 1024, 384), (255, 777, 1312), (257, 256, 256), (520, 2811, 1056), (1000, 520, 640), (1, 5120, 13824), (7, 1100, 4096),
          (300, 1, 64), (70, 8, 32), (1000, 100, 96), (2100, 193, 160), (64, 3, 13824), (4099, 1537, 96),
          (2048, 4608, 2048), (1999, 4601, 2016)]                           # enough tiles and stages for the 256-feature tile


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(mx, native, cuda_dev, m, n, k):
    a, sa, va = _operand(mx, m, k, 1 + m + n + k, cuda_dev)
    b, sb, vb = _operand(mx, n, k, 2 + m + n + k, cuda_dev)
    exact = va @ vb.t()
    for dtype in (torch.bfloat16, torch.float16):
        for with_bias in (False, True):
            bias = (torch.randn((n,), generator=torch.Generator().manual_seed(3)) * 4).to(dtype).to(cuda_dev) if with_bias else None
            ref = exact + bias.double() if with_bias else exact
            y = mx.scaled_mm_mxfp4(a, sa, b, sb, bias, dtype)
            native.check_device_status(cuda_dev)
            assert y.shape == (m, n) and y.dtype == dtype
            top = 65504.0 if dtype == torch.float16 else 3e38
            keep = ref.abs() < top * 0.99
            err = (y.double() - ref).abs()
            limit = mx_ref.product_bound(va, vb, ref, dtype)
            worst = float((err[keep] / limit[keep]).max()) if keep.any() else 0.0
            assert worst <= 1.0, (dtype, with_bias, worst)
            again = mx.scaled_mm_mxfp4(a, sa, b, sb, bias, dtype)
            assert torch.equal(again.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("m,n", [(3, 200), (70, 130), (150, 300), (600, 300)])
def test_product_finds_each_element(mx, cuda_dev, m, n):
    """One non-zero element of a (and all of b different powers of two and codes): a wrong scale, nibble or row shows exactly."""
    k = 544
    b, sb, vb = _operand(mx, n, k, 9, cuda_dev, spread=7)
    g = torch.Generator().manual_seed(m)
    codes = torch.zeros((m, k), dtype=torch.uint8)
    at = torch.randint(0, k, (m,), generator=g)
    codes[torch.arange(m), at] = torch.randint(1, 8, (m,), generator=g).to(torch.uint8)
    scales = (127 + torch.randint(-7, 8, (m, k // 32), generator=g)).to(torch.uint8)
    a, sa = mx_ref.pack(codes).to(cuda_dev), mx.prepack_mxfp4_scales(scales).to(cuda_dev)
    y = mx.scaled_mm_mxfp4(a, sa, b, sb, None, torch.bfloat16)
    exact = mx_ref.values(codes, scales).to(cuda_dev) @ vb.t()
    assert torch.equal(y.double(), exact.to(torch.bfloat16).double())


@pytest.mark.parametrize("m", [1, 40, 130, 300])
def test_product_with_nan_blocks_and_dirty_padding(mx, cuda_dev, m):
    """A NaN scale poisons its row (a) or column (b) and nothing else; what lies in the scale tiles beyond the last row does not matter."""
    n, k = 150, 320
    a, sa, va = _operand(mx, m, k, 21, cuda_dev)
    b, sb, vb = _operand(mx, n, k, 22, cuda_dev)
    clean = mx.scaled_mm_mxfp4(a, sa, b, sb)

    def tiled(plain, fill):
        rows, blocks = plain.shape
        full = torch.full(((rows + 127) // 128 * 128, (blocks + 3) // 4 * 4), fill, dtype=torch.uint8, device=cuda_dev)
        full[:rows] = 0
        full[:rows, :blocks] = plain
        return mx.prepack_mxfp4_scales(full)

    pa, pb = mx.unprepack_mxfp4_scales(sa, m, k), mx.unprepack_mxfp4_scales(sb, n, k)
    dirty = mx.scaled_mm_mxfp4(a, tiled(pa, 255), b, tiled(pb, 255))
    assert torch.equal(dirty.view(torch.int16), clean.view(torch.int16))
    pa[m // 2, 3], pb[n - 2, 9] = 255, 255
    y = mx.scaled_mm_mxfp4(a, mx.prepack_mxfp4_scales(pa), b, mx.prepack_mxfp4_scales(pb))
    nan = torch.zeros((m, n), dtype=torch.bool, device=cuda_dev)
    nan[m // 2], nan[:, n - 2] = True, True
    assert torch.equal(torch.isnan(y), nan)
    assert torch.equal(y[~nan].view(torch.int16), clean[~nan].view(torch.int16))


def test_product_into_a_column_slice(mx, native, cuda_dev):
    for m, n, k in ((5, 72, 128), (300, 200, 256), (40, 129, 96)):
        a, sa, _ = _operand(mx, m, k, 31, cuda_dev)
        b, sb, _ = _operand(mx, n, k, 32, cuda_dev)
        ref = mx.scaled_mm_mxfp4(a, sa, b, sb)
        for left, pad in ((8, 8), (3, 4), (0, 1)):
            wide = torch.full((m, left + n + pad), 7.0, dtype=torch.bfloat16, device=cuda_dev)
            native.mxfp4_mm_into(a, sa, b, sb, None, wide[:, left:left + n])
            assert torch.equal(wide[:, left:left + n], ref)
            assert (wide[:, :left] == 7).all() and (wide[:, left + n:] == 7).all()


def test_linear_is_quantise_then_product(mx, cuda_dev):
    w = (torch.randn((300, 256), generator=torch.Generator().manual_seed(1)) / 16).to(cuda_dev)
    b, sb = mx.quantize_mxfp4(w)
    bias = torch.randn(300, generator=torch.Generator().manual_seed(2)).to(cuda_dev)
    for dtype, out in ((torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.bfloat16)):
        x = torch.randn((2, 70, 256), generator=torch.Generator().manual_seed(3)).to(dtype).to(cuda_dev)
        y = mx.linear_mxfp4(x, b, sb, bias.to(out))
        a, sa = mx.quantize_mxfp4(x.view(-1, 256))
        assert y.shape == (2, 70, 300) and torch.equal(y.view(-1, 300), mx.scaled_mm_mxfp4(a, sa, b, sb, bias.to(out), out))
        exact = mx_ref.values(*mx_ref.quantize(x.view(-1, 256))) @ mx_ref.values(*mx_ref.quantize(w)).t() + bias.to(out).double()
        mx_ref.within(y.view(-1, 300), exact, mx_ref.product_bound(mx_ref.values(*mx_ref.quantize(x.view(-1, 256))), mx_ref.values(*mx_ref.quantize(w)), exact, out), "linear")


def test_streams_and_graphs(mx, cuda_dev):
    """The same bits on a side stream, from a captured graph, and from two graphs replayed side by side."""
    w = torch.randn((512, 1024), generator=torch.Generator().manual_seed(1)).to(cuda_dev)
    b, sb = mx.quantize_mxfp4(w)
    xs = [torch.randn((m, 1024), generator=torch.Generator().manual_seed(m)).to(torch.bfloat16).to(cuda_dev) for m in (3, 200)]
    ref = [mx.linear_mxfp4(x, b, sb) for x in xs]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in xs]
    for s, x, r in zip(sides, xs, ref):
        with torch.cuda.stream(s):
            y = mx.linear_mxfp4(x, b, sb)
        s.synchronize()
        assert torch.equal(y, r)
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mx.linear_mxfp4(x, b, sb))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, sides):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, r) for o, r in zip(outs, ref))


def test_custom_ops_and_fakes(mx, cuda_dev):
    x = torch.randn((40, 128), device=cuda_dev)
    data, scales = torch.ops.feather_ops_internal.quantize_mxfp4(x)
    y = torch.ops.feather_ops_internal.scaled_mm_mxfp4(data, scales, data, scales, None, torch.float16)
    assert torch.equal(y, mx.scaled_mm_mxfp4(data, scales, data, scales, None, torch.float16))
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        f = torch.empty((40, 128), device="cuda")
        fd, fs = torch.ops.feather_ops_internal.quantize_mxfp4(f)
        assert fd.shape == data.shape and fs.shape == scales.shape and fd.dtype == fs.dtype == torch.uint8
        fy = torch.ops.feather_ops_internal.scaled_mm_mxfp4(fd, fs, fd, fs, None, torch.float16)
        assert fy.shape == y.shape and fy.dtype == y.dtype


def test_first_call_inside_a_capture(tmp_path):
    """A process whose first calls of these operators are captured: the graph replays right, nothing kept from the capture (a status word)
    outlives it, and eager calls follow."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    script = tmp_path / "first.py"
    script.write_text("""
import gc, importlib, sys
sys.path.insert(0, %r)
import torch, __graft_entry__
__graft_entry__.load_package()
mx = importlib.import_module("feather_b200.kernel.mxfp4")
norm = importlib.import_module("feather_b200.kernel.norm").gated_residual_norm
native = importlib.import_module("feather_b200.kernel.b200.native")
w, x = torch.randn((640, 512), device="cuda"), torch.randn((2500, 512), device="cuda", dtype=torch.bfloat16)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    b = mx.quantize_mxfp4(w)
    r, h = norm(x, x, gate=w[0], packed=True)
    out = mx.scaled_mm_mxfp4(*h, *b), mx.linear_mxfp4(x[:5], *b), r
g.replay()
torch.cuda.synchronize()
got = [o.clone() for o in out]
del g, b, r, h, out
gc.collect()
torch.cuda.empty_cache()
b = mx.quantize_mxfp4(w)
r, h = norm(x, x, gate=w[0], packed=True)
ref = mx.scaled_mm_mxfp4(*h, *b), mx.linear_mxfp4(x[:5], *b), r
native.check_device_status()
assert all(torch.equal(a, c) for a, c in zip(got, ref))
print("captured first")
""" % root)
    res = subprocess.run([sys.executable, str(script)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert res.returncode == 0 and "captured first" in res.stdout, res.stdout[-2000:]


def test_threads_on_streams_of_their_own(mx, cuda_dev):
    """Several threads at once, each on its own stream: few tokens (clusters), many tokens (pairs) and the norm in between."""
    import threading

    norm = importlib.import_module("feather_b200.kernel.norm").gated_residual_norm
    b, sb = mx.quantize_mxfp4(torch.randn((768, 640), generator=torch.Generator().manual_seed(1)).to(cuda_dev))
    xs = [torch.randn((m, 640), generator=torch.Generator().manual_seed(m)).to(torch.bfloat16).to(cuda_dev) for m in (1, 40, 300, 2600)]

    def step(x):
        r, h = norm(x, x, post_norm=True, packed=True)
        return r, mx.scaled_mm_mxfp4(*h, b, sb), mx.linear_mxfp4(x, b, sb)

    ref = [step(x) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = step(xs[i])
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, c) for a, c in zip(got, ref[i])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_fakes_of_the_other_operators(mx, cuda_dev):
    from torch._subclasses.fake_tensor import FakeTensorMode

    importlib.import_module("feather_b200.kernel.norm")
    ops = torch.ops.feather_ops_internal
    x = torch.randn((2, 40, 128), device=cuda_dev, dtype=torch.bfloat16)
    data, scales = mx.quantize_mxfp4(x[0])

    def results(x, data, scales):
        n = (x, x, None, 1.0, False, None, None, None, None, None, "rms", 1e-6)
        return [ops.dequantize_mxfp4(data, scales, torch.float16), ops.linear_mxfp4(x, data, scales, None, None), *ops.gated_residual_norm(*n, torch.bfloat16, True, False),
                *ops.gated_residual_norm(*n, torch.bfloat16, True, True), *ops.gated_residual_norm(*n, torch.bfloat16, False, False), *ops.gated_residual_norm(x, *[None] * 2, *n[3:], torch.float32, True, False)]

    real = results(x, data, scales)
    with FakeTensorMode():
        fake = results(*(torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (x, data, scales)))
    assert [(t.shape, t.dtype) for t in real] == [(t.shape, t.dtype) for t in fake]
