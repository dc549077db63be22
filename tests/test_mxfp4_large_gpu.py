"""GPU: element offsets past 31 and 32 bits, and the row pitches of the C entry of the fused norm."""

import ctypes
import importlib

import pytest
import torch

from tests import mx_ref

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("feather_b200.kernel.mxfp4")


@pytest.fixture(scope="module")
def norm(pkg):
    return importlib.import_module("feather_b200.kernel.norm")


def _rows_at(dev, rows, cols):
    """bf16 rows whose last ones begin past element 2^32, and where to look: the first rows, those around 2^31 and 2^32, the last."""
    assert rows * cols > 1 << 32
    x = torch.empty((rows, cols), dtype=BF16, device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(rows))
    looks = []
    for at in (0, (1 << 31) // cols, (1 << 32) // cols, rows):
        first = max(0, min(at - 128, rows - 256)) // 128 * 128             # scale tiles are of 128 rows
        looks.append(slice(first, min(first + 256, rows)))
    return x, looks


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def test_quantise_and_dequantise_past_32_bits(mx, cuda_dev):
    rows, cols = 540001, 8192
    x, looks = _rows_at(cuda_dev, rows, cols)
    data, scales = mx.quantize_mxfp4(x)
    y = mx.dequantize_mxfp4(data, scales, BF16)
    for s in looks:
        codes, ref = mx_ref.quantize(x[s])
        tiles = scales[s.start // 128:(s.stop + 127) // 128]
        assert torch.equal(data[s], mx_ref.pack(codes)) and torch.equal(mx.unprepack_mxfp4_scales(tiles, s.stop - s.start, cols), ref)
        assert torch.equal(y[s].double(), mx_ref.values(codes, ref))


@pytest.mark.parametrize("cols", [8192, 8193])
def test_norm_past_32_bits(norm, mx, cuda_dev, cols):
    rows = 540001
    x, looks = _rows_at(cuda_dev, rows, cols)
    y = x.flip(-1) if cols == 8193 else x
    gate = torch.randn(cols, device=cuda_dev)
    r, h = norm.gated_residual_norm(x, y, gate=gate, kind="layer")
    for s in looks:
        ref_r, ref_h, off_r, off_h = mx_ref.gated_norm(x[s], y[s], gate=gate, kind="layer")
        mx_ref.within(r[s], ref_r, off_r, "r")
        mx_ref.within(h[s], ref_h, off_h, "h")
    if cols % 32 == 0:
        _, (data, scales) = norm.gated_residual_norm(x, y, gate=gate, kind="layer", packed=True)
        for s in looks:
            codes, ref = mx_ref.quantize(h[s])
            assert torch.equal(data[s], mx_ref.pack(codes)) and torch.equal(mx.unprepack_mxfp4_scales(scales[s.start // 128:(s.stop + 127) // 128], s.stop - s.start, cols), ref)


@pytest.mark.parametrize("n", [8192, 8197])
def test_product_past_32_bits(mx, native, cuda_dev, n):
    """An output of more than 2^32 elements, with and without rows that TMA can store."""
    m, k = 540001, 96
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    x = torch.randn((m, k), device=cuda_dev, generator=g).to(BF16)
    b, sb = mx.quantize_mxfp4(torch.randn((n, k), device=cuda_dev, generator=g))
    y = mx.linear_mxfp4(x, b, sb)
    native.check_device_status(cuda_dev)
    vb = mx_ref.values(mx_ref.unpack(b), mx.unprepack_mxfp4_scales(sb, n, k))
    for at in (0, (1 << 31) // n, (1 << 32) // n, m):
        s = slice(max(0, min(at - 100, m - 200)), min(max(at + 100, 200), m))
        va = mx_ref.values(*mx_ref.quantize(x[s]))
        exact = va @ vb.t()
        mx_ref.within(y[s], exact, mx_ref.product_bound(va, vb, exact, BF16), f"rows {s}")


@pytest.mark.parametrize("rows", [5, 700, 3000])
@pytest.mark.parametrize("cols,pitches", [(1024, (1032, 1040, 1056, 1064)), (520, (521, 528, 536, 523)), (77, (80, 77, 79, 101)), (5120, (5128, 5120, 5136, 5152))])
def test_pitches_of_the_c_entry(native, cuda_dev, rows, cols, pitches):
    """x, y, r and h each with a pitch of their own: the results stand in their rows and nothing is written between them."""
    g = torch.Generator().manual_seed(cols + rows)
    bufs = [torch.randn((rows, p), generator=g).to(BF16).to(cuda_dev) for p in pitches[:2]] + [torch.full((rows, p), 7.0, dtype=BF16, device=cuda_dev) for p in pitches[2:]]
    gate = torch.randn((2, cols + 8), generator=g).to(cuda_dev)             # a row for each half of the rows, pitched too
    half = (rows + 1) // 2
    x, y, r, h = bufs
    status = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    a = native.NormArgs(x=x.data_ptr(), y=y.data_ptr(), r=r.data_ptr(), h=h.data_ptr(), rows=rows, cols=cols, ldx=pitches[0], ldy=pitches[1], ldr=pitches[2], ldh=pitches[3], residual_scale=0.5,
                        eps=1e-6, x_dtype=1, y_dtype=1, h_dtype=1, gate=gate.data_ptr(), gate_rows=half, gate_ld=cols + 8, status_dev=status.data_ptr())
    assert native.load_library().feather_gated_norm(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert int(status) == 0
    each = gate[:, :cols].repeat_interleave(half, dim=0)[:rows]
    ref_r, ref_h, off_r, off_h = mx_ref.gated_norm(x[:, :cols], y[:, :cols], gate=each, residual_scale=0.5)
    mx_ref.within(r[:, :cols], ref_r, off_r, "r")
    mx_ref.within(h[:, :cols], ref_h, off_h, "h")
    assert (r[:, cols:] == 7).all() and (h[:, cols:] == 7).all()
