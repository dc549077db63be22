"""MXFP4 (OCP microscaling) weights and activations: quantise, dequantise, and the product of two MXFP4 matrices.

    quantize_mxfp4(x)                                          x [R, K] -> (data, scales)
    dequantize_mxfp4(data, scales, dtype)                      -> [R, K]
    scaled_mm_mxfp4(a, a_scales, b, b_scales, bias, out_dtype) round(a @ b^T + bias), [M, N]
    linear_mxfp4(x, b, b_scales, bias, out_dtype)              quantises x [..., K], then the product, [..., N]
    prepack_mxfp4_scales(scales) / unprepack_mxfp4_scales(scales, rows, k)    [R, K/32] E8M0 bytes <-> the tiles the kernels read

A row of K elements (K % 32 == 0) has K/32 blocks; a block is one E8M0 scale byte s (factor 2^(s - 127), 255 = NaN) and 32 E2M1
elements.  data is uint8 [R, K/2], the even element in the low nibble; scales is uint8 [ceil(R/128), ceil(K/128), 512], a tile for
every 128 rows x 4 blocks (the byte of row r and block j of a tile is at (r % 32) * 16 + (r / 32) * 4 + j).  Quantising takes the
largest power of two not above max|x| / 4 as a block's scale, rounds to nearest even and saturates; a block that holds a NaN or an
infinity becomes NaN.  Sums are fp32 and the result is rounded once.

The operators serve: they have no derivatives.  A call with an input that requires a gradient is refused while gradients are enabled, one
with a dual tensor of forward-mode differentiation always.  The reference (fp8e5m2 weights, per-tensor scale) has no such format.
"""

import torch

from .b200 import native


# What E8M0 bytes are stored as; older torch has no type for them.
SCALE_DTYPES = tuple(getattr(torch, name) for name in ("uint8", "float8_e8m0fnu") if hasattr(torch, name))


def _tiles(rows, k):
    return ((rows + 127) // 128, (k + 127) // 128, 512)


# ------------------------------------------------------------------------------------------------
# format
#
# An operator is one call into the binding; where torch's dispatcher is watched (torch.compile, jit.trace, make_fx, a fake tensor, a dispatch
# mode) the binding says NotImplemented and the registered operator is called, which the watcher sees.
# ------------------------------------------------------------------------------------------------
@torch.library.custom_op("feather_ops_internal::quantize_mxfp4", mutates_args=())
def _quantize_op(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return native.binding().quantize(x, True)


@_quantize_op.register_fake
def _(x):
    rows, k = x.shape
    return torch.empty((rows, k // 2), dtype=torch.uint8, device=x.device), torch.empty(_tiles(rows, k), dtype=torch.uint8, device=x.device)


def quantize_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [R, K] fp32 / bf16 / fp16 on the GPU, K % 32 == 0 -> (data uint8 [R, K/2], scales uint8 [ceil(R/128), ceil(K/128), 512]).
    Rows may be strided; a tensor whose columns are strided is copied first.  Scale bytes of rows past R are not written."""
    out = NotImplemented if torch.compiler.is_compiling() else native.binding().quantize(x)
    return _quantize_op(x) if out is NotImplemented else out


@torch.library.custom_op("feather_ops_internal::dequantize_mxfp4", mutates_args=())
def _dequantize_op(data: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return native.binding().dequantize(data, scales, dtype, True)


@_dequantize_op.register_fake
def _(data, scales, dtype):
    return torch.empty((data.shape[0], data.shape[1] * 2), dtype=dtype, device=data.device)


def dequantize_mxfp4(data: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The values MXFP4 rows stand for, rounded once to `dtype` (exact in fp32 and, for scales from 2^-125 on, in bf16)."""
    out = NotImplemented if torch.compiler.is_compiling() else native.binding().dequantize(data, scales, dtype)
    return _dequantize_op(data, scales, dtype) if out is NotImplemented else out


def prepack_mxfp4_scales(scales: torch.Tensor) -> torch.Tensor:
    """E8M0 scale bytes [R, K/32] as a checkpoint stores them -> [ceil(R/128), ceil(K/128), 512] tiles, padded with zeros."""
    if scales.dim() != 2 or scales.dtype not in SCALE_DTYPES:
        raise RuntimeError(f"scales must be a 2D tensor of E8M0 bytes [rows, K/32] (uint8 or float8_e8m0fnu), got {scales.dtype} {list(scales.shape)}")
    scales = scales.contiguous().view(torch.uint8)
    rows, blocks = scales.shape
    tr, tk, _ = _tiles(rows, blocks * 32)
    full = torch.zeros((tr * 128, tk * 4), dtype=torch.uint8, device=scales.device)
    full[:rows, :blocks] = scales
    return full.view(tr, 4, 32, tk, 4).permute(0, 3, 2, 1, 4).reshape(tr, tk, 512).contiguous()


def unprepack_mxfp4_scales(scales: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """The inverse of `prepack_mxfp4_scales`: tiles -> [rows, K/32]."""
    if k <= 0 or k % 32 != 0 or tuple(scales.shape) != _tiles(rows, k):
        raise RuntimeError(f"scales {list(scales.shape)} are not the tiles of {rows} x {k}")
    tr, tk, _ = scales.shape
    return scales.view(tr, tk, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tr * 128, tk * 4)[:rows, : k // 32].contiguous()


# ------------------------------------------------------------------------------------------------
# product
# ------------------------------------------------------------------------------------------------
@torch.library.custom_op("feather_ops_internal::scaled_mm_mxfp4", mutates_args=())
def _mm_op(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, bias: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor:
    return native.binding().mm(a, a_scales, b, b_scales, bias, out_dtype, None)


@_mm_op.register_fake
def _(a, a_scales, b, b_scales, bias, out_dtype):
    return torch.empty((a.shape[0], b.shape[0]), dtype=out_dtype, device=a.device)


def scaled_mm_mxfp4(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, bias: torch.Tensor | None = None,
                    out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """round(a @ b^T + bias): a [M, K] and b [N, K] in MXFP4 (`quantize_mxfp4`), bias [N] of out_dtype, result [M, N] fp16 / bf16."""
    out = NotImplemented if torch.compiler.is_compiling() else native.binding().mm(a, a_scales, b, b_scales, bias, out_dtype)
    return _mm_op(a, a_scales, b, b_scales, bias, out_dtype) if out is NotImplemented else out


@torch.library.custom_op("feather_ops_internal::linear_mxfp4", mutates_args=())
def _linear_op(x: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, bias: torch.Tensor | None, out_dtype: torch.dtype | None) -> torch.Tensor:
    return native.binding().linear(x, b, b_scales, bias, out_dtype, True)


@_linear_op.register_fake
def _(x, b, b_scales, bias, out_dtype):
    dtype = out_dtype if out_dtype is not None else (torch.bfloat16 if x.dtype == torch.float32 else x.dtype)
    return torch.empty((*x.shape[:-1], b.shape[0]), dtype=dtype, device=x.device)


def linear_mxfp4(x: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., K] fp32 / bf16 / fp16 -> [..., N]: the rows of x are quantised to MXFP4 and multiplied with the weight b [N, K].
    out_dtype: fp16 or bf16; by default x's dtype if that is one of them, else bf16."""
    out = NotImplemented if torch.compiler.is_compiling() else native.binding().linear(x, b, b_scales, bias, out_dtype)
    return _linear_op(x, b, b_scales, bias, out_dtype) if out is NotImplemented else out


class MXFP4Linear:
    """y = round(x @ W^T + bias) with the weight held as MXFP4; x is a tensor, quantised on the way in, or the pair (data, scales) that
    `quantize_mxfp4` and `gated_residual_norm(..., packed=True)` give."""

    def __init__(self, weight, bias=None, device=None):
        """weight [N, K] fp32 / bf16 / fp16, bias [N] or None; both are taken to `device` (default: the weight's)."""
        device = weight.device if device is None else device
        self.data, self.scales = quantize_mxfp4(weight.to(device))
        self.bias = None if bias is None else bias.to(device).contiguous()

    def __call__(self, x, out_dtype=torch.bfloat16):
        if isinstance(x, tuple):
            return scaled_mm_mxfp4(*x, self.data, self.scales, self.bias, out_dtype)
        return linear_mxfp4(x, self.data, self.scales, self.bias, out_dtype)
