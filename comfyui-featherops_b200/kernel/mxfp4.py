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

The operators serve: they have no backward pass, and a call with an input that requires a gradient is refused while gradients are
enabled.  The reference (fp8e5m2 weights, per-tensor scale) has no such format.
"""

import torch

from .b200 import native

_SOURCES = (torch.float32, torch.bfloat16, torch.float16)
_RESULTS = (torch.float16, torch.bfloat16)


def _no_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("MXFP4 operators have no backward pass: detach the inputs or call under torch.no_grad()")


def _tiles(rows, k):
    return ((rows + 127) // 128, (k + 127) // 128, 512)


def _check_packed(data, scales, what):
    """The checks of one MXFP4 operand; returns (rows, k)."""
    if data.dim() != 2 or data.dtype != torch.uint8:
        raise RuntimeError(f"{what} must be a uint8 [rows, K/2] tensor")
    rows, k = data.shape[0], data.shape[1] * 2
    if k == 0 or k % 32 != 0:
        raise RuntimeError(f"{what}: K must be a positive multiple of 32, got {k}")
    if scales.dtype != torch.uint8 or tuple(scales.shape) != _tiles(rows, k):
        raise RuntimeError(f"{what}_scales must be uint8 {list(_tiles(rows, k))} (prepack_mxfp4_scales lays [rows, K/32] bytes out), got {scales.dtype} {list(scales.shape)}")
    if not (data.is_cuda and scales.is_cuda):
        raise RuntimeError(f"{what} and its scales must be CUDA tensors")
    if scales.device != data.device:
        raise RuntimeError(f"{what}_scales must be on the same device as {what}")
    if not (data.is_contiguous() and scales.is_contiguous()):
        raise RuntimeError(f"{what} and its scales must be contiguous")
    if data.data_ptr() % 16 != 0 or scales.data_ptr() % 16 != 0:
        raise RuntimeError(f"{what} and its scales must be 16-byte aligned")
    return rows, k


# ------------------------------------------------------------------------------------------------
# format
# ------------------------------------------------------------------------------------------------
def _quantize_impl(x):
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    if x.dtype not in _SOURCES:
        raise RuntimeError(f"cannot quantise {x.dtype} (expected float32, bfloat16 or float16)")
    if x.dim() != 2 or x.shape[1] == 0 or x.shape[1] % 32 != 0:
        raise RuntimeError(f"MXFP4 needs a 2D tensor with K a positive multiple of 32, got {tuple(x.shape)}")
    rows, k = x.shape
    if x.stride(1) != 1 or (rows > 1 and x.stride(0) < k):
        x = x.contiguous()
    data = torch.empty((rows, k // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty(_tiles(rows, k), dtype=torch.uint8, device=x.device)
    if rows:
        native.mxfp4_quantize_into(x, data, scales)
    return data, scales


def _dequantize_impl(data, scales, dtype):
    if dtype not in _SOURCES:
        raise RuntimeError("dtype must be float32, bfloat16 or float16")
    rows, k = _check_packed(data, scales, "data")
    out = torch.empty((rows, k), dtype=dtype, device=data.device)
    if rows:
        native.mxfp4_dequantize_into(data, scales, out)
    return out


@torch.library.custom_op("feather_ops_internal::quantize_mxfp4", mutates_args=())
def _quantize_op(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _quantize_impl(x)


@_quantize_op.register_fake
def _(x):
    rows, k = x.shape
    return torch.empty((rows, k // 2), dtype=torch.uint8, device=x.device), torch.empty(_tiles(rows, k), dtype=torch.uint8, device=x.device)


def quantize_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [R, K] fp32 / bf16 / fp16 on the GPU, K % 32 == 0 -> (data uint8 [R, K/2], scales uint8 [ceil(R/128), ceil(K/128), 512]).
    Rows may be strided; a tensor whose columns are strided is copied first.  Scale bytes of rows past R are not written."""
    _no_grad(x)
    return _quantize_op(x) if torch.compiler.is_compiling() else _quantize_impl(x)


def dequantize_mxfp4(data: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The values MXFP4 rows stand for, rounded once to `dtype` (exact in fp32 and, for scales from 2^-125 on, in bf16)."""
    return _dequantize_impl(data, scales, dtype)


def prepack_mxfp4_scales(scales: torch.Tensor) -> torch.Tensor:
    """E8M0 scale bytes [R, K/32] as a checkpoint stores them -> [ceil(R/128), ceil(K/128), 512] tiles, padded with zeros."""
    if scales.dim() != 2 or scales.element_size() != 1:
        raise RuntimeError("scales must be a 2D tensor of bytes [rows, K/32]")
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
def _mm_impl(a, a_scales, b, b_scales, bias, out_dtype):
    if out_dtype not in _RESULTS:
        raise RuntimeError("out_dtype must be float16 or bfloat16")
    m, k = _check_packed(a, a_scales, "a")
    n, kb = _check_packed(b, b_scales, "b")
    if k != kb:
        raise RuntimeError(f"a and b must have the same K, got {k} and {kb}")
    if b.device != a.device:
        raise RuntimeError("b must be on the same device as a")
    if n == 0:
        raise RuntimeError("b must have at least one row")
    if bias is not None:
        if bias.device != a.device:
            raise RuntimeError("bias must be on the same device as a")
        if bias.dtype != out_dtype:
            raise RuntimeError("bias must have the out dtype")
        if bias.numel() != n or not bias.is_contiguous():
            raise RuntimeError("bias must be contiguous with N elements")
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    if m:
        native.mxfp4_mm_into(a, a_scales, b, b_scales, bias, out)
    return out


@torch.library.custom_op("feather_ops_internal::scaled_mm_mxfp4", mutates_args=())
def _mm_op(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, bias: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor:
    return _mm_impl(a, a_scales, b, b_scales, bias, out_dtype)


@_mm_op.register_fake
def _(a, a_scales, b, b_scales, bias, out_dtype):
    return torch.empty((a.shape[0], b.shape[0]), dtype=out_dtype, device=a.device)


def scaled_mm_mxfp4(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, bias: torch.Tensor | None = None,
                    out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """round(a @ b^T + bias): a [M, K] and b [N, K] in MXFP4 (`quantize_mxfp4`), bias [N] of out_dtype, result [M, N] fp16 / bf16."""
    _no_grad(bias)
    if torch.compiler.is_compiling():
        return _mm_op(a, a_scales, b, b_scales, bias, out_dtype)
    return _mm_impl(a, a_scales, b, b_scales, bias, out_dtype)


def linear_mxfp4(x: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., K] fp32 / bf16 / fp16 -> [..., N]: the rows of x are quantised to MXFP4 and multiplied with the weight b [N, K].
    out_dtype: fp16 or bf16; by default x's dtype if that is one of them, else bf16."""
    if x.dim() == 0:
        raise RuntimeError("x must have at least one dimension")
    if out_dtype is None:
        out_dtype = x.dtype if x.dtype in _RESULTS else torch.bfloat16
    data, scales = quantize_mxfp4(x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x)
    y = scaled_mm_mxfp4(data, scales, b, b_scales, bias, out_dtype)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[1])
