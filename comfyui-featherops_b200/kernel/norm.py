"""The norms before and after a block fused with its gate and its residual: one pass over the rows (`feather_gated_norm`).

    z = y                      or, with post_norm, norm(y) * post_weight
    r = x + residual_scale * gate * z
    h = (norm(r) * weight + bias) * (1 + scale) + shift

r is the residual stream after the block, h what the next block's first linear reads; with `packed=True` h leaves as the MXFP4
operand of that linear.  Statistics are fp32 and taken over r before it is rounded.

The operator serves: it has no derivatives.  A call with an input that requires a gradient is refused while gradients are enabled, one with a
dual tensor of forward-mode differentiation always.  The reference has no norm; a model around it runs these as five to ten elementwise passes.
"""

import torch

from .b200 import native


@torch.library.custom_op("feather_ops_internal::gated_residual_norm", mutates_args=())
def _norm_op(
    x: torch.Tensor,
    y: torch.Tensor | None,
    gate: torch.Tensor | None,
    residual_scale: float,
    post_norm: bool,
    post_weight: torch.Tensor | None,
    weight: torch.Tensor | None,
    bias: torch.Tensor | None,
    scale: torch.Tensor | None,
    shift: torch.Tensor | None,
    kind: str,
    eps: float,
    out_dtype: torch.dtype,
    want_norm: bool,
    packed: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(r, h, scales of h); what a call does not ask for is empty, as is r without y."""
    r, h = native.binding().norm(x, y, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift, kind, eps, out_dtype, want_norm, packed, True)
    h, scales = h if packed else (h, x.new_empty((0,), dtype=torch.uint8))
    return r if y is not None else x.new_empty((0,)), h if h is not None else x.new_empty((0,), dtype=out_dtype), scales


@_norm_op.register_fake
def _(x, y, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift, kind, eps, out_dtype, want_norm, packed):
    cols = x.shape[-1]
    rows = x.numel() // cols
    r = torch.empty(x.shape, dtype=x.dtype, device=x.device) if y is not None else x.new_empty((0,))
    if packed:
        return r, x.new_empty((rows, cols // 2), dtype=torch.uint8), x.new_empty(((rows + 127) // 128, (cols + 127) // 128, 512), dtype=torch.uint8)
    return r, torch.empty(x.shape, dtype=out_dtype, device=x.device) if want_norm else x.new_empty((0,), dtype=out_dtype), x.new_empty((0,), dtype=torch.uint8)


def gated_residual_norm(x, y=None, gate=None, residual_scale=1.0, post_norm=False, post_weight=None, weight=None, bias=None, scale=None, shift=None, kind="rms", eps=1e-6,
                        out_dtype=None, want_norm=True, packed=False):
    """(r, h): the residual stream after a block and the normalised input of the next one.

    x [..., C] residual stream (fp32 / bf16 / fp16; r has its dtype), y the block's output of the same shape (any of the three).
    gate, scale, shift: [C], or x's leading dimensions with those after some point replaced by 1 ([B, 1, C] or [B, L, C] for
    x [B, L, C]); rows may be strided (a chunk of one projection).  weight, bias, post_weight: [C].  Each may have its own dtype.
    kind "rms" or "layer" holds for both norms.  Without y, r is x itself and h its norm.  want_norm=False returns (r, None).
    out_dtype: h's dtype (default: the 16-bit one of x and y, x's first).  packed=True: h is the pair (data, scales) that
    `quantize_mxfp4` gives for the [rows, C] h of out_dtype, bit for bit.
    """
    if not torch.compiler.is_compiling():
        out = native.binding().norm(x, y, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift, kind, eps, out_dtype, want_norm, packed)
        if out is not NotImplemented:
            return out
    if out_dtype is None:                                                   # through the dispatcher, for whoever watches it (kernel/mxfp4.py)
        out_dtype = x.dtype if x.dtype != torch.float32 or y is None else y.dtype
        if packed and out_dtype == torch.float32:
            out_dtype = torch.bfloat16
    r, h, scales = _norm_op(x, y, gate, float(residual_scale), post_norm, post_weight, weight, bias, scale, shift, kind, float(eps), out_dtype, want_norm, packed)
    return (x if y is None else r), ((h, scales) if packed else h if want_norm else None)
