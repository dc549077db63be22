"""The norms before and after a block fused with its gate and its residual: one pass over the rows (`feather_gated_norm`).

    z = y                      or, with post_norm, norm(y) * post_weight
    r = x + residual_scale * gate * z
    h = (norm(r) * weight + bias) * (1 + scale) + shift

r is the residual stream after the block, h what the next block's first linear reads; with `packed=True` h leaves as the MXFP4
operand of that linear.  Statistics are fp32 and taken over r before it is rounded.

The operator serves: it has no backward pass, and a call with an input that requires a gradient is refused while gradients are
enabled.  The reference has no norm; a model around it runs these as five to ten elementwise passes.
"""

import torch

from .b200 import native

_CODE = {torch.float32: native.SRC_FP32, torch.bfloat16: native.SRC_BF16, torch.float16: native.SRC_FP16}
_KINDS = {"rms": 0, "layer": 1}
MAX_COLS = 16384


def _rows(t, cols):
    """t as [rows, cols] with unit column stride, without a copy where its layout allows."""
    t = t if t.dim() == 2 else t.reshape(-1, cols)
    if t.stride(1) != 1 and cols > 1 or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t


def _vector(t, name, cols, device):
    if t is None:
        return None
    if t.dtype not in _CODE:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16")
    if t.device != device:
        raise RuntimeError(f"{name} must be on the same device as x")
    if t.numel() != cols or not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous with {cols} elements")
    return t


def _modulation(t, name, lead, cols, device):
    """[cols], or x's shape with a number of trailing token dimensions of size 1 -> ([G, cols] rows, token rows that share one of them)."""
    if t is None:
        return None, 1
    if t.dtype not in _CODE:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16")
    if t.device != device:
        raise RuntimeError(f"{name} must be on the same device as x")
    if t.dim() == 0 or t.shape[-1] != cols or t.dim() > len(lead) + 1:
        raise RuntimeError(f"{name} must end in {cols} elements and have no more dimensions than x, got {list(t.shape)}")
    total = 1
    for d in lead:
        total *= d
    own = (1,) * (len(lead) + 1 - t.dim()) + tuple(t.shape[:-1])
    groups, i = 1, 0
    while i < len(lead) and own[i] == lead[i]:
        groups *= lead[i]
        i += 1
    if any(d != 1 for d in own[i:]):
        raise RuntimeError(f"{name} {list(t.shape)} must have x's leading dimensions {list(lead)}, those after some point replaced by 1")
    return _rows(t.reshape(groups, cols), cols), max(1, total // max(1, groups))


def _impl(x, y, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift, kind, eps, out_dtype, want_norm, packed):
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    if x.dtype not in _CODE:
        raise RuntimeError("x must be float32, bfloat16 or float16")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError("x must have at least one element in its last dimension")
    if kind not in _KINDS:
        raise RuntimeError("kind must be 'rms' or 'layer'")
    if not eps >= 0.0:
        raise RuntimeError("eps must not be negative")
    cols, lead, dev = x.shape[-1], tuple(x.shape[:-1]), x.device
    if cols > MAX_COLS:
        raise RuntimeError(f"the last dimension must be at most {MAX_COLS}, got {cols}")
    if y is None:
        if gate is not None or post_norm or post_weight is not None:
            raise RuntimeError("gate, post_norm and post_weight need y")
        if not want_norm:
            raise RuntimeError("without y there is only the norm to compute")
    else:
        if y.dtype not in _CODE:
            raise RuntimeError("y must be float32, bfloat16 or float16")
        if y.device != dev:
            raise RuntimeError("y must be on the same device as x")
        if y.shape != x.shape:
            raise RuntimeError(f"y must have x's shape {list(x.shape)}, got {list(y.shape)}")
        if post_weight is not None and not post_norm:
            raise RuntimeError("post_weight needs post_norm")
    if not want_norm and (weight is not None or bias is not None or scale is not None or shift is not None or packed):
        raise RuntimeError("weight, bias, scale, shift and packed belong to the norm that want_norm=False leaves out")
    if out_dtype is None:
        out_dtype = x.dtype if x.dtype != torch.float32 else (y.dtype if y is not None else x.dtype)
        if packed and out_dtype == torch.float32:
            out_dtype = torch.bfloat16
    if out_dtype not in _CODE:
        raise RuntimeError("out_dtype must be float32, bfloat16 or float16")
    if packed:
        if cols % 32 != 0:
            raise RuntimeError(f"an MXFP4 result needs a last dimension that is a multiple of 32, got {cols}")
        if out_dtype == torch.float32:
            raise RuntimeError("an MXFP4 result is rounded to out_dtype first: float16 or bfloat16")

    a = native.NormArgs()
    x2 = _rows(x, cols)
    rows = x2.shape[0]
    y2 = _rows(y, cols) if y is not None else None
    weight, bias, post_weight = (_vector(t, name, cols, dev) for t, name in ((weight, "weight"), (bias, "bias"), (post_weight, "post_weight")))
    gate, a.gate_rows = _modulation(gate, "gate", lead, cols, dev)
    scale, a.scale_rows = _modulation(scale, "scale", lead, cols, dev)
    shift, a.shift_rows = _modulation(shift, "shift", lead, cols, dev)
    if packed:
        # the packed form reads whole vectors only: rows that are not 16-byte aligned are copied
        def aligned(t):
            return t if t is None or (t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or t.dim() == 1 or t.stride(0) * t.element_size() % 16 == 0)) else t.clone(memory_format=torch.contiguous_format)

        x2, y2, weight, bias, post_weight, gate, scale, shift = (aligned(t) for t in (x2, y2, weight, bias, post_weight, gate, scale, shift))
    r = torch.empty(x.shape, dtype=x.dtype, device=dev) if y is not None else None
    h = h_scales = None
    if want_norm:
        if packed:
            h = torch.empty((rows, cols // 2), dtype=torch.uint8, device=dev)
            h_scales = torch.empty(((rows + 127) // 128, (cols + 127) // 128, 512), dtype=torch.uint8, device=dev)
        else:
            h = torch.empty(x.shape, dtype=out_dtype, device=dev)
    if rows:
        a.rows, a.cols = rows, cols
        a.x, a.x_dtype, a.ldx = x2.data_ptr(), _CODE[x.dtype], x2.stride(0)
        a.ldr = a.ldh = cols
        a.residual_scale, a.eps, a.kind, a.post_norm = residual_scale, eps, _KINDS[kind], 1 if post_norm else 0
        if y2 is not None:
            a.y, a.y_dtype, a.ldy, a.r = y2.data_ptr(), _CODE[y.dtype], y2.stride(0), r.data_ptr()
        if h is not None:
            a.h, a.h_dtype = h.data_ptr(), _CODE[out_dtype]
        if h_scales is not None:
            a.h_scales = h_scales.data_ptr()
        if weight is not None:
            a.weight, a.weight_dtype = weight.data_ptr(), _CODE[weight.dtype]
        if bias is not None:
            a.bias, a.bias_dtype = bias.data_ptr(), _CODE[bias.dtype]
        if post_weight is not None:
            a.post_weight, a.post_weight_dtype = post_weight.data_ptr(), _CODE[post_weight.dtype]
        if gate is not None:
            a.gate, a.gate_dtype, a.gate_ld = gate.data_ptr(), _CODE[gate.dtype], gate.stride(0)
        if scale is not None:
            a.scale, a.scale_dtype, a.scale_ld = scale.data_ptr(), _CODE[scale.dtype], scale.stride(0)
        if shift is not None:
            a.shift, a.shift_dtype, a.shift_ld = shift.data_ptr(), _CODE[shift.dtype], shift.stride(0)
        native.gated_norm(a, dev)
    return (x if r is None else r), ((h, h_scales) if packed else h)


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
    if torch.is_grad_enabled():
        for t in (x, y, gate, post_weight, weight, bias, scale, shift):
            if t is not None and t.requires_grad:
                raise RuntimeError("gated_residual_norm has no backward pass: detach the inputs or call under torch.no_grad()")
    return _impl(x, y, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift, kind, eps, out_dtype, want_norm, packed)
