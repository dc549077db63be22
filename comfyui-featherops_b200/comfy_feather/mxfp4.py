"""MXFP4 weights of the ComfyUI operator: `feather_ops(..., weight_format="mxfp4")` keeps a Linear's weight as MXFP4
(kernel/mxfp4.py: 4-bit elements, one power-of-two scale for every 32 along K) in a quantised-tensor layout of its own, beside the
reference's fp8e5m2 layout (comfy_feather/quant.py:77-159 there; it has no 4-bit format).

    FeatherMXFP4Layout                  quantize / dequantize / get_plain_tensors / state_dict_tensors
    make_mxfp4_weight                   loader: a float weight is quantised (e5m2 and other scaled checkpoints through fp32), a weight that
                                        is MXFP4 already (uint8 [N, K/2] with E8M0 scales [N, K/32]) only has its scales laid out
    quantize_mxfp4_weight / is_mxfp4_weight / get_mxfp4_plain_tensors

Rounding is to nearest whatever the seed.  As in quant.py there is no CPU implementation: a tensor in host memory is copied to the
current CUDA device, processed there, and the result is returned on the tensor's own device.
"""

from dataclasses import dataclass

import torch
from comfy.quant_ops import QuantizedLayout, QuantizedTensor, register_layout_class

from ..kernel import mxfp4
from .quant import FeatherFP8E5M2PackedParams, _compute_device

FEATHER_MXFP4_LAYOUT = "FeatherMXFP4Layout"

_SOURCES = (torch.float32, torch.bfloat16, torch.float16)


@dataclass(frozen=True)
class FeatherMXFP4Params(FeatherFP8E5M2PackedParams):
    """`scale` is the uint8 tiles of the block scales; moved, cloned and overwritten like the packed fp8 weight's scale."""


def _quantize(x):
    if x.ndim != 2:
        raise ValueError(f"MXFP4 weights require a 2D tensor, got {x.ndim}D")
    if x.shape[1] % 32 != 0:
        raise ValueError(f"MXFP4 weights require K divisible by 32, got {tuple(x.shape)}")
    if x.dtype not in _SOURCES:
        raise TypeError(f"cannot quantise a {x.dtype} weight (expected float32, bfloat16 or float16)")
    data, scales = mxfp4.quantize_mxfp4(x.detach().to(_compute_device(x)))
    return data.to(x.device), scales.to(x.device)


class FeatherMXFP4Layout(QuantizedLayout):
    Params = FeatherMXFP4Params

    @classmethod
    def quantize(cls, tensor, scale="recalculate", stochastic_rounding=0, inplace_ops=False):
        if not (scale is None or (isinstance(scale, str) and scale == "recalculate")):
            raise ValueError("MXFP4 scales follow from the blocks: scale must be 'recalculate'")
        data, scales = _quantize(tensor)
        return data, cls.Params(scale=scales, orig_dtype=tensor.dtype, orig_shape=tuple(tensor.shape))

    @classmethod
    def dequantize(cls, qdata, params):
        dev = _compute_device(qdata)
        return mxfp4.dequantize_mxfp4(qdata.to(dev), params.scale.to(dev), params.orig_dtype).to(qdata.device)

    @classmethod
    def get_plain_tensors(cls, qtensor):
        return qtensor._qdata, qtensor._params.scale

    @classmethod
    def state_dict_tensors(cls, qdata, params):
        n, k = params.orig_shape
        return {"": qdata, "_scale": mxfp4.unprepack_mxfp4_scales(params.scale, n, k)}


def scaled_weight(weight, scale):
    """The values of a scaled checkpoint weight, in fp32; scale: one element, or a column of one for each row of the weight."""
    weight = weight.to(torch.float32)
    if scale is None:
        return weight
    if scale.numel() == 1:
        scale = scale.reshape(())
    elif weight.ndim != 2 or tuple(scale.shape) != (weight.shape[0], 1):
        raise ValueError(f"the scale of a weight {tuple(weight.shape)} has one element or a column of one for each row, got {tuple(scale.shape)}")
    return weight * scale.to(device=weight.device, dtype=torch.float32)


def make_mxfp4_weight(weight, scale, orig_dtype):
    """The weight of a checkpoint as an MXFP4 `QuantizedTensor` that reads as `orig_dtype`."""
    if weight.ndim != 2:
        raise ValueError(f"MXFP4 weights require a 2D tensor, got {weight.ndim}D")
    if weight.dtype == torch.uint8:
        n, k = weight.shape[0], weight.shape[1] * 2
        if scale is None or scale.dtype not in mxfp4.SCALE_DTYPES or tuple(scale.shape) != (n, k // 32) or k % 32 != 0:
            raise ValueError(f"a packed MXFP4 weight {tuple(weight.shape)} needs E8M0 scale bytes (uint8 or float8_e8m0fnu) of shape {(n, k // 32)}")
        params = FeatherMXFP4Params(scale=mxfp4.prepack_mxfp4_scales(scale.to(weight.device)), orig_dtype=orig_dtype, orig_shape=(n, k))
        weight = weight.contiguous()
        if weight.data_ptr() % 16 != 0:                            # a view into a loader's buffer; the kernels need 16-byte alignment
            weight = weight.clone()
        return QuantizedTensor(weight, FEATHER_MXFP4_LAYOUT, params)
    if scale is not None or weight.dtype not in _SOURCES:
        weight = scaled_weight(weight, scale)
    data, scales = _quantize(weight)
    return QuantizedTensor(data, FEATHER_MXFP4_LAYOUT, FeatherMXFP4Params(scale=scales, orig_dtype=orig_dtype, orig_shape=tuple(weight.shape)))


def quantize_mxfp4_weight(weight):
    data, params = FeatherMXFP4Layout.quantize(weight)
    return QuantizedTensor(data, FEATHER_MXFP4_LAYOUT, params)


def is_mxfp4_weight(weight):
    return isinstance(weight, QuantizedTensor) and weight._layout_cls == FEATHER_MXFP4_LAYOUT


def get_mxfp4_plain_tensors(weight):
    if not is_mxfp4_weight(weight):
        raise TypeError(f"Expected {FEATHER_MXFP4_LAYOUT}, got {type(weight).__name__}")
    return FeatherMXFP4Layout.get_plain_tensors(weight)


register_layout_class(FEATHER_MXFP4_LAYOUT, FeatherMXFP4Layout)
