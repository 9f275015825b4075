"""Serving in 8 bits: products of int8 codes with a scale for each token and
each output channel, and the deformable convolution on such products.

A row ``x`` is kept as ``codes = round(x / scale)`` with ``scale = max|x| / 127``;
the sums of the products of codes are exact, the scales and the bias are
applied to them in fp32.  In a deformable convolution the row is the sampled
column of one output pixel (and group).  Forward only; no reference
counterpart.
"""
from __future__ import annotations

import copy
from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from .module import DeformConv2d, DeformConv2dPack
from .ops import MASK_LOGITS, _ops, _pair
from .optim import _cuda_only, _no_grad_only


def quantize_int8(x: Tensor) -> Tuple[Tensor, Tensor]:
    """8-bit codes of the rows of ``x`` (..., K) and their float32 scales (...).

    ``scale = max|x| / 127``, ``code = x / scale`` rounded to the nearest whole
    number (ties to even); a row of zeros gets scale 0.  A row with NaN or an
    infinity gets that as its scale and zeros, so that its products are NaN.
    A weight (outC, ...) is quantised as
    ``quantize_int8(weight.detach().flatten(1))``.  Not differentiable.
    """
    _cuda_only("x", "quantize_int8", x)
    _no_grad_only("quantize_int8", x)
    return _ops().quantize_int8.default(x)


def int8_linear(x: Tensor, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor] = None,
                *, x_scale: Optional[Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``x @ weight.T`` in 8 bits: x (..., in), weight int8 (out, in).

    ``x`` is int8 with ``x_scale`` (...), or floating and coded inside the call
    as by :func:`quantize_int8`.  ``out_dtype`` defaults to ``x``'s type
    (float32 for int8).  Rows of a multiple of 16 features are read where they
    lie; others, and operands off a 16-byte boundary, are copied first.  At
    most 131071 features.
    """
    _cuda_only("x", "int8_linear", x)
    _no_grad_only("int8_linear", x, weight_scale, bias, x_scale)
    return _ops().int8_linear.default(x, weight, weight_scale, bias, x_scale, out_dtype)


def deform_conv2d_int8(input: Tensor, offset: Tensor, weight: Tensor, weight_scale: Tensor,
                       bias: Optional[Tensor] = None, stride=(1, 1), padding=(0, 0),
                       dilation=(1, 1), mask: Optional[Tensor] = None, *,
                       mask_logits: bool = False,
                       out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """:func:`deform_conv2d` with an int8 weight (outC, C/groups, kh, kw).

    ``weight_scale`` holds a float32 scale for each output channel; a
    channels-last weight is read where it lies, another is laid out anew in
    every call.  Each output pixel's sampled column is coded as by
    :func:`quantize_int8` (for each convolution group), but times one reciprocal
    of its scale: a value within that rounding of the middle of two codes may
    take the other.  input, offset and mask share one of float32, bfloat16 and
    float16; ``out_dtype`` defaults to it.  ``mask_logits`` as in
    :func:`deform_conv2d_ex`.

    A layer of hundreds of channels takes about the time of
    :func:`deform_conv2d` in 16 bits, with half of the weight's bytes; groups of
    a few channels are several times slower than there.
    """
    stride, padding, dilation = _pair(stride), _pair(padding), _pair(dilation)
    _cuda_only("input", "deform_conv2d_int8", input)
    _no_grad_only("deform_conv2d_int8", input, offset, weight_scale, bias, mask)
    shape = weight.shape
    if len(shape) != 4 or shape[1] == 0:
        raise RuntimeError("weight must be 4-D (outC, C/groups, kh, kw) with C/groups > 0")
    groups = input.shape[1] // shape[1]
    deformable_groups = offset.shape[1] // (2 * shape[2] * shape[3])
    return _ops().deform_conv2d_int8.default(
        input, weight, weight_scale, offset, mask, bias, stride[0], stride[1], padding[0],
        padding[1], dilation[0], dilation[1], groups, deformable_groups, out_dtype,
        MASK_LOGITS if mask_logits and mask is not None else 0)


class Int8DeformConv2d(nn.Module):
    """A trained :class:`DeformConv2d` or :class:`DeformConv2dPack` in 8 bits
    (:meth:`from_float`): the codes and scales of its weight as buffers, copies
    of its bias and of a pack's ``conv_offset``, which stays floating and asks
    for no gradient.  Inputs that ask for one are refused."""

    def __init__(self, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor], stride,
                 padding, dilation, conv_offset: Optional[nn.Module] = None,
                 deformable_groups: int = 1, modulated: bool = True):
        super().__init__()
        # channels last, the order the kernels sample in
        self.register_buffer("weight", weight.contiguous(memory_format=torch.channels_last))
        self.register_buffer("weight_scale", weight_scale)
        self.register_buffer("bias", bias)
        self.stride, self.padding, self.dilation = _pair(stride), _pair(padding), _pair(dilation)
        self.conv_offset = conv_offset
        self.deformable_groups = deformable_groups
        self.modulated = modulated

    @classmethod
    def from_float(cls, module: DeformConv2d) -> "Int8DeformConv2d":
        """The module's weight quantised on its device (CUDA)."""
        w = module.weight.detach()
        codes, scale = quantize_int8(w.flatten(1))
        bias = None if module.bias is None else module.bias.detach().clone()
        pack = isinstance(module, DeformConv2dPack)
        # its own: .half() here, or a step of the module's training, stays apart
        conv_offset = copy.deepcopy(module.conv_offset).requires_grad_(False) if pack else None
        return cls(codes.view(w.shape), scale, bias, module.stride, module.padding,
                   module.dilation, conv_offset,
                   module.deformable_groups if pack else 1, module.modulated if pack else True)

    def _apply(self, fn, *args, **kwargs):
        # .half() and the like leave the scales in float32
        scale = self.weight_scale
        super()._apply(fn, *args, **kwargs)
        if self.weight_scale.dtype != scale.dtype:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def forward(self, input: Tensor, offset: Optional[Tensor] = None,
                mask: Optional[Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> Tensor:
        _no_grad_only("Int8DeformConv2d", input, offset, mask)
        logits = False
        if self.conv_offset is not None:
            if offset is not None or mask is not None:
                raise TypeError("a pack predicts its own offset and mask")
            om = self.conv_offset(input)
            taps = self.deformable_groups * self.weight.shape[-2] * self.weight.shape[-1]
            offset, logits = om[:, :2 * taps], self.modulated
            mask = om[:, 2 * taps:] if self.modulated else None
        elif offset is None:
            raise TypeError("offset is needed")
        return deform_conv2d_int8(input, offset, self.weight, self.weight_scale, self.bias,
                                  self.stride, self.padding, self.dilation, mask,
                                  mask_logits=logits, out_dtype=out_dtype)

    def extra_repr(self) -> str:
        o, c, kh, kw = self.weight.shape
        return (f"{o} x {c} x {kh} x {kw}, stride={self.stride}, padding={self.padding}, "
                f"dilation={self.dilation}, bias={self.bias is not None}")
