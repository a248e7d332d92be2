"""Projections with 4-bit weights over torch device tensors (hx_w4_*).

A weight [out_features, in_features] is kept as 4-bit codes with an fp16 scale,
and optionally a 4-bit zero point, for every `group` (32, 64 or 128)
consecutive inputs of a row:  w = scale * (code - zero),  zero = 8 if not given.
"""
from __future__ import annotations

import torch

from ._lib import HX_FP16, HX_FP32, check, load
from .kv import _addr, _need_device, _need_shape, _on_stream, _ptr, _raw_stream, _stream, _used_on


class W4Weight:
    """A 4-bit weight, laid out on the device for w4_linear."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor,
                 zeros: torch.Tensor | None = None, stream=None):
        """codes: uint8 [out, in], one code (0..15) per byte; scales: fp16
        [out, in/group]; zeros: uint8 [out, in/group] (0..15) or None.  The
        group size follows from the shapes; the arguments are not kept."""
        _need_device(codes, scales, zeros)
        if codes.dim() != 2 or scales.dim() != 2 or codes.shape[0] != scales.shape[0]:
            raise ValueError("codes must be [out, in] and scales [out, in/group]")
        self.out_features, self.in_features = codes.shape
        self.group = self.in_features // max(1, scales.shape[1])
        if self.group * scales.shape[1] != self.in_features:
            raise ValueError(f"{scales.shape[1]} groups do not divide {self.in_features} inputs")
        self.has_zeros = zeros is not None
        _need_shape("codes", codes, (torch.uint8,), codes.numel())
        _need_shape("scales", scales, (torch.float16,), scales.numel())
        if zeros is not None:
            _need_shape("zeros", zeros, (torch.uint8,), scales.numel())
        nbytes = int(load().hx_w4_packed_bytes(self.out_features, self.in_features, self.group,
                                               int(self.has_zeros)))
        with _on_stream(stream):
            self.packed = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=codes.device)
        check(load().hx_w4_pack(_ptr(codes), _ptr(scales), _ptr(zeros), self.out_features,
                                self.in_features, self.group, _ptr(self.packed), nbytes,
                                _stream(stream)), "w4 pack")
        _used_on(stream, codes, scales, zeros)

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 128, stream=None) -> "W4Weight":
        """A finite fp16 weight [out, in] rounded to 4 bits (hx_w4_quantize)."""
        codes, scales = w4_quantize(weight, group, stream=stream)
        return cls(codes, scales, stream=stream)


def w4_quantize(weight: torch.Tensor, group: int = 128, stream=None):
    """(codes uint8 [out, in], scales fp16 [out, in/group]) of a finite fp16
    weight: scale = max|w| / 7 over the group, code = 8 + round(w / scale)."""
    _need_device(weight)
    if weight.dim() != 2:
        raise ValueError("weight must be [out, in]")
    _need_shape("weight", weight, (torch.float16,), weight.numel())
    o, k = weight.shape
    if group < 1 or k % group:
        raise ValueError(f"groups of {group} do not divide {k} inputs")
    with _on_stream(stream):
        codes = torch.empty((o, k), dtype=torch.uint8, device=weight.device)
        scales = torch.empty((o, k // group), dtype=torch.float16, device=weight.device)
    check(load().hx_w4_quantize(_ptr(weight), o, k, group, _ptr(codes), _ptr(scales),
                                _stream(stream)), "w4 quantize")
    _used_on(stream, weight)
    return codes, scales


def w4_linear(x: torch.Tensor, weight: W4Weight, *, bias: torch.Tensor | None = None,
              out: torch.Tensor | None = None, out_dtype=torch.float16,
              stream=None) -> torch.Tensor:
    """x [n, in] (fp16) times the weight's transpose, plus bias (fp16 [out]):
    [n, out] in fp16 or fp32, accumulated in fp32 (hx_w4_linear).  Meant for
    the few rows of a decode step."""
    _need_device(x, weight.packed, bias, out)
    shape = x.shape
    if len(shape) != 2 or shape[1] != weight.in_features:
        raise ValueError(f"x of shape {tuple(shape)} for {weight.in_features} inputs")
    n = shape[0]
    _need_shape("x", x, (torch.float16,), n * weight.in_features)
    if bias is not None:
        _need_shape("bias", bias, (torch.float16,), weight.out_features)
    if out is None:
        with _on_stream(stream):
            out = torch.empty((n, weight.out_features), dtype=out_dtype, device=x.device)
    _need_shape("out", out, (torch.float16, torch.float32), n * weight.out_features)
    check(load().hx_w4_linear(x.data_ptr(), n, weight.in_features, weight.packed.data_ptr(),
                              weight.packed.numel(), weight.out_features, weight.group,
                              weight.has_zeros, _addr(bias), out.data_ptr(),
                              HX_FP32 if out.dtype == torch.float32 else HX_FP16,
                              _raw_stream(stream)), "w4 linear")
    _used_on(stream, x, weight.packed, bias, out)
    return out
