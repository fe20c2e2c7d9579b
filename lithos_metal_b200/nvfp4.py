"""Weights in the microscaled 4-bit format (NVFP4): 4-bit codes, an e4m3 scale for every 16 of a row's columns, one float32 scale for all.

``quantize_nvfp4`` makes one from a BF16 or FP32 matrix, ``Nvfp4Weight(codes, scales, scale)`` wraps the tensors of a checkpoint; ``lm_head`` takes
it in the place of a BF16 weight (the reference's weight formats: monolith/formats)."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from .sampler import _dtype_code, _row_stride

BLOCK = 16                               # columns that share a scale


def _padded_scales(rows: int, blocks: int, device: torch.device) -> torch.Tensor:
    """uint8 [rows, blocks] whose rows start at multiples of 16 bytes."""
    return torch.empty(rows, (blocks + 15) // 16 * 16, dtype=torch.uint8, device=device)[:, :blocks]


class Nvfp4Weight:
    """A matrix [rows, cols] in the 4-bit format: ``codes`` uint8 [rows, cols / 2] (the even column in the low nibble), ``scales`` float8_e4m3fn (or
    uint8, the same bytes) [rows, cols / 16], ``scale`` float32 with one element; CUDA tensors on one device, unit stride along a row. Element (r, c) is
    e2m1(code) * scales[r, c // 16] * scale. (Scales whose rows do not start at multiples of 16 bytes are copied once, to rows padded to that.) A slice of rows, ``weight[lo:hi]``, is a view (a shard of a vocabulary)."""

    __slots__ = ("codes", "scales", "scale")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, scale: torch.Tensor) -> None:
        if not all(isinstance(t, torch.Tensor) and t.is_cuda for t in (codes, scales, scale)):
            raise RuntimeError("lithos_metal_b200 runs on CUDA tensors only (there is no CPU path)")
        if codes.dim() != 2 or codes.dtype != torch.uint8 or codes.shape[1] % (BLOCK // 2) != 0:
            raise ValueError("Nvfp4Weight: codes uint8 [rows, cols / 2], cols a multiple of 16")
        if scales.dtype not in (torch.uint8, torch.float8_e4m3fn) or scales.shape != (codes.shape[0], codes.shape[1] * 2 // BLOCK):
            raise ValueError("Nvfp4Weight: scales float8_e4m3fn (or uint8) [rows, cols / 16]")
        if scale.dtype != torch.float32 or scale.numel() != 1:
            raise ValueError("Nvfp4Weight: scale float32 with one element")
        if scales.device != codes.device or scale.device != codes.device:
            raise ValueError("Nvfp4Weight: tensors on one device")
        if (codes.shape[1] > 1 and codes.stride(1) != 1) or (scales.shape[1] > 1 and scales.stride(1) != 1):
            raise ValueError("Nvfp4Weight: the rows must be contiguous")
        scales = scales.view(torch.uint8)
        if scales.numel() and (scales.data_ptr() % 16 or (scales.shape[0] > 1 and scales.stride(0) % 16)):
            scales = _padded_scales(*scales.shape, scales.device).copy_(scales)
        self._hold(codes, scales, scale)

    def _hold(self, *tensors: torch.Tensor) -> "Nvfp4Weight":
        for name, t in zip(self.__slots__, tensors):
            object.__setattr__(self, name, t)
        return self

    def __setattr__(self, name: str, value: object) -> None:                 # (they were checked together; what they hold may change)
        raise AttributeError("Nvfp4Weight: its tensors stay the same; make another weight")

    def __reduce__(self):
        return Nvfp4Weight, (self.codes, self.scales, self.scale)

    @property
    def shape(self) -> Tuple[int, int]:
        return self.codes.shape[0], self.codes.shape[1] * 2

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def __getitem__(self, rows: slice) -> "Nvfp4Weight":
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise TypeError("Nvfp4Weight: a slice of consecutive rows")
        return Nvfp4Weight(self.codes[rows], self.scales[rows], self.scale)

    def dequantize(self, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The float32 values [rows, cols]."""
        r = _lib.host().dequantize_nvfp4(self.codes, self.scales, self.scale, out)
        if r is not None:
            return r
        rows, cols = self.shape
        if out is None:
            out = torch.empty(rows, cols, dtype=torch.float32, device=self.device)
        if out.shape != (rows, cols) or out.dtype != torch.float32 or out.device != self.device or (cols > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < cols):
            raise ValueError("dequantize: out must be [rows, cols] float32 on the same device")
        a = _lib.DequantizeNvfp4Args()
        a.struct_size = C.sizeof(a)
        a.codes, a.codes_stride, a.scales, a.scales_stride, a.scale = (self.codes.data_ptr(), _row_stride(self.codes), self.scales.data_ptr(), _row_stride(self.scales),
                                                                       self.scale.data_ptr())
        a.rows, a.cols, a.out, a.out_stride = rows, cols, out.data_ptr(), _row_stride(out)
        a.stream = torch.cuda.current_stream(self.device).cuda_stream
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().lm_dequantize_nvfp4(C.byref(a)), "lm_dequantize_nvfp4")
        return out


def quantize_nvfp4(x: torch.Tensor, scale: Optional[torch.Tensor] = None) -> Nvfp4Weight:
    """``x`` [rows, cols] (bfloat16 or float32, CUDA, cols a multiple of 16) in the 4-bit format. ``scale`` (float32, one element, on the same device) is taken as given;
    without it, it is the largest finite magnitude divided by 2688. Every rounding is to nearest, ties to even, of the real quotient: the codes do not depend on the
    arithmetic. A block of 16 that holds a NaN or an infinity becomes NaN. Asynchronous on the current stream."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("lithos_metal_b200 runs on CUDA tensors only (there is no CPU path)")
    r = _lib.host().quantize_nvfp4(x, scale)
    if r is not None:
        return Nvfp4Weight.__new__(Nvfp4Weight)._hold(*r)                     # (tensors of the right kind: nothing to check)
    if x.dim() != 2 or x.shape[1] % BLOCK != 0:
        raise ValueError("quantize_nvfp4: x must be [rows, cols], cols a multiple of 16")
    dtype = _dtype_code(x)
    if scale is not None and (scale.dtype != torch.float32 or scale.numel() != 1 or scale.device != x.device):
        raise ValueError("quantize_nvfp4: scale float32 with one element on the same device")
    rows, cols = x.shape
    if x.stride(1) != 1 or (rows > 1 and x.stride(0) < cols):
        x = x.contiguous()
    with torch.cuda.device(x.device):
        codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device=x.device)
        scales = _padded_scales(rows, cols // BLOCK, x.device)
        a = _lib.QuantizeNvfp4Args()
        a.struct_size = C.sizeof(a)
        if scale is None:
            scale = torch.ones(1, dtype=torch.float32, device=x.device) if x.numel() == 0 else torch.empty(1, dtype=torch.float32, device=x.device)
            amax = torch.empty(1, dtype=torch.int32, device=x.device)
            a.find_scale, a.amax = 1, amax.data_ptr()
        a.dtype, a.x, a.rows, a.cols, a.row_stride = dtype, x.data_ptr(), rows, cols, _row_stride(x)
        a.scale, a.codes, a.codes_stride, a.scales, a.scales_stride = scale.data_ptr(), codes.data_ptr(), _row_stride(codes), scales.data_ptr(), _row_stride(scales)
        a.stream = torch.cuda.current_stream(x.device).cuda_stream
        _lib.check(_lib.lib().lm_quantize_nvfp4(C.byref(a)), "lm_quantize_nvfp4")
    return Nvfp4Weight(codes, scales, scale)
