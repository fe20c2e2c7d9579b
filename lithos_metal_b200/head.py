"""The vocabulary projection of a decode step (the reference's ``lm_head`` op, monolith/nn/lm_head.py:50-60): BF16 logits of at
most 8 rows from the hidden states and the [vocab, hidden] weight, the final RMSNorm fused on the input. The logits are what
``sample`` / ``argmax`` / ``verify`` take next on the same stream."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Union

import torch

from . import _lib
from .nvfp4 import Nvfp4Weight
from .sampler import _row_stride


def lm_head(hidden: torch.Tensor, weight: Union[torch.Tensor, Nvfp4Weight], norm_weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6, one_plus: bool = True,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``bf16(x @ weightᵀ)`` with FP32 accumulation; ``x = hidden`` or, with ``norm_weight``, ``bf16(rms_norm(hidden) * (1 + norm_weight))``
    (``one_plus=False``: ``* norm_weight``), as monolith/nn/oracle.py:20-32 defines both. ``hidden`` [rows <= 8, H] and ``weight`` [V, H]
    bfloat16 CUDA tensors with unit stride along H; returns [rows, V] bfloat16. With an ``Nvfp4Weight`` [V, H] any number of rows (to 65,536), H a multiple of 64
    up to 12,736, the products with the weight's values exact."""
    if isinstance(weight, Nvfp4Weight):
        return _lm_head_nvfp4(hidden, weight, norm_weight, eps, one_plus, out)
    r = _lib.host().lm_head(hidden, weight, norm_weight, eps, one_plus, out)
    if r is not None:
        return r
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError("lm_head: hidden [rows, H] and weight [V, H]")
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16 or not hidden.is_cuda or weight.device != hidden.device:
        raise ValueError("lm_head: bfloat16 CUDA tensors on one device")
    rows, H = hidden.shape
    V = weight.shape[0]
    if rows > 8:
        raise ValueError("lm_head: at most 8 rows (a decode step)")
    if hidden.stride(1) != 1:
        hidden = hidden.contiguous()
    if weight.stride(1) != 1:
        raise ValueError("lm_head: the weight's rows must be contiguous")
    if norm_weight is not None:
        if norm_weight.shape != (H,) or norm_weight.dtype != torch.bfloat16 or norm_weight.device != hidden.device:
            raise ValueError("lm_head: norm_weight [H] bfloat16 on the same device")
        norm_weight = norm_weight.contiguous()
    logits = out if out is not None else torch.empty(rows, V, dtype=torch.bfloat16, device=hidden.device)
    if logits.shape != (rows, V) or logits.dtype != torch.bfloat16 or logits.stride(1) != 1 or logits.device != hidden.device:
        raise ValueError("lm_head: out must be [rows, V] bfloat16 on the same device")
    a = _lib.HeadArgs()
    a.struct_size = C.sizeof(_lib.HeadArgs)
    a.rows, a.hidden, a.hidden_stride = rows, hidden.data_ptr(), hidden.stride(0) if rows > 1 else H
    a.weight, a.weight_stride, a.hidden_dim, a.vocab = weight.data_ptr(), weight.stride(0) if V > 1 else H, H, V
    a.norm_weight = norm_weight.data_ptr() if norm_weight is not None else None
    a.eps, a.one_plus = float(eps), 1 if one_plus else 0
    a.logits, a.logits_stride = logits.data_ptr(), logits.stride(0) if rows > 1 else V
    a.stream = torch.cuda.current_stream(hidden.device).cuda_stream
    with torch.cuda.device(hidden.device):
        _lib.check(_lib.lib().lm_head(C.byref(a)), "lm_head")
    return logits


def _lm_head_nvfp4(hidden: torch.Tensor, weight: Nvfp4Weight, norm_weight: Optional[torch.Tensor], eps: float, one_plus: bool, out: Optional[torch.Tensor]) -> torch.Tensor:
    r = _lib.host().lm_head_nvfp4(hidden, weight.codes, weight.scales, weight.scale, norm_weight, eps, one_plus, out)
    if r is not None:
        return r
    V, H = weight.shape
    dev = weight.device
    if hidden.dim() != 2 or hidden.shape[1] != H or hidden.dtype != torch.bfloat16 or hidden.device != dev:
        raise ValueError("lm_head: hidden [rows, H] bfloat16 on the weight's device")
    rows = hidden.shape[0]
    if (H > 1 and hidden.stride(1) != 1) or (rows > 1 and hidden.stride(0) < H):
        hidden = hidden.contiguous()
    if norm_weight is not None:
        if norm_weight.shape != (H,) or norm_weight.dtype != torch.bfloat16 or norm_weight.device != dev:
            raise ValueError("lm_head: norm_weight [H] bfloat16 on the same device")
        norm_weight = norm_weight.contiguous()
    logits = out if out is not None else torch.empty(rows, V, dtype=torch.bfloat16, device=dev)
    if logits.shape != (rows, V) or logits.dtype != torch.bfloat16 or logits.device != dev or (V > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < V):
        raise ValueError("lm_head: out must be [rows, V] bfloat16 on the same device")
    L = _lib.lib()
    a = _lib.HeadNvfp4Args()
    a.struct_size = C.sizeof(a)
    a.rows, a.hidden, a.hidden_stride = rows, hidden.data_ptr(), _row_stride(hidden)
    a.codes, a.codes_stride, a.scales, a.scales_stride, a.scale = (weight.codes.data_ptr(), _row_stride(weight.codes), weight.scales.data_ptr(), _row_stride(weight.scales),
                                                                   weight.scale.data_ptr())
    a.hidden_dim, a.vocab = H, V
    a.norm_weight = norm_weight.data_ptr() if norm_weight is not None else None
    a.eps, a.one_plus = float(eps), 1 if one_plus else 0
    a.logits, a.logits_stride = logits.data_ptr(), _row_stride(logits)
    nbytes = L.lm_head_nvfp4_workspace_bytes(rows, H)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None      # (of the call: calls that overlap never share one)
    a.workspace, a.workspace_bytes = ws.data_ptr() if ws is not None else None, nbytes
    a.stream = torch.cuda.current_stream(dev).cuda_stream
    with torch.cuda.device(dev):
        _lib.check(L.lm_head_nvfp4(C.byref(a)), "lm_head_nvfp4")
    return logits
