"""The logits' processing between the projection and the sampler: penalties for repeated tokens by request (repetition, presence, frequency), biases by
token, and grammar masks, in one launch. ``sample`` applies one repetition and presence penalty for the whole batch by itself; what differs by request, counts or is
masked goes through :func:`process_logits` first."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from .sampler import Knob, _check_logits, _dtype_code, _knob, _row_stride


def _converted(t: torch.Tensor, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """`t` as `dtype` on the device. What int32 does not hold becomes its nearest end, which is as much outside every vocabulary, length and number of masks; a plain conversion would keep the low bits, and
    2^32 + 5 would name token 5."""
    if dtype == torch.int32 and t.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8, torch.bool):
        wide = t.to(device=device, dtype=torch.int64)
        if t.dtype == torch.uint64:                                           # (2^63 and more: negative by now)
            wide = wide.masked_fill(wide < 0, 2 ** 31 - 1)
        t = wide.clamp(-2 ** 31, 2 ** 31 - 1)
    return t.to(device=device, dtype=dtype)


def _rows_of(t: torch.Tensor, rows: int, dtype: torch.dtype, device: torch.device, name: str) -> torch.Tensor:
    """[n] (one list for every row) or [rows, n], as a tensor of `dtype` with unit stride along a row (a row stride of 0 is fine)."""
    if t.dim() == 1:
        t = t.unsqueeze(0).expand(rows, t.shape[0])
    if t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f"{name} must be [rows, n] or [n]")
    t = _converted(t, dtype, device)
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _lengths(t: Optional[torch.Tensor], rows: int, device: torch.device, name: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.numel() != rows:
        raise ValueError(f"{name}: expected {rows} per-row values, got {t.numel()}")
    return _converted(t, torch.int32, device).contiguous()


def process_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None, history_len: Optional[torch.Tensor] = None, prompt_len: Optional[torch.Tensor] = None,
                   repetition_penalty: Knob = 1.0, presence_penalty: Knob = 0.0, frequency_penalty: Knob = 0.0, bias_ids: Optional[torch.Tensor] = None,
                   bias_values: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, mask_rows: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``logits`` [rows, vocab] (bfloat16 or float32, CUDA) with penalties, biases and masks applied, in this order, in float32, rounded once.

    ``history`` [rows, n] (or [n]: the same for every row) int32 token ids, of which the first ``history_len[r]`` count (default: all) and the first ``prompt_len[r]``
    are the prompt's (default: none). A token of the history: ``z / repetition_penalty`` if z > 0, else ``z * repetition_penalty``; one that occurs c > 0 times behind the
    prompt: ``- presence_penalty - frequency_penalty * c``. The penalties are numbers or per-row tensors. ``bias_ids`` int32 / ``bias_values`` float32 [rows, n] (or [n]):
    added to the tokens' logits, one that is listed twice in list order; ids outside the vocabulary (-1) are padding (so a vocabulary shard takes the ids less its first index). ``mask`` int32 [m, >= ceil(vocab / 32)]: bit v & 31 of
    word v >> 5 set = token v allowed, the others become -inf; row r has mask ``mask_rows[r]`` (negative: none; m or more: everything masked), or mask r.

    ``out``: the result's place, ``logits`` itself (in place: only what changes is written) or a tensor that shares nothing with it; a new tensor by default. A row
    whose mask allows nothing is all -inf. Ids, lengths and ``mask_rows`` of another type or on another device are converted, those beyond int32 staying outside. Asynchronous on the current
    stream; nothing is copied to the host.
    """
    r = _lib.host().process_logits(logits, history, history_len, prompt_len, repetition_penalty, presence_penalty, frequency_penalty, bias_ids, bias_values, mask, mask_rows, out)
    if r is not None:
        return r
    given = logits
    logits = _check_logits(logits)
    rows, vocab = logits.shape
    dev = logits.device
    if rows > 1 and logits.stride(0) < vocab:
        logits = logits.contiguous()
    if out is None:
        out = torch.empty(rows, vocab, dtype=logits.dtype, device=dev)
    elif out is given and logits is not given:
        raise ValueError("process_logits: logits that are processed in place must have unit stride along the vocabulary")
    if out.shape != (rows, vocab) or out.dtype != logits.dtype or out.device != dev or (vocab > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < vocab):
        raise ValueError("process_logits: out must be [rows, vocab] of the logits' type on the same device")
    a = _lib.LogitsArgs()
    a.struct_size = C.sizeof(a)
    a.dtype, a.logits, a.rows, a.vocab, a.row_stride = _dtype_code(logits), logits.data_ptr(), rows, vocab, _row_stride(logits)
    a.out, a.out_stride = out.data_ptr(), _row_stride(out)
    if history is not None:
        history = _rows_of(history, rows, torch.int32, dev, "history")
        history_len, prompt_len = _lengths(history_len, rows, dev, "history_len"), _lengths(prompt_len, rows, dev, "prompt_len")
        a.history, a.hist_len, a.hist_stride = history.data_ptr(), history.shape[1], history.stride(0)
        a.history_len = history_len.data_ptr() if history_len is not None else None
        a.prompt_len = prompt_len.data_ptr() if prompt_len is not None else None
    if not isinstance(repetition_penalty, torch.Tensor) and not repetition_penalty > 0:
        raise ValueError("repetition_penalty must be positive")
    ptr, s, k0 = _knob(repetition_penalty, rows, torch.float32, dev, "repetition_penalty"); a.repetition, a.repetition_s = ptr, float(s)
    ptr, s, k1 = _knob(presence_penalty, rows, torch.float32, dev, "presence_penalty"); a.presence, a.presence_s = ptr, float(s)
    ptr, s, k2 = _knob(frequency_penalty, rows, torch.float32, dev, "frequency_penalty"); a.frequency, a.frequency_s = ptr, float(s)
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("process_logits: bias_ids and bias_values go together")
    if bias_ids is not None:
        bias_ids, bias_values = _rows_of(bias_ids, rows, torch.int32, dev, "bias_ids"), _rows_of(bias_values, rows, torch.float32, dev, "bias_values")
        if bias_ids.shape != bias_values.shape:
            raise ValueError("process_logits: bias_ids and bias_values must have the same shape")
        a.bias_ids, a.bias_ids_stride, a.bias_values, a.bias_values_stride = bias_ids.data_ptr(), bias_ids.stride(0), bias_values.data_ptr(), bias_values.stride(0)
        a.bias_len = bias_ids.shape[1]
    if mask is not None:
        if mask.dim() != 2 or mask.dtype != torch.int32 or mask.device != dev or mask.shape[1] < (vocab + 31) // 32:
            raise ValueError("process_logits: mask int32 [m, ceil(vocab / 32)] on the same device")
        if mask.stride(1) != 1 or (mask.shape[0] > 1 and mask.stride(0) < mask.shape[1]):
            mask = mask.contiguous()
        mask_rows = _lengths(mask_rows, rows, dev, "mask_rows")
        if mask_rows is None and mask.shape[0] != rows:
            raise ValueError("process_logits: one mask per row, or mask_rows")
        a.mask_rows = mask_rows.data_ptr() if mask_rows is not None else None
        a.mask, a.mask_stride, a.mask_count = mask.data_ptr() if mask.shape[0] else a.mask_rows, _row_stride(mask), mask.shape[0]     # (no masks: an address that is never read)
    elif mask_rows is not None:
        raise ValueError("process_logits: mask_rows without a mask")
    a.stream = torch.cuda.current_stream(dev).cuda_stream
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().lm_process_logits(C.byref(a)), "lm_process_logits")
    return out
