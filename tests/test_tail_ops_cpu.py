"""The 4-bit weight, the projection with it and the logits' processing without a GPU: the ctypes structures have the C layout, argument checks answer before any CUDA work, and the
restatements the GPU tests use hold against elementary definitions."""
import ctypes as C
import os
import subprocess
import tempfile
from fractions import Fraction

import numpy as np
import pytest
import torch

import lithos_metal_b200 as lm
from lithos_metal_b200 import _lib
from oracle import logits as o_logits
from oracle import nvfp4 as o

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_ctypes_structs_match_the_c_layout():
    structs = {"lm_quantize_nvfp4_args": _lib.QuantizeNvfp4Args, "lm_dequantize_nvfp4_args": _lib.DequantizeNvfp4Args, "lm_head_nvfp4_args": _lib.HeadNvfp4Args, "lm_logits_args": _lib.LogitsArgs}
    lines, want = [], []
    for name, t in structs.items():
        lines.append(f'printf("%zu ", sizeof({name}));')
        want.append(C.sizeof(t))
        for f, _ in t._fields_:
            lines.append(f'printf("%zu ", offsetof({name}, {f}));')
            want.append(getattr(t, f).offset)
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "lithos_b200.h"\nint main(){' + "\n".join(lines) + "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "t.c"), "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", os.path.join(d, "t"), os.path.join(d, "t.c")], check=True)
        out = subprocess.run([os.path.join(d, "t")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in out] == want


def test_argument_checks_need_no_device():
    L = _lib.lib()
    INVALID, UNSUPPORTED = -1, -4
    a = _lib.QuantizeNvfp4Args()
    assert L.lm_quantize_nvfp4(C.byref(a)) == INVALID                       # struct_size not set
    a.struct_size = C.sizeof(a)
    assert L.lm_quantize_nvfp4(C.byref(a)) == 0                             # nothing to do
    a.rows, a.cols, a.row_stride = 2, 24, 24
    assert L.lm_quantize_nvfp4(C.byref(a)) == INVALID                       # no input
    a.x = a.codes = a.scales = a.scale = 256
    a.codes_stride, a.scales_stride = 12, 2
    assert L.lm_quantize_nvfp4(C.byref(a)) == UNSUPPORTED                   # 24 columns
    a.cols, a.row_stride, a.codes_stride, a.find_scale = 32, 32, 16, 1
    assert L.lm_quantize_nvfp4(C.byref(a)) == INVALID                       # no scratch
    d = _lib.DequantizeNvfp4Args()
    d.struct_size = C.sizeof(d)
    d.rows, d.cols = 1, 16
    assert L.lm_dequantize_nvfp4(C.byref(d)) == INVALID
    h = _lib.HeadNvfp4Args()
    h.struct_size = C.sizeof(h)
    h.rows, h.vocab, h.hidden_dim, h.hidden_stride, h.logits_stride, h.codes_stride, h.scales_stride = 1, 10, 96, 96, 10, 48, 6
    h.hidden = h.codes = h.scales = h.scale = h.logits = 256
    assert L.lm_head_nvfp4(C.byref(h)) == UNSUPPORTED                       # 96 columns: no multiple of 64
    h.hidden_dim = h.hidden_stride = 12800
    h.codes_stride, h.scales_stride = 6400, 800
    assert L.lm_head_nvfp4(C.byref(h)) == UNSUPPORTED                       # longer than the rows in shared memory
    h.hidden_dim = h.hidden_stride = 64
    h.codes = 264
    assert L.lm_head_nvfp4(C.byref(h)) == UNSUPPORTED                       # codes off their alignment
    h.codes, h.rows = 256, 65537
    assert L.lm_head_nvfp4(C.byref(h)) == UNSUPPORTED
    h.rows, h.logits_stride = 2, 9
    assert L.lm_head_nvfp4(C.byref(h)) == INVALID
    p = _lib.LogitsArgs()
    assert L.lm_process_logits(C.byref(p)) == INVALID
    p.struct_size = C.sizeof(p)
    p.rows, p.vocab, p.row_stride, p.out_stride = 4, 100, 100, 100
    assert L.lm_process_logits(C.byref(p)) == INVALID                       # no logits
    p.logits, p.out, p.dtype = 4096, 4096, 1
    assert L.lm_process_logits(C.byref(p)) == 0                             # in place, nothing named
    for out in (4096 + 4 * 50, 4096 + 400, 4096 - 400, 4096 + 4 * 399):
        p.out = out
        assert L.lm_process_logits(C.byref(p)) == INVALID                   # overlaps
    p.out, p.history, p.hist_len, p.hist_stride = 4096, 256, 65537, 65537
    p.repetition_s = 1.0
    assert L.lm_process_logits(C.byref(p)) == UNSUPPORTED
    p.hist_len, p.repetition_s = 5, 0.0
    assert L.lm_process_logits(C.byref(p)) == INVALID                       # a repetition penalty of 0
    p.history, p.bias_len = None, 3
    assert L.lm_process_logits(C.byref(p)) == INVALID                       # a list without its arrays
    p.bias_len, p.mask, p.mask_stride, p.mask_count = 0, 256, 3, 4
    assert L.lm_process_logits(C.byref(p)) == INVALID                       # masks shorter than the vocabulary
    p.mask_stride, p.mask_count = 4, 3
    assert L.lm_process_logits(C.byref(p)) == INVALID                       # fewer masks than rows
    p.mask_count, p.logits = 4, 4097
    assert L.lm_process_logits(C.byref(p)) == INVALID                       # not even an element's alignment


def test_only_cuda_tensors():
    with pytest.raises(RuntimeError):
        lm.quantize_nvfp4(torch.zeros(2, 32))
    with pytest.raises(RuntimeError):
        lm.Nvfp4Weight(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), torch.ones(1))
    with pytest.raises(RuntimeError):
        lm.process_logits(torch.zeros(2, 32))


def test_the_format_restated_in_fractions():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((6, 32)) * np.exp(rng.standard_normal((6, 1)))).astype(np.float32)
    g = o.global_scale(x)
    codes, scales = o.quantize(x, g)
    assert torch.equal(torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double(), torch.from_numpy(o.E4M3))

    def nearest(q, grid):
        return min(range(len(grid)), key=lambda i: (abs(Fraction(float(grid[i])) - q), i % 2))

    for r in range(6):
        for b in range(2):
            block = [Fraction(float(v)) for v in x[r, 16 * b:16 * b + 16]]
            s = nearest(max(abs(v) for v in block) / (6 * Fraction(float(g))), o.E4M3)
            assert s == scales[r, b]
            for i, v in enumerate(block):
                c = codes[r, 8 * b + i // 2] >> (4 * (i % 2)) & 15
                assert c == nearest(abs(v) / (Fraction(float(o.E4M3[s])) * Fraction(float(g))), o.E2M1) + 8 * (v < 0)
    assert np.abs(o.values(codes, scales, g) - x).max() <= 0.5 * 2 / 6 * np.abs(x).max() * 1.1


def test_the_logits_restated_token_by_token():
    z = np.array([[1.0, -2.0, 3.0, -4.0, 5.0]])
    got, _, touched = o_logits.process(z, history=[[1, 2, 2, 9, -1, 4, 0]], history_len=[6], prompt_len=[2], repetition=2.0, presence=0.5, frequency=0.25,
                                       bias_ids=[[4, 4, -1]], bias_values=np.array([[1.0, 2.0, 7.0]]), mask=np.array([[0b11110]], dtype=np.int32))
    assert got.tolist() == [[-np.inf, -4.0, 1.5 - 0.5 - 0.25, -4.0, 2.5 - 0.5 - 0.25 + 3.0]] and touched.tolist() == [[False, True, True, False, True]]


def wrong_looks(places, total):
    """The batch projection's codes: orders 0, 1, 2 .. are copied into place (order mod places), the copies complete in any order, pair (order mod 2) takes them, and looks at order i when the
    products of order i - 4 are done (all before i - 3 taken). A place is filled again when it has been taken. Every state that can be reached; those where a wait by parity ends although the
    order's copy is not the place's last completed one."""
    seen, wrong, queue = set(), set(), [(0, frozenset(), 0, 1)]
    while queue:
        state = queue.pop()
        if state in seen:
            continue
        seen.add(state)
        issued, there, even, odd = state
        taken = lambda i: i < (odd if i % 2 else even)
        if issued < total and (issued < places or taken(issued - places)):
            queue.append((issued + 1, there, even, odd))
        queue += [(issued, there | {f}, even, odd) for f in range(issued) if f not in there]
        for i in (even, odd):
            if i < total and all(taken(j) for j in range(i - 3)):
                done = sum(f % places == i % places for f in there)
                if done % 2 != (i // places) % 2:                           # the wait for the phase of parity (i // places) % 2 ends
                    if done != i // places + 1:
                        wrong.add((i, done))
                    else:
                        queue.append((issued, there, even, i + 2) if i % 2 else (issued, there, i + 2, odd))
    return wrong


def test_an_even_number_of_places_for_codes_cannot_be_misread():
    assert wrong_looks(3, 8)                                                # (the check can fail)
    assert not any(wrong_looks(places, 9) for places in (2, 4, 6))
    source = open(os.path.join(ROOT, "lithos_metal_b200", "csrc", "tail_ops.cu")).read()
    assert "P.code_slots = kB4MaxCodeSlots;" in source and "P.code_slots -= 2;" in source
    header = open(os.path.join(ROOT, "lithos_metal_b200", "csrc", "lm_head_nvfp4_batch.cuh")).read()
    assert "kB4MaxCodeSlots = 8" in header
