"""numpy restatement of the logits' processing (penalties by request, biases, masks) in binary64. TEST INFRASTRUCTURE ONLY."""
from __future__ import annotations

import numpy as np


def process(z, history=None, history_len=None, prompt_len=None, repetition=1.0, presence=0.0, frequency=0.0, bias_ids=None, bias_values=None, mask=None, mask_rows=None):
    """(values, bound, touched) [rows, vocab]: bound is what binary32 arithmetic may add up to before the last rounding -- half a unit (2^-24) of the largest
    intermediate for each operation; touched: the logits that a list names and no mask hides."""
    z = np.asarray(z, dtype=np.float64).copy()
    rows, vocab = z.shape
    knob = lambda k, r: float(np.float32(np.broadcast_to(np.asarray(k, dtype=np.float32), (rows,))[r]))
    bound, touched = np.zeros_like(z), np.zeros(z.shape, dtype=bool)
    for r in range(rows):
        operations, size = np.zeros(vocab), np.abs(z[r])
        if history is not None:
            h = np.broadcast_to(np.asarray(history), (rows, np.shape(history)[-1]))[r]
            n = len(h) if history_len is None else min(max(int(history_len[r]), 0), len(h))
            p = 0 if prompt_len is None else int(prompt_len[r])
            count = lambda ids: np.bincount(ids[(ids >= 0) & (ids < vocab)], minlength=vocab)
            every, behind = count(h[:n]), count(h[max(p, 0):n])
            rho, pi, phi = knob(repetition, r), knob(presence, r), knob(frequency, r)
            z[r] = np.where(every > 0, np.where(z[r] > 0, z[r] / rho, z[r] * rho), z[r])
            size = np.maximum(size, np.abs(z[r]))
            z[r] = np.where(behind > 0, z[r] - pi - phi * behind, z[r])
            size = size + np.where(behind > 0, abs(pi) + abs(phi) * behind, 0.0)
            operations += 4 * (every > 0)
            touched[r] |= every > 0
        if bias_ids is not None:
            ids, values = (np.broadcast_to(np.asarray(t), (rows, np.shape(t)[-1]))[r] for t in (bias_ids, bias_values))
            for i, v in zip(ids.tolist(), values.astype(np.float64).tolist()):
                if 0 <= i < vocab:
                    z[r, i] += v
                    size[i] += abs(v)
                    operations[i] += 1
                    touched[r, i] = True
        if mask is not None:
            m = r if mask_rows is None else int(mask_rows[r])
            if m >= len(mask):
                allowed = np.zeros(vocab, dtype=bool)
            elif m >= 0:
                allowed = np.unpackbits(np.ascontiguousarray(mask[m]).view(np.uint8), bitorder="little")[:vocab].astype(bool)
            else:
                allowed = np.ones(vocab, dtype=bool)
            z[r] = np.where(allowed, z[r], -np.inf)
            touched[r] &= allowed
        with np.errstate(invalid="ignore"):
            bound[r] = np.where(operations > 0, operations * 2.0 ** -24 * np.where(np.isfinite(size), size, 0.0), 0.0)
    return z, bound, touched
