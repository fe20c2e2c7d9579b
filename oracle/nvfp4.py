"""numpy restatement of the microscaled 4-bit weight format and of the projection with it, in binary64. TEST INFRASTRUCTURE ONLY.

Codes and block scales are the roundings of real quotients (ties to even): a quotient is compared with a border by comparing its numerator with border * denominator,
which binary64 holds exactly (at most 24 + 24 + 7 bits), so nothing here depends on a division's rounding."""
from __future__ import annotations

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([(m / 8.0 * 2.0 ** -6) if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])     # the values of codes 0 .. 126
NAN_SCALE = 127


def _nearest(numerator: np.ndarray, denominator: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the grid value nearest to numerator / denominator (>= 0), ties to the even index, the last index beyond the grid."""
    code = np.zeros(np.broadcast(numerator, denominator).shape, dtype=np.int64)
    for i, border in enumerate((grid[:-1] + grid[1:]) / 2):
        b = border * denominator
        code += (numerator > b) | ((numerator == b) & (i % 2 == 1))
    return code


def global_scale(x: np.ndarray) -> np.float32:
    a = np.abs(np.asarray(x, dtype=np.float64))
    a = a[np.isfinite(a)]
    g = np.float32(np.float32(a.max() if a.size else 0.0) / np.float32(2688.0))
    return g if g >= np.float32(2.0 ** -126) else np.float32(1.0)


def quantize(x: np.ndarray, g: np.float32):
    """(codes uint8 [rows, cols / 2], scales uint8 [rows, cols / 16]) of a float matrix under the scale g."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    b = x.reshape(rows, cols // 16, 16)
    finite = np.isfinite(b).all(-1)
    if not (g >= np.float32(2.0 ** -126) and np.isfinite(g)):
        finite[:] = False
    b = np.where(finite[..., None], b, 0.0)
    gd = np.float64(g) if np.isfinite(g) else 1.0
    s = _nearest(np.abs(b).max(-1), 6.0 * gd, E4M3)
    unit = (E4M3[s] * gd)[..., None]
    c = np.where(unit > 0, _nearest(np.abs(b), unit, E2M1), 0) + 8 * np.signbit(b)
    c = np.where(finite[..., None], c, 0).reshape(rows, cols).astype(np.uint8)
    return c[:, 0::2] | (c[:, 1::2] << 4), np.where(finite, s, NAN_SCALE).astype(np.uint8)


def scale_values(scales: np.ndarray) -> np.ndarray:
    v = np.concatenate([E4M3, [np.nan]])
    return np.concatenate([v, -v])[np.asarray(scales, dtype=np.int64)]


def values(codes: np.ndarray, scales: np.ndarray, g: np.float32) -> np.ndarray:
    """binary64 values [rows, cols]."""
    rows, half = codes.shape
    n = np.empty((rows, 2 * half), dtype=np.int64)
    n[:, 0::2], n[:, 1::2] = codes & 15, codes >> 4
    v = np.concatenate([E2M1, -E2M1])[n]
    return v * np.repeat(scale_values(scales), 16, axis=1) * np.float64(g)


def head(x: np.ndarray, codes: np.ndarray, scales: np.ndarray, g: np.float32):
    """(logits, bound): x [rows, H] float values times the weight's values, and how far an FP32 accumulation of the exact products may be from it in any order -- 2^-23 of the sum of the
    magnitudes for each of the H additions -- before the rounding to BF16."""
    w = values(codes, scales, g)
    x = np.asarray(x, dtype=np.float64)
    return x @ w.T, (w.shape[1] + 4) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)
