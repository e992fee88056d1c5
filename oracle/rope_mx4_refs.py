"""Rotary positions and microscaled 4-bit floating point in plain numpy, 64 bits: the definitions that include/sh_ops.h
states (no counterpart in the reference but sh_rope's formula)."""
from __future__ import annotations

import numpy as np

HALF, PAIRS = 0, 1
NONE, LINEAR, BANDS, RAMP = 0, 1, 2, 3


# ---- rotary positions ---------------------------------------------------------------------------------------------
def frequencies(rot: int, base: float, scaling: int = NONE, factor: float = 1.0, lo: float = 1.0, hi: float = 4.0, ctx: int = 0) -> np.ndarray:
    """Radians a position of each pair, one after the other."""
    w = []
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        keep = 1.0
        if scaling == LINEAR:
            keep = 0.0
        elif scaling == BANDS:
            keep = min(1.0, max(0.0, (f * ctx / (2 * np.pi) - lo) / (hi - lo)))
        elif scaling == RAMP:
            per = rot / (2 * np.log(base))
            first = max(0.0, np.floor(per * np.log(ctx / (2 * np.pi * hi))))
            last = min(rot - 1.0, np.ceil(per * np.log(ctx / (2 * np.pi * lo))))
            keep = 1.0 - min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
        w.append(f * (keep + (1 - keep) / factor) if scaling != NONE else f)
    return np.array(w)


def steps(w: np.ndarray) -> np.ndarray:
    """Turns a position as 64-bit fractions."""
    return np.array([int((x / (2 * np.pi)) % 1.0 * 2.0 ** 64) for x in w], dtype=np.uint64)


def turn(x, step, pos, heads: int, dh: int, layout: int, mscale: float = 1.0) -> np.ndarray:
    """[rows, heads dh] in 64 bits, the first 2 len(step) columns of each head turned; rows at negative positions are NaN."""
    n = len(step)
    x = np.asarray(x, np.float64).reshape(len(pos), heads, dh)
    out = x.copy()
    for r, p in enumerate(pos):
        if p < 0:
            out[r] = np.nan
            continue
        phase = np.array([(int(s) * int(p)) % (1 << 64) for s in step], dtype=np.float64)         # whole turns fall off in integers
        a = phase * 2.0 ** -64 * 2 * np.pi
        c, s = mscale * np.cos(a), mscale * np.sin(a)
        i = np.arange(n)
        i, j = (i, i + n) if layout == HALF else (2 * i, 2 * i + 1)
        out[r][:, i] = x[r][:, i] * c - x[r][:, j] * s
        out[r][:, j] = x[r][:, j] * c + x[r][:, i] * s
    return out.reshape(len(pos), -1)


# ---- microscaled 4-bit floating point --------------------------------------------------------------------------------
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([E2M1, -E2M1])


def code(x: np.ndarray) -> np.ndarray:
    """The nearest code of x, |x| <= 6, ties to the even one."""
    a = np.abs(x)
    i = np.clip(np.searchsorted(E2M1, a), 1, 7)
    lo, hi = a - E2M1[i - 1], E2M1[i] - a
    c = np.where((hi < lo) | ((hi == lo) & (i % 2 == 0)), i, i - 1)
    return (c + np.where(np.signbit(x), 8, 0)).astype(np.uint8)


def quant(x: np.ndarray) -> tuple:
    """(codes [rows, 32 nb], scale bytes [rows, nb]) of fp16 rows, one block after the other."""
    rows, cols = x.shape
    nb = -(-cols // 32)
    codes, scales = np.zeros((rows, 32 * nb), np.uint8), np.zeros((rows, nb), np.uint8)
    for b in range(nb):
        v = x[:, 32 * b: 32 * b + 32].astype(np.float64)
        top = np.abs(v).max(1)
        for r in range(rows):
            if not np.isfinite(top[r]):
                scales[r, b] = 255
                continue
            e = -32
            while top[r] > 6 * 2.0 ** e:
                e += 1
            scales[r, b] = e + 127
            codes[r, 32 * b: 32 * b + v.shape[1]] = code(v[r] / 2.0 ** e)
    return codes, scales


def pack(codes: np.ndarray) -> np.ndarray:
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(b: np.ndarray) -> np.ndarray:
    out = np.empty((b.shape[0], 2 * b.shape[1]), np.uint8)
    out[:, 0::2], out[:, 1::2] = b & 15, b >> 4
    return out


def value(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """The numbers that codes [rows, 32 nb] with scale bytes [rows, nb] stand for."""
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return VALUES[codes] * np.repeat(s, 32, 1)


def gemm(x: np.ndarray, w: np.ndarray, bias=None, gelu: bool = False) -> tuple:
    """(x . w^T [+ bias] [gelu], sum |x||w|) of values in 64 bits."""
    z = x @ w.T
    if bias is not None:
        z = z + bias.astype(np.float64)
    if gelu:
        z = 0.5 * z * (1 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
    return z, np.abs(x) @ np.abs(w).T
