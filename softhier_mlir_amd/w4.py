"""Weights for sh_gemm_w4 (include/sh_ops.h), laid out once on the host: an fp16 / fp32 weight [K, N] to 4-bit codes with a
scale and a zero for each group of k and column, eight codes of consecutive k in a word."""
from __future__ import annotations

import numpy as np


def pack(codes: np.ndarray) -> np.ndarray:
    """[K, N] codes 0 .. 15, K a multiple of 8 -> uint32 words [K / 8, N]: bits 4 j .. 4 j + 3 hold k = 8 i + j."""
    K, N = codes.shape
    if K % 8 or codes.min(initial=0) < 0 or codes.max(initial=0) > 15:
        raise ValueError(f"codes of 0 .. 15 over a multiple of 8 rows (got {K})")
    c = codes.astype(np.uint32).reshape(K // 8, 8, N)
    w = np.zeros((K // 8, N), np.uint32)
    for j in range(8):
        w |= c[:, j] << np.uint32(4 * j)
    return w


def unpack(words: np.ndarray) -> np.ndarray:
    """The codes [8 * rows, N] of packed words."""
    return np.stack([(words >> np.uint32(4 * j)) & 15 for j in range(8)], 1).reshape(-1, words.shape[1]).astype(np.uint8)


def quantize(w: np.ndarray, group: int = 128) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """(words [K / 8, N], fp16 scales [G, N], zeros [G, N] uint8): for each group and column the range of its values, zero
    among them, on 15 steps of `scale`, the smallest fp16 number that covers it (2^-24 at least); code = round(w / scale) + zero.
    A value is off by at most half a step. Values that are not finite, and ranges beyond 15 x 65504, are refused."""
    K, N = w.shape
    if K % 8 or group % 32 or group <= 0:
        raise ValueError(f"K {K} must be a multiple of 8 and group {group} of 32")
    w = w.astype(np.float32)
    if not np.isfinite(w).all():
        raise ValueError("the weight has values that are not finite")
    G = -(-K // group)
    scale, zero = np.empty((G, N), np.float16), np.empty((G, N), np.uint8)
    codes = np.empty((K, N), np.uint8)
    for g in range(G):
        x = w[g * group:(g + 1) * group]
        lo, hi = np.minimum(x.min(0), 0), np.maximum(x.max(0), 0)
        step = np.maximum((hi.astype(np.float64) - lo) / 15, 2.0 ** -24)
        if step.max(initial=0) > 65504:
            raise ValueError(f"a group's range, {15 * step.max():g}, is beyond 15 steps of the largest fp16 scale")
        s = step.astype(np.float16)
        up = s < step                                                       # (fp16 against fp64: exact)
        s[up] = np.nextafter(s[up], np.float16(np.inf))
        sf = s.astype(np.float32)
        z = np.clip(np.rint(-lo / sf), 0, 15)
        codes[g * group:(g + 1) * group] = np.clip(np.rint(x / sf) + z, 0, 15)
        scale[g], zero[g] = s, z
    return pack(codes), scale, zero


def dequantize(words: np.ndarray, scale: np.ndarray, zero: np.ndarray, group: int) -> np.ndarray:
    """The fp32 weight [K, N] that sh_gemm_w4 multiplies with."""
    c = unpack(words).astype(np.float32)
    of = np.arange(c.shape[0]) // group
    return (c - zero.astype(np.float32)[of]) * scale.astype(np.float32)[of]
