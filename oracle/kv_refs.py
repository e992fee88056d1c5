"""The 8-bit paged key / value cache and the products with 4-bit weights in plain numpy, 64 bits: the definitions that
include/sh_ops.h states (no counterpart in the reference), one request, page and head at a time."""
from __future__ import annotations

import numpy as np

INT8, FP8 = 3, 1                                     # SH_INT8, SH_FP8
QMAX = {INT8: 127.0, FP8: 448.0}


def _e4m3_table() -> np.ndarray:
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        v[c] = np.nan if c & 127 == 127 else -x if c & 128 else x
    return v


E4M3 = _e4m3_table()


def value(codes: np.ndarray, fmt: int) -> np.ndarray:
    return codes.view(np.int8).astype(np.float64) if fmt == INT8 else E4M3[codes]


def code(x: np.ndarray, fmt: int) -> np.ndarray:
    """The nearest code of x, ties to the even one, saturated."""
    if fmt == INT8:
        return np.clip(np.rint(x), -127, 127).astype(np.int8).view(np.uint8)
    a = np.minimum(np.abs(x), 448.0)
    pos = E4M3[:127]
    i = np.clip(np.searchsorted(pos, a), 1, 126)
    lo, hi = a - pos[i - 1], pos[i] - a
    c = np.where((hi < lo) | ((hi == lo) & (i % 2 == 0)), i, i - 1)
    return (c + np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def pow2_scale(amax: float, fmt: int) -> float:
    """The smallest power of two s >= 2^-32 with amax <= s * QMAX."""
    s = 2.0 ** -32
    while amax > s * QMAX[fmt]:
        s *= 2
    return s


def slots(table, lens, add, pool, state, bs: int, rows: int) -> dict:
    """sh_kv_slots, one request after the other."""
    table, pool = table.copy(), pool.copy()
    B, ld = table.shape
    pages = len(pool)
    head, count = int(state[0]), int(state[1])
    cdiv = lambda a, b: -(-a // b)  # noqa: E731
    out = dict(row_start=np.zeros(B + 1, np.int32), slots=np.full(rows, -1, np.int32), pos=np.full(rows, -1, np.int32),
               kv_len=np.zeros(B, np.int32), lens_out=lens.copy())
    asked = used = back = refused = end = 0
    given = []
    for b in range(B):
        n, have = max(int(add[b]), 0), cdiv(int(lens[b]), bs)
        start, end = end, end + n
        out["row_start"][b + 1] = end
        if add[b] < 0:
            given += table[b, :have].tolist()
            out["lens_out"][b] = 0
            continue
        new = int(lens[b]) + n
        if new > ld * bs or end > rows:
            refused += 1
            continue
        need = cdiv(new, bs) - have
        asked += need
        if need and asked > count:
            refused += 1
            continue
        for i in range(need):
            table[b, have + i] = pool[(head + asked - need + i) % pages]
        if need:
            used = asked
        out["kv_len"][b] = out["lens_out"][b] = new
        p = np.arange(int(lens[b]), new)
        pg = table[b, p // bs]
        out["slots"][start:end] = np.where((pg >= 0) & (pg < pages), pg * bs + p % bs, -1)
        out["pos"][start:end] = p
    for i, p in enumerate(given):
        pool[(head + count + i) % pages] = p
    back = len(given)
    out.update(table=table, pool=pool, state_out=np.array([(head + used) % pages, min(count - used + back, pages), refused], np.int32))
    return out


def append(k, v, ks, vs, xk, xv, slot, fmt: int) -> tuple:
    """sh_kv_append on codes k [pages, hkv, bs, dh], v [pages, hkv, dh, bs] and scales [pages, hkv]: the new arrays."""
    k, v, ks, vs = k.copy(), v.copy(), ks.copy(), vs.copy()
    pages, hkv, bs, dh = k.shape
    clean = lambda x: np.clip(np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=65504.0, neginf=-65504.0), -65504, 65504)  # noqa: E731
    xs = [clean(x).reshape(len(slot), hkv, dh) for x in (xk, xv)]
    i = 0
    while i < len(slot):
        if not 0 <= slot[i] < pages * bs:
            i += 1
            continue
        e = i + 1
        while e < len(slot) and slot[e] == slot[e - 1] + 1 and slot[e] // bs == slot[i] // bs:
            e += 1
        page, off = slot[i] // bs, slot[i] % bs
        for x, c, s in ((xs[0], k, ks), (xs[1], v.transpose(0, 1, 3, 2), vs)):
            for h in range(hkv):
                new = pow2_scale(np.abs(x[i:e, h]).max(), fmt)
                if off:
                    was = float(s[page, h])
                    new = max(new, was)
                    if new != was:
                        c[page, h, :off] = code(value(np.ascontiguousarray(c[page, h, :off]), fmt) * (was / new), fmt)
                s[page, h] = new
                c[page, h, off:off + e - i] = code(x[i:e, h] / new, fmt)
        i = e
    return k, v, ks, vs


def attention(q, k, v, ks, vs, table, kv_len, row_start, H: int, scale: float, fmt: int, window: int = 0, max_q: int = 1 << 30) -> tuple:
    """sh_attention_kv: (o, reach, spread): the outputs (NaN in rows of no request), the softmax-weighted |v| and the largest
    scale sum |q||k| of each output (what its rounding errors are relative to)."""
    pages, hkv, bs, dh = k.shape
    grp, rows = H // hkv, q.shape[0]
    o, reach, spread = (np.full((rows, H, dh), np.nan) for _ in range(3))
    q = q.astype(np.float64).reshape(rows, H, dh)
    for b in range(len(kv_len)):
        L = min(max(int(kv_len[b]), 0), table.shape[1] * bs)
        r0, r1 = (b, b + 1) if row_start is None else (int(row_start[b]), int(row_start[b + 1]))
        t = np.arange(L)
        page = table[b, t // bs]
        ok = (page >= 0) & (page < pages)
        page = np.where(ok, page, 0)
        for h in range(hkv):
            K = np.where(ok[:, None], value(k[page, h, t % bs], fmt) * ks[page, h].astype(np.float64)[:, None], 0.0)
            V = np.where(ok[:, None], value(v[page, h, :, t % bs], fmt) * vs[page, h].astype(np.float64)[:, None], 0.0)
            for r in range(r0, min(r1, r0 + max_q)):
                pos = L - (r1 - r0) + (r - r0)
                see = ok & (t <= pos) & ((t > pos - window) if window else True)
                for g in range(h * grp, h * grp + grp):
                    if not see.any():
                        o[r, g], reach[r, g], spread[r, g] = 0.0, 0.0, 0.0
                        continue
                    s = K[see] @ q[r, g] * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    o[r, g] = p @ V[see]
                    reach[r, g] = p @ np.abs(V[see])
                    spread[r, g] = (np.abs(K[see]) @ np.abs(q[r, g]) * abs(scale)).max()
    return o.reshape(rows, -1), reach.reshape(rows, -1), spread.reshape(rows, -1)


def w4_pack(codes: np.ndarray) -> np.ndarray:
    """[K, N] codes 0 .. 15 -> [K / 8, N] words."""
    K, N = codes.shape
    c = codes.astype(np.uint32).reshape(K // 8, 8, N)
    return np.bitwise_or.reduce(c << (4 * np.arange(8, dtype=np.uint32))[None, :, None], axis=1)


def gemm_w4(x, codes, scale, zero, group: int, bias=None, gelu: bool = False) -> tuple:
    """(x . W [+ bias] [gelu], sum |x||W|) in 64 bits."""
    K = codes.shape[0]
    of = np.arange(K) // group
    w = (codes.astype(np.float64) - (8.0 if zero is None else zero.astype(np.float64)[of])) * scale.astype(np.float64)[of]
    x = x.astype(np.float64)
    z = x @ w
    if bias is not None:
        z = z + bias.astype(np.float64)
    if gelu:
        z = 0.5 * z * (1 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
    return z, np.abs(x) @ np.abs(w)
