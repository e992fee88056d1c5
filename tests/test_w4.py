"""The 4-bit weight layout on the host, and the definitions the GPU tests of the 8-bit cache and of these weights compare with."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import kv_refs as R
from softhier_mlir_amd import w4


def test_pack_layout():
    c = np.random.default_rng(0).integers(0, 16, (24, 5)).astype(np.uint8)
    w = w4.pack(c)
    assert w.shape == (3, 5) and w.dtype == np.uint32
    assert all((int(w[i, n]) >> (4 * j)) & 15 == c[8 * i + j, n] for i in range(3) for j in range(8) for n in range(5))
    assert np.array_equal(w4.unpack(w), c) and np.array_equal(R.w4_pack(c), w)
    for bad in (np.zeros((12, 3)), np.full((8, 1), 16), np.full((8, 1), -1)):
        with pytest.raises(ValueError):
            w4.pack(bad)


@pytest.mark.parametrize("K,N,group", [(128, 7, 32), (720, 40, 128), (8, 3, 32)])
def test_quantize_error(K, N, group):
    """Half a step, plus half a step where the zero's rounding pushes the range's end past the last code; the fp16 scale is off by 2^-11,
    15 codes of it by 15 * 2^-11 steps."""
    rng = np.random.default_rng(K)
    w = (rng.standard_normal((K, N)) * 0.05).astype(np.float16)
    w[:, 0] = 0
    w[:, 1] = np.abs(w[:, 1])
    words, s, z = w4.quantize(w, group)
    assert z.max() <= 15 and words.shape == (K // 8, N) and s.shape == (-(-K // group), N)
    step = s.astype(np.float64)[np.arange(K) // group]
    err = np.abs(w4.dequantize(words, s, z, group) - w.astype(np.float64))
    assert (err <= step * (1.0 + 15 * 2.0 ** -11)).all() and (err <= step * 0.51).mean() > 0.98
    assert (w4.dequantize(words, s, z, group)[:, 0] == 0).all()
    x = rng.standard_normal((2, K)).astype(np.float16)
    assert np.allclose(x.astype(np.float64) @ w4.dequantize(words, s, z, group).astype(np.float64), R.gemm_w4(x, w4.unpack(words), s, z, group)[0],
                       rtol=1e-5, atol=1e-6)
    with pytest.raises(ValueError):
        w4.quantize(w, 48)


@pytest.mark.parametrize("std", [1e-8, 1e-6, 3e-6, 1e-5, 0.05, 1e3, 1e5])
@pytest.mark.parametrize("side", ["both", "above", "below"])
def test_quantize_is_off_by_half_a_step(std, side):
    """Scales from the subnormal ones to the largest. The scale covers its group's range, so no code is clipped; the quotient w / scale in
    fp32 is off by 15 * 2^-24 steps at most."""
    rng = np.random.default_rng(int(np.log10(std) + 20))
    w = (rng.standard_normal((256, 300)) * std).astype(np.float32)
    w = np.abs(w) if side == "above" else -np.abs(w) if side == "below" else w
    w[:32, 0], w[32:64, 1], w[5, 2] = 0, std, -15 * std
    if 15 * std > 15 * 65504:                                       # (the row of -15 std is beyond the largest scale)
        with pytest.raises(ValueError):
            w4.quantize(w, 32)
        w[5, 2] = 0
    words, s, z = w4.quantize(w, 32)
    step = s.astype(np.float64)[np.arange(256) // 32]
    assert np.isfinite(step).all() and z.max() <= 15
    err = np.abs(w4.dequantize(words, s, z, 32).astype(np.float64) - w)
    assert (err <= step * (0.5 + 2.0 ** -20)).all(), float((err / step).max())


def test_quantize_refuses_what_has_no_scale():
    w = np.zeros((64, 4), np.float32)
    for bad in (np.nan, np.inf, -np.inf, 15 * 65504 * 1.001):
        w[33, 2] = bad
        with pytest.raises(ValueError):
            w4.quantize(w, 32)
    w[33, 2], w[34, 2] = 15 * 65504 * 0.6, -15 * 65504 * 0.6             # each in range, not both
    with pytest.raises(ValueError):
        w4.quantize(w, 32)
    w[34, 2], w[33, 2] = 0, 15 * 65504
    assert w4.dequantize(*w4.quantize(w, 32), 32)[33, 2] == 15 * 65504


def test_reference_codes_are_e4m3():
    import torch
    c = np.arange(256, dtype=np.uint8)
    t = torch.from_numpy(c.copy()).view(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert np.array_equal(R.E4M3, t, equal_nan=True)
    x = np.concatenate([np.random.default_rng(1).standard_normal(20000) * 2.0 ** np.random.default_rng(2).integers(-12, 9, 20000), t[~np.isnan(t)],
                        (t[:126] + t[1:127]) / 2]).astype(np.float32)
    want = torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(R.code(x.astype(np.float64), R.FP8), want)


@pytest.mark.parametrize("fmt", [R.INT8, R.FP8])
def test_reference_scales(fmt):
    for a in (0.0, 6e-8, 1.0, 126.9, 127.0, 127.1, 448.0, 449.0, 65504.0):
        s = R.pow2_scale(a, fmt)
        assert a <= s * R.QMAX[fmt] and (s == 2.0 ** -32 or a > s / 2 * R.QMAX[fmt]) and np.log2(s) % 1 == 0


def test_reference_attention_is_softmax_of_dequantized_rows():
    rng = np.random.default_rng(3)
    k, v = rng.integers(0, 256, (4, 1, 16, 16)).astype(np.uint8), rng.integers(0, 256, (4, 1, 16, 16)).astype(np.uint8)
    ks, vs = np.full((4, 1), 0.01, np.float32), np.full((4, 1), 0.02, np.float32)
    table = np.array([[2, 0, 3]])
    q = rng.standard_normal((3, 32)).astype(np.float16)
    o = R.attention(q, k, v, ks, vs, table, [37], np.array([0, 3]), 2, 0.25, R.INT8)[0]
    K = np.concatenate([k[p, 0] for p in (2, 0, 3)]).view(np.int8).astype(np.float64) * np.float64(np.float32(0.01))
    V = np.concatenate([v[p, 0].T for p in (2, 0, 3)]).copy().view(np.int8).astype(np.float64) * np.float64(np.float32(0.02))
    for r in range(3):
        n = 35 + r
        for h in range(2):
            s = K[:n] @ q[r, 16 * h:16 * h + 16].astype(np.float64) * 0.25
            p = np.exp(s - s.max())
            assert np.allclose(o[r, 16 * h:16 * h + 16], p @ V[:n] / p.sum(), rtol=1e-12)


def test_reference_slots_hands_every_page_out_once():
    table, lens = np.full((3, 4), -1, np.int32), np.zeros(3, np.int32)
    pool, state = np.arange(6, dtype=np.int32), np.array([0, 6, 0], np.int32)
    r = R.slots(table, lens, np.array([20, 33, 40], np.int32), pool, state, 16, 100)
    assert r["state_out"].tolist() == [5, 1, 1] and r["kv_len"].tolist() == [20, 33, 0] and r["row_start"].tolist() == [0, 20, 53, 93]
    assert r["table"][0, :2].tolist() == [0, 1] and r["table"][1, :3].tolist() == [2, 3, 4] and (r["slots"][53:] == -1).all()
    r2 = R.slots(r["table"], r["lens_out"], np.array([-1, 1, 16], np.int32), r["pool"], r["state_out"], 16, 100)
    assert r2["state_out"].tolist() == [0, 2, 0] and r2["pool"][[0, 1]].tolist() == [0, 1]
