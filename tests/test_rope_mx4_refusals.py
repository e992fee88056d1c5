"""What sh_rope_steps, sh_rope_pos, sh_kv_append_rope, sh_mx4_quant, sh_gemm_mx4 and sh_gemm_mx4_f16 refuse, without a GPU: every
check comes before any GPU work, with its code and message. And the definitions' own checks."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from oracle import rope_mx4_refs as R
from softhier_mlir_amd import shops

ONE = 1 << 20                                   # never dereferenced: the checks fail first


def _plan(**kw):
    d = dict(step=ONE, rot=64, layout=shops.SH_ROPE_HALF, mscale=1.0)
    d.update(kw)
    return C.byref(shops.rope_plan(**d))


BAD_PLANS = [dict(step=0), dict(step=ONE + 4), dict(rot=0), dict(rot=63), dict(rot=66), dict(layout=2), dict(mscale=float("nan")), dict(mscale=float("inf"))]


def _cache(**kw):
    d = dict(k=ONE, v=ONE, ks=ONE, vs=ONE, pages=8, hkv=2, dh=64, bs=16, fmt=shops.SH_INT8)
    d.update(kw)
    return C.byref(shops.kv_cache(**d))


def _refused(lib, fn, good, bad, name):
    for i, v in bad:
        a = list(good)
        a[i] = v
        assert fn(*a) == -1, (i, v)
        code, text = shops.last_error()
        assert code == -1 and f"[{name}]" in text, (i, v, text)


def test_rope_pos(lib):
    good = [ONE, 2 * ONE, ONE, _plan(), 3, 4, 64, 256, 300]
    bad = [(0, 0), (1, 0), (2, 0), (0, ONE + 1), (1, ONE + 1), (2, ONE + 2), (3, None), (4, 1 << 31), (6, 0), (6, 63), (6, 32), (7, 255), (8, 255), (5, 1 << 26),
           (1, ONE)]                                                         # in place with two leading dims
    _refused(lib, lib.sh_rope_pos, good, bad + [(3, _plan(**p)) for p in BAD_PLANS], "sh_rope_pos")
    for i in (4, 5):                                                        # no rows or heads: nothing to do
        a = list(good)
        a[i] = 0
        assert lib.sh_rope_pos(*a) == 0


def test_rope_steps(lib):
    good = [ONE, 64, 1e4, shops.SH_ROPE_BANDS, 8.0, 1.0, 4.0, 8192]
    bad = [(0, 0), (0, ONE + 4), (1, 0), (1, 3), (1, 65538), (2, 1.0), (2, 0.0), (2, float("nan")), (2, float("inf")), (3, 4), (4, 0.0), (4, -2.0),
           (4, float("nan")), (4, float("inf")), (5, 0.0), (5, 4.0), (5, float("nan")), (6, float("inf")), (6, 0.5), (7, 0)]
    _refused(lib, lib.sh_rope_steps, good, bad, "sh_rope_steps")


def test_kv_append_rope(lib):
    good = [_cache(), _plan(), ONE, 2 * ONE, ONE, ONE, ONE, ONE, 5, 4, 256, 256, 128, 128]
    bad = [(0, None), (0, _cache(bs=8)), (0, _cache(fmt=shops.SH_FP16)), (1, None), (1, _plan(rot=36)), (2, 0), (3, 0), (4, 0), (5, 0), (6, 0), (7, 0), (2, ONE + 1),
           (3, ONE + 1), (4, ONE + 1), (5, ONE + 1), (6, ONE + 2), (7, ONE + 2), (8, 1 << 31), (10, 255), (11, 255), (12, 127), (13, 127)]
    _refused(lib, lib.sh_kv_append_rope, good, bad + [(1, _plan(**p)) for p in BAD_PLANS], "sh_kv_append_rope")
    a = list(good)
    a[3], a[11] = ONE, 257                                                  # in place with two leading dims
    assert lib.sh_kv_append_rope(*a) == -1
    a = list(good)
    a[8] = 0
    assert lib.sh_kv_append_rope(*a) == 0


def test_mx4_quant(lib):
    good = [ONE, ONE, ONE, 3, 100, 64, 4, 100]
    bad = [(0, 0), (1, 0), (2, 0), (0, ONE + 8), (1, ONE + 2), (2, ONE + 1), (4, 129), (5, 48), (5, 72), (6, 3), (6, 0), (7, 99)]
    _refused(lib, lib.sh_mx4_quant, good, bad, "sh_mx4_quant")
    a = [ONE, ONE, ONE, 1, (1 << 30) + 32, 1 << 30, 1 << 30, 1 << 31]
    assert lib.sh_mx4_quant(*a) == -1
    for i in (3, 4):
        a = list(good)
        a[i] = 0
        assert lib.sh_mx4_quant(*a) == 0


def _epilogues(i):
    e = lambda **kw: C.byref(shops.epi(**kw))  # noqa: E731
    return [(i, e(act=2)), (i, e(bias=ONE, bias_fmt=2)), (i, e(bias=ONE + 1)), (i, e(bias=ONE + 2, bias_fmt=shops.SH_BIAS_FP32)), (i, e(residual=ONE, ldr=63)),
            (i, e(residual=ONE + 1, ldr=64)), (i, e(splits=2)), (i, e(ln_stats=ONE)), (i, e(ln_c=ONE)), (i, e(stats_out=ONE)), (i, e(ln_parts=4))]


def test_gemm_mx4(lib):
    good = [ONE, ONE, ONE, ONE, ONE, 2, 64, 100, 64, 4, 64, 4, 64, None]
    bad = [(i, 0) for i in range(5)] + [(0, ONE + 8), (2, ONE + 8), (1, ONE + 2), (3, ONE + 2), (4, ONE + 1), (5, (1 << 26) + 1), (6, (1 << 26) + 1), (7, 0), (7, 129),
                                        (8, 48), (8, 72), (9, 0), (9, 5), (10, 48), (10, 72), (11, 0), (11, 6), (12, 63)]
    _refused(lib, lib.sh_gemm_mx4, good, bad + _epilogues(13), "sh_gemm_mx4")
    for i in (5, 6):
        a = list(good)
        a[i] = 0
        assert lib.sh_gemm_mx4(*a) == 0


def test_gemm_mx4_f16(lib):
    good = [ONE, ONE, ONE, ONE, 2, 64, 100, 100, 64, 4, 64, None]
    bad = [(i, 0) for i in range(4)] + [(0, ONE + 1), (1, ONE + 8), (2, ONE + 2), (3, ONE + 1), (4, 17), (5, (1 << 26) + 1), (6, 0), (6, 129), (7, 99), (8, 48), (8, 72),
                                        (9, 0), (9, 6), (10, 63)]
    _refused(lib, lib.sh_gemm_mx4_f16, good, bad + _epilogues(11), "sh_gemm_mx4_f16")
    for i in (4, 5):
        a = list(good)
        a[i] = 0
        assert lib.sh_gemm_mx4_f16(*a) == 0


def test_codes_are_the_nearest_values():
    x = np.linspace(-6, 6, 4801)
    c = R.code(x)
    err = np.abs(R.VALUES[c] - x)
    assert (err <= np.abs(R.VALUES[None, :] - x[:, None]).min(1)).all()
    for tie, even in ((0.25, 0.0), (0.75, 1.0), (1.25, 1.0), (1.75, 2.0), (2.5, 2.0), (3.5, 4.0), (5.0, 4.0)):
        assert R.VALUES[R.code(np.array([tie, -tie]))].tolist() == [even, -even]
    assert R.code(np.array([-0.0, 0.0, -0.1])).tolist() == [8, 0, 8]


def test_quantised_rows_are_within_a_step():
    """|x - value| <= scale / 2 below 2 scale, scale below 4, 2 scale to 6: at most 1/6 of a block's largest value (half of the step 2 scale, at amax > 3 scale: 1/3)."""
    x = np.random.default_rng(0).standard_normal((20, 70)).astype(np.float16)
    c, s = R.quant(x)
    v = R.value(c, s)
    assert (v[:, 70:] == 0).all()
    top = np.abs(np.pad(x.astype(np.float64), ((0, 0), (0, 26)))).reshape(20, 3, 32).max(2)
    scale = np.exp2(s.astype(np.float64) - 127)
    assert (top <= 6 * scale).all() and (top > 3 * scale).all()
    assert (np.abs(v[:, :70] - x.astype(np.float64)) <= np.repeat(scale, 32, 1)[:, :70]).all()
    assert np.array_equal(R.unpack(R.pack(c)), c)


@pytest.mark.parametrize("layout", [R.HALF, R.PAIRS])
def test_turns_keep_lengths_and_differences(layout):
    """A turn keeps each pair's length, and the product of two turned rows depends on the difference of their positions alone."""
    rng = np.random.default_rng(4)
    q, k = rng.standard_normal((2, 1, 64))
    step = R.steps(R.frequencies(48, 1e4))
    t = lambda x, p: R.turn(x, step, [p], 1, 64, layout)  # noqa: E731
    assert np.allclose(np.linalg.norm(t(q, 12345)), np.linalg.norm(q), rtol=1e-12)
    for far in (0, 1000, 1 << 28):
        assert np.allclose((t(q, far + 7) * t(k, far)).sum(), (t(q, 7) * t(k, 0)).sum(), rtol=0, atol=1e-9)
    assert np.isnan(t(q, -1)).all()
