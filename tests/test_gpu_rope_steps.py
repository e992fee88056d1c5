"""How exact sh_rope_steps' frequencies are, and the positions turned by them, against frequencies of fifty digits."""
from __future__ import annotations

import ctypes as C
import functools
from decimal import Decimal as D, getcontext

import numpy as np
import pytest

from conftest import _KEEP, to_dev, to_np
from oracle import rope_mx4_refs as R
from softhier_mlir_amd import shops

pytestmark = pytest.mark.gpu
A = shops.addr
getcontext().prec = 50
TWO_PI = 2 * D("3.14159265358979323846264338327950288419716939937510")
BOUND = 1.5e-16                      # turns a position, as include/sh_ops.h states it

PLANS = [(128, 1e4, R.NONE, 1.0, 1.0, 4.0, 0), (64, 5e5, R.NONE, 1.0, 1.0, 4.0, 0), (256, 1e6, R.NONE, 1.0, 1.0, 4.0, 0), (20, 1.5, R.NONE, 1.0, 1.0, 4.0, 0),
         (2048, 1e4, R.NONE, 1.0, 1.0, 4.0, 0), (128, 5e5, R.LINEAR, 3.0, 1.0, 4.0, 0), (128, 5e5, R.BANDS, 8.0, 1.0, 4.0, 8192), (20, 1e4, R.BANDS, 32.0, 0.5, 8.0, 2048),
         (64, 1e4, R.RAMP, 40.0, 1.0, 32.0, 4096), (128, 1e6, R.RAMP, 4.0, 1.0, 32.0, 32768)]


@functools.lru_cache(maxsize=None)
def _turns(rot, base, scaling, factor, lo, hi, ctx):
    """Turns a position of each pair."""
    out = []
    log = D(base).ln()
    for i in range(rot // 2):
        w, keep = (log * D(-2 * i) / D(rot)).exp(), D(1)
        if scaling == R.LINEAR:
            keep = D(0)
        elif scaling == R.BANDS:
            keep = min(D(1), max(D(0), (w * ctx / TWO_PI - D(lo)) / (D(hi) - D(lo))))
        elif scaling == R.RAMP:
            at = [D(rot) / (2 * log) * (D(ctx) / (TWO_PI * D(n))).ln() for n in (hi, lo)]
            first, last = max(D(0), at[0].to_integral_value("ROUND_FLOOR")), min(D(rot - 1), at[1].to_integral_value("ROUND_CEILING"))
            keep = 1 - min(D(1), max(D(0), (D(i) - first) / (last - first)))
        out.append(w * (keep + (1 - keep) / D(factor)) / TWO_PI)
    return out


def _steps(lib, plan):
    import torch
    t = torch.zeros(plan[0] // 2, dtype=torch.int64, device="cuda")
    _KEEP.append(t)
    torch.cuda.synchronize()
    assert lib.sh_rope_steps(A(t), *plan) == 0, shops.last_error()
    return t


@pytest.mark.parametrize("plan", PLANS, ids=str)
def test_steps(lib, gpu, plan):
    """w in fp64 is off by |ln w| + 8 units of 2^-53 at most (its exponent's rounding, two steps of the power, three more operations and the constant), so turns by
    w (|ln w| + 8) 2^-53 / 2 pi: at most 1.42e-16, where w is 1. What scaling adds for bands is below hi / ctx times thirty such units."""
    got, want = to_np(_steps(lib, plan)).view(np.uint64), _turns(*plan)
    err = [abs(D(int(g)) / D(2) ** 64 - w) for g, w in zip(got, want)]
    assert max(err) <= D(BOUND), float(max(err))


@pytest.mark.parametrize("layout", [R.HALF, R.PAIRS])
@pytest.mark.parametrize("plan", [p for p in PLANS if p[0] <= 128], ids=str)
def test_positions(lib, gpu, plan, layout):
    """Rows turned by that plan, near and up to the last position: an angle is off by 2 pi BOUND times the position, the rest as for a given step (one rounding
    to fp16, cosine and sine 2^-37 off and rounded to fp32, two products and a sum: 3 x 2^-24)."""
    rot, heads, dh = plan[0], 2, plan[0]
    pos = np.array([0, 1, 77, 4095, 131071, (1 << 20) - 3, (1 << 24) + 1, 123456789, (1 << 30) - 1, 2 ** 31 - 1], np.int32)
    x = np.random.default_rng(rot).standard_normal((len(pos), heads * dh)).astype(np.float16)
    step, X, P = _steps(lib, plan), to_dev(x), None
    import torch
    P, Y = torch.from_numpy(pos).cuda(), torch.zeros((len(pos), heads * dh), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    assert lib.sh_rope_pos(A(Y), A(X), A(P), C.byref(shops.rope_plan(A(step), rot, layout)), len(pos), heads, dh, heads * dh, heads * dh) == 0, shops.last_error()
    i = np.arange(rot // 2)
    i, j = (i, i + rot // 2) if layout == R.HALF else (2 * i, 2 * i + 1)
    got, v = (a.astype(np.float64).reshape(len(pos), heads, dh) for a in (to_np(Y), x))
    for r, p in enumerate(pos):
        a = np.array([float(t * int(p) % 1) for t in _turns(*plan)]) * 2 * np.pi          # (whole turns fall off in fifty digits)
        c, s = np.cos(a), np.sin(a)
        both = np.abs(v[r][:, i]) + np.abs(v[r][:, j])
        for col, want in ((i, v[r][:, i] * c - v[r][:, j] * s), (j, v[r][:, j] * c + v[r][:, i] * s)):
            tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (3 * 2.0 ** -24 + 2.0 ** -36 + 2 * np.pi * BOUND * int(p)) * both
            assert (np.abs(got[r][:, col] - want) <= tol).all(), int(p)
