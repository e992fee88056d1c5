"""sh_rope_steps, sh_rope_pos and sh_kv_append_rope on the GPU against 64 bits (oracle/rope_mx4_refs.py, oracle/kv_refs.py)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from conftest import _KEEP, codes, to_dev, to_np
from oracle import kv_refs as K
from oracle import rope_mx4_refs as R
from softhier_mlir_amd import shops

pytestmark = pytest.mark.gpu
A = shops.addr


def dev(a):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    _KEEP.append(t)
    return t


def _plan(step, layout, mscale=1.0):
    return C.byref(shops.rope_plan(A(dev(step.view(np.int64))), 2 * len(step), layout, mscale))


def _turn(lib, x, step, pos, heads, dh, layout, mscale=1.0, pad=0, off=0, in_place=False):
    """The call with rows `pad` wider than they need be and bases `off` halves off the allocation; what must not be written is checked."""
    import torch
    rows, wide = x.shape
    X = torch.full((off + rows * (wide + pad),), 5.0, dtype=torch.float16, device="cuda")
    X[off:].view(rows, -1)[:, :wide] = to_dev(x)
    Y, ldy = (X, wide + pad) if in_place else (torch.full((off + rows * (wide + 2 * pad),), 9.0, dtype=torch.float16, device="cuda"), wide + 2 * pad)
    _KEEP.extend([X, Y])
    before = to_np(Y).copy()
    assert lib.sh_rope_pos(A(Y, off), A(X, off), A(dev(pos)), _plan(step, layout, mscale), rows, heads, dh, ldy, wide + pad) == 0, shops.last_error()
    y = to_np(Y)
    assert np.array_equal(y[:off], before[:off])
    y, b = y[off:].reshape(rows, ldy), before[off:].reshape(rows, ldy)
    assert np.array_equal(y[:, wide:], b[:, wide:])
    assert np.array_equal(y[pos < 0].view(np.uint16), b[pos < 0].view(np.uint16))
    return y[:, :wide]


def _check(got, x, step, pos, heads, dh, layout, mscale=1.0):
    """One rounding to fp16 (half a step, 2^-11 of the value, 2^-25 where that is subnormal); before it cosine and sine are rounded to fp32 and lie
    2^-37 off, two products and their sum are rounded: 3 x 2^-24 of |x1 c| + |x2 s| at most, which is below mscale (|x1| + |x2|)."""
    want = R.turn(x, step, pos, heads, dh, layout, mscale)
    size = np.abs(x.astype(np.float64)).reshape(len(pos), heads, dh)
    n = len(step)
    i = np.arange(n)
    i, j = (i, i + n) if layout == R.HALF else (2 * i, 2 * i + 1)
    both = np.zeros_like(size)
    both[:, :, i] = both[:, :, j] = (size[:, :, i] + size[:, :, j]) * abs(mscale)
    live = pos >= 0
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + (3 * 2.0 ** -24 + 2.0 ** -36) * both.reshape(len(pos), -1)
    err = np.abs(got.astype(np.float64) - want)
    assert (err[live] <= tol[live]).all(), float(np.nanmax((err - tol)[live]))
    kept = np.ones(dh, bool)
    kept[: 2 * n] = False
    same = np.tile(kept, heads)
    assert np.array_equal(got[live][:, same].view(np.uint16), x[live][:, same].view(np.uint16))


SHAPES = [(1, 1, 2, 2), (1, 15, 64, 64), (3, 5, 72, 72), (5, 2, 80, 20), (64, 40, 128, 128), (33, 3, 96, 24), (7, 4, 128, 64), (2, 1, 256, 256),
          (900, 40, 128, 64), (6, 3, 10, 6), (9, 2, 18, 14), (1, 64, 80, 80), (1030, 33, 144, 48), (300, 1, 48, 40), (17, 7, 128, 126)]


@pytest.mark.parametrize("layout", [R.HALF, R.PAIRS])
@pytest.mark.parametrize("rows,heads,dh,rot", SHAPES)
def test_rows(lib, gpu, rows, heads, dh, rot, layout):
    rng = np.random.default_rng(rows + rot)
    x = rng.standard_normal((rows, heads * dh)).astype(np.float16)
    step = R.steps(R.frequencies(rot, 1e4))
    pos = rng.integers(0, 131072, rows).astype(np.int32)
    pos[rng.random(rows) < 0.1] = -1
    _check(_turn(lib, x, step, pos, heads, dh, layout), x, step, pos, heads, dh, layout)


@pytest.mark.parametrize("layout", [R.HALF, R.PAIRS])
@pytest.mark.parametrize("pad,off,in_place", [(1, 1, False), (8, 3, False), (3, 2, True), (0, 0, True)])
@pytest.mark.parametrize("rows,heads,dh,rot", [(5, 3, 64, 32), (4, 2, 24, 20), (1100, 33, 128, 96)])
def test_strides_alignment_in_place(lib, gpu, rows, heads, dh, rot, pad, off, in_place, layout):
    rng = np.random.default_rng(pad + rot)
    x = rng.standard_normal((rows, heads * dh)).astype(np.float16)
    step = R.steps(R.frequencies(rot, 5e5))
    pos = np.arange(rows, dtype=np.int32) * 7 - 14
    if in_place:                                                    # a row that is left holds x
        got = _turn(lib, x, step, pos, heads, dh, layout, pad=pad, off=off, in_place=True)
        assert np.array_equal(got[pos < 0].view(np.uint16), x[pos < 0].view(np.uint16))
    else:
        got = _turn(lib, x, step, pos, heads, dh, layout, pad=pad, off=off)
    _check(got, x, step, pos, heads, dh, layout)


@pytest.mark.parametrize("mscale", [1.0, 1.25, -0.5, 0.0])
def test_far_positions_and_mscale(lib, gpu, mscale):
    """Positions up to the largest: whole turns fall off, so far ones are as exact as near ones."""
    rng = np.random.default_rng(3)
    pos = np.array([0, 1, 2, 3, 1 << 20, (1 << 24) + 1, (1 << 30) - 1, 2 ** 31 - 1, 123456789], np.int32)
    x = rng.standard_normal((len(pos), 2 * 64)).astype(np.float16)
    for base in (1e4, 1.5):
        step = R.steps(R.frequencies(64, base))
        _check(_turn(lib, x, step, pos, 2, 64, R.HALF, mscale), x, step, pos, 2, 64, R.HALF, mscale)


def test_quarter_turns_are_exact(lib, gpu):
    """Steps of 1/8 of a turn: every second position turns by a quarter, with cosine and sine 0 or 1."""
    x = np.random.default_rng(1).standard_normal((16, 8)).astype(np.float16)
    step = np.full(4, 1 << 61, np.uint64)
    pos = np.arange(0, 32, 2, dtype=np.int32)
    got = _turn(lib, x, step, pos, 1, 8, R.PAIRS).reshape(16, 4, 2)
    a, b = x.reshape(16, 4, 2)[..., 0], x.reshape(16, 4, 2)[..., 1]
    for r in range(16):
        want = [(a[r], b[r]), (-b[r], a[r]), (-a[r], -b[r]), (b[r], -a[r])][r % 4]
        assert np.array_equal(got[r, :, 0], want[0]) and np.array_equal(got[r, :, 1], want[1])


def test_specials_stay_in_their_pair(lib, gpu):
    x = np.ones((2, 64), np.float16)
    x[0, 3], x[1, 20] = np.nan, np.inf
    step = R.steps(R.frequencies(32, 1e4))
    got = _turn(lib, x, step, np.array([5, 9], np.int32), 1, 64, R.HALF)
    bad = ~np.isfinite(got)
    assert np.argwhere(bad).tolist() == [[0, 3], [0, 19], [1, 4], [1, 20]]
    assert np.isfinite(_turn(lib, np.full((1, 64), 65504, np.float16), step, np.array([0], np.int32), 1, 64, R.PAIRS)).all()


@pytest.mark.parametrize("rot,base,scaling,factor,lo,hi,ctx", [
    (128, 1e4, R.NONE, 0.0, 0.0, 0.0, 0), (64, 5e5, R.LINEAR, 4.0, 0.0, 0.0, 0), (128, 5e5, R.BANDS, 8.0, 1.0, 4.0, 8192), (20, 1e4, R.BANDS, 32.0, 0.5, 8.0, 2048),
    (64, 1e4, R.RAMP, 40.0, 1.0, 32.0, 4096), (128, 1e6, R.RAMP, 4.0, 1.0, 32.0, 32768), (2, 1e4, R.RAMP, 2.0, 1.0, 32.0, 100), (1024, 10.0, R.LINEAR, 0.5, 0, 0, 0)])
def test_steps(lib, gpu, rot, base, scaling, factor, lo, hi, ctx):
    """Turns a position to 2^-45 of their value (powers, logarithms and divisions in 64 bits, a few of 2^-53 each, times log(base)),
    and to 2^-65, because a step is a whole number of 2^-64 turns."""
    import torch
    t = torch.full((rot // 2 + 1,), -7, dtype=torch.int64, device="cuda")
    assert lib.sh_rope_steps(A(t), rot, base, scaling, factor, lo, hi, ctx) == 0, shops.last_error()
    got = to_np(t)
    assert got[-1] == -7
    w = R.frequencies(rot, base, scaling, factor, lo, hi, ctx) / (2 * np.pi)
    assert (np.abs(got[:-1].view(np.uint64).astype(np.float64) * 2.0 ** -64 - w) <= 2.0 ** -45 * w + 2.0 ** -65).all()


def test_rows_far_apart(lib, gpu):
    """A leading dim with which offsets pass 32 bits, in the builds for few and for many columns."""
    import torch
    rng = np.random.default_rng(8)
    far = (1 << 32) // 50
    for heads, dh, rot in ((3, 64, 64), (2, 20, 14)):
        x = rng.standard_normal((60, heads * dh)).astype(np.float16)
        step, pos = R.steps(R.frequencies(rot, 1e4)), np.arange(60, dtype=np.int32) * 1000
        X, Y = (torch.zeros((60, far), dtype=torch.float16, device="cuda") for _ in "xy")
        X[:, : heads * dh] = to_dev(x)
        torch.cuda.synchronize()
        assert lib.sh_rope_pos(A(Y), A(X), A(dev(pos)), _plan(step, R.PAIRS), 60, heads, dh, far, far) == 0, shops.last_error()
        _check(to_np(Y[:, : heads * dh].contiguous()), x, step, pos, heads, dh, R.PAIRS)


# ---- sh_kv_append_rope ----------------------------------------------------------------------------------------------
class Cache:
    def __init__(self, rng, pages, hkv, dh, bs, fmt, pad=0):
        import torch
        pg = hkv * bs * dh + 16 * pad
        raw = rng.integers(0, 120, (2, pages * pg)).astype(np.uint8)
        self.k, self.v = (dev(raw[i]) for i in (0, 1))
        self.ks, self.vs = (dev(np.exp2(rng.integers(-9, -5, (pages, hkv + pad))).astype(np.float32)) for _ in "kv")
        self.c = shops.kv_cache(A(self.k), A(self.v), A(self.ks), A(self.vs), pages, hkv, dh, bs, fmt, pg, pg, hkv + pad)
        self.t = (self.k, self.v, self.ks, self.vs)
        torch.cuda.synchronize()

    def bits(self):
        return [to_np(t).view(np.uint8) for t in self.t]


def _rows(rng, bs, pages, counts, idle=0, far=100000):
    """Slots and positions of requests that add `counts` rows each, from anywhere in a page; idle rows behind."""
    perm, slots, pos, n = rng.permutation(pages), [], [], 0
    for c in counts:
        off = int(rng.integers(0, bs)) if rng.random() < 0.7 else 0
        slots += [int(perm[n + p // bs]) * bs + p % bs for p in range(off, off + c)]
        p0 = int(rng.integers(0, far))
        pos += range(p0, p0 + c)
        n += (off + c - 1) // bs + 1
    assert n <= pages
    return np.array(slots + [-1] * idle, np.int32), np.array(pos + [-1] * idle, np.int32)


def _both(lib, seed, counts, H, hkv, dh, bs, fmt, rot, layout, idle=0, pages=None, pad=0, off=0, mscale=1.0, edit=None, in_place=False):
    """The one call and the three that it stands for, on two caches that begin alike: the same bits. Returns what the first wrote."""
    import torch
    rng = np.random.default_rng(seed)
    pages = pages or sum(c // bs + 2 for c in counts) + 1
    slots, pos = _rows(rng, bs, pages, counts, idle)
    rows, nq, nk = len(slots), H * dh, hkv * dh
    x = rng.standard_normal((rows, nq + 2 * nk)).astype(np.float16)
    if edit:
        edit(x, slots, pos)
    wide = nq + 2 * nk + pad
    xp = np.zeros(off + rows * wide, np.float16)
    xp[off:].reshape(rows, wide)[:, : nq + 2 * nk] = x
    step = R.steps(R.frequencies(rot, 1e4))
    plan, S, P = _plan(step, layout, mscale), dev(slots), dev(pos)
    one, two = (Cache(np.random.default_rng(seed + 1), pages, hkv, dh, bs, fmt, pad) for _ in "ab")
    X = to_dev(xp)
    Q = X if in_place else torch.full((rows, nq + pad), 3.0, dtype=torch.float16, device="cuda")
    X2 = X.clone()
    q2 = torch.full((rows, nq + pad), 3.0, dtype=torch.float16, device="cuda")
    k2 = torch.zeros((rows, nk), dtype=torch.float16, device="cuda")
    _KEEP.extend([Q, X2, q2, k2])
    torch.cuda.synchronize()
    qa, ldq = (A(X, off), wide) if in_place else (A(Q), nq + pad)
    assert lib.sh_kv_append_rope(C.byref(one.c), plan, qa if H else 0, A(X, off) if H else 0, A(X, off + nq), A(X, off + nq + nk), A(P), A(S), rows, H, ldq, wide,
                                 wide, wide) == 0, shops.last_error()
    if H:
        assert lib.sh_rope_pos(A(q2), A(X2, off), A(P), plan, rows, H, dh, nq + pad, wide) == 0
    assert lib.sh_rope_pos(A(k2), A(X2, off + nq), A(P), plan, rows, hkv, dh, nk, wide) == 0
    S2 = dev(np.where(pos < 0, -1, slots).astype(np.int32))
    assert lib.sh_kv_append(C.byref(two.c), A(k2), A(X2, off + nq + nk), nk, wide, A(S2), rows) == 0
    for a, b, name in zip(one.bits(), two.bits(), ("k", "v", "ks", "vs")):
        assert np.array_equal(a, b), (name, int((a != b).sum()))
    if in_place:
        live = pos >= 0
        y = to_np(X)[off:].reshape(rows, wide)
        assert np.array_equal(y[live, :nq].view(np.uint16), codes(q2)[live, :nq])
        assert np.array_equal(y[:, nq:].view(np.uint16), xp[off:].reshape(rows, wide)[:, nq:].view(np.uint16))
        assert np.array_equal(y[~live].view(np.uint16), xp[off:].reshape(rows, wide)[~live].view(np.uint16))
    elif H:
        assert np.array_equal(codes(Q), codes(q2))
    return dict(slots=slots, pos=pos, x=x, step=step, cache=one, pages=pages)


APPENDS = [([1], 15, 5, 64, 16, 64), ([1] * 64, 32, 8, 128, 16, 128), ([4] * 7, 8, 1, 80, 16, 32), ([100, 1, 33], 4, 2, 96, 32, 24), ([300, 700], 8, 8, 128, 32, 64),
           ([2500, 2000, 41], 10, 5, 64, 64, 64), ([5, 60, 130], 2, 2, 256, 64, 256), ([37] * 30, 3, 3, 32, 16, 8), ([17, 2], 6, 6, 112, 64, 104), ([600], 1, 1, 16, 16, 16)]


@pytest.mark.parametrize("fmt", [shops.SH_INT8, shops.SH_FP8])
@pytest.mark.parametrize("layout", [R.HALF, R.PAIRS])
@pytest.mark.parametrize("counts,H,hkv,dh,bs,rot", APPENDS)
def test_append_is_the_three_calls(lib, gpu, counts, H, hkv, dh, bs, rot, layout, fmt):
    _both(lib, 5 + len(counts), counts, H, hkv, dh, bs, fmt, rot, layout, idle=len(counts) // 3)


@pytest.mark.parametrize("kw", [dict(pad=1, off=1), dict(pad=3, off=2, mscale=1.3), dict(H=0), dict(in_place=True), dict(in_place=True, pad=8, off=5), dict(idle=50)], ids=str)
def test_append_strides_and_queries(lib, gpu, kw):
    kw = {**dict(H=6), **kw}
    H = kw.pop("H")
    for counts in ([3, 1, 40], [700, 1]):
        _both(lib, 9, counts, H, 3, 64, 16, shops.SH_FP8, 32, R.HALF, **kw)


def test_append_rows_between_that_are_skipped(lib, gpu):
    """Rows at negative positions with a good slot, and rows at good positions without one: neither is stored; the queries of the latter are turned."""
    def edit(x, slots, pos):
        pos[[0, 45]] = -1
        slots[[1, 70]] = (1 << 20, -5)
    _both(lib, 11, [1] * 90, 4, 2, 64, 16, shops.SH_INT8, 64, R.HALF, edit=edit)


def test_append_specials(lib, gpu):
    """NaN and infinities in keys (both columns of the pair are NaN then, stored as 0) and values."""
    def edit(x, slots, pos):
        x[2, 128 + 5], x[7, 128 + 64 + 9], x[3, 256 + 4], x[4, 256 + 70] = np.nan, np.inf, np.nan, -np.inf
    for layout in (R.HALF, R.PAIRS):
        _both(lib, 13, [12, 3], 2, 2, 64, 16, shops.SH_FP8, 64, layout, edit=edit)


@pytest.mark.parametrize("fmt", [shops.SH_INT8, shops.SH_FP8])
def test_append_against_numpy(lib, gpu, fmt):
    """Against 64-bit angles: the turned keys rounded to fp16, then the codes of oracle/kv_refs.py. A turned key may be one fp16 step off where it
    lies near a border of that rounding; so may then its code: each code is that of one of the three neighbouring halves."""
    hkv, dh, bs, H = 3, 64, 16, 3
    r = _both(lib, 17, [40, 1, 9], H, hkv, dh, bs, fmt, 32, R.HALF, pages=12)
    one, x, pages = r["cache"], r["x"], r["pages"]
    key = R.turn(x[:, H * dh: (H + hkv) * dh], r["step"], r["pos"], hkv, dh, R.HALF).astype(np.float16)
    fresh = Cache(np.random.default_rng(18), pages, hkv, dh, bs, fmt)
    k, v, ks, vs = fresh.bits()
    k, v = k.reshape(pages, hkv, bs, dh), v.reshape(pages, hkv, dh, bs)
    ks, vs = (s.view(np.float32).reshape(pages, hkv) for s in (ks, vs))
    got = one.bits()
    want = [K.append(k, v, ks, vs, np.nextafter(key, np.float16(t)) if t else key, x[:, (H + hkv) * dh:], r["slots"], fmt) for t in (0, np.inf, -np.inf)]
    gk = got[0].reshape(k.shape)
    assert ((gk == want[0][0]) | (gk == want[1][0]) | (gk == want[2][0])).all()
    assert np.array_equal(got[1].reshape(v.shape), want[0][1])
    assert np.array_equal(got[3].view(np.float32).reshape(vs.shape), want[0][3])
    assert np.mean(gk != want[0][0]) < 0.01


def test_append_in_a_graph(lib, gpu):
    """Captured as the first call of its kernel for this width, replayed with other rows, positions and slots: the bits of the eager calls."""
    import torch
    rng = np.random.default_rng(23)
    H, hkv, dh, bs, pages, rows = 4, 2, 192, 32, 40, 12
    step = R.steps(R.frequencies(96, 1e4))
    plan = _plan(step, R.PAIRS)
    nq, nk = H * dh, hkv * dh
    one, two = (Cache(np.random.default_rng(1), pages, hkv, dh, bs, shops.SH_FP8) for _ in "ab")
    X, S, P = to_dev(np.zeros((rows, nq + 2 * nk), np.float16)), dev(np.full(rows, -1, np.int32)), dev(np.full(rows, -1, np.int32))
    q = [torch.zeros((rows, nq), dtype=torch.float16, device="cuda") for _ in "ab"]

    def call(cache, yq):
        assert lib.sh_kv_append_rope(C.byref(cache.c), plan, A(yq), A(X), A(X, nq), A(X, nq + nk), A(P), A(S), rows, H, nq, nq + 2 * nk, nq + 2 * nk,
                                     nq + 2 * nk) == 0, shops.last_error()
    torch.cuda.synchronize()
    s, g, prev = torch.cuda.Stream(), torch.cuda.CUDAGraph(), lib.sh_get_stream()
    with torch.cuda.graph(g, stream=s):
        lib.sh_set_stream(s.cuda_stream)
        call(one, q[0])
    lib.sh_set_stream(prev)
    for i in range(4):
        slots, pos = _rows(rng, bs, pages, [1] * 5 + [4, 1], idle=2)
        X.copy_(torch.from_numpy(rng.standard_normal(X.shape).astype(np.float16)))
        S[: len(slots)] = torch.from_numpy(slots).cuda()
        P[: len(pos)] = torch.from_numpy(pos).cuda()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        call(two, q[1])
        assert np.array_equal(codes(q[0]), codes(q[1]))
        for a, b in zip(one.bits(), two.bits()):
            assert np.array_equal(a, b), i


def test_append_into_a_cache_of_gigabytes(lib, gpu):
    """Pages whose bytes lie past 32 bits: the bits that the same rows have in the first pages."""
    import torch
    rng = np.random.default_rng(31)
    H, hkv, dh, bs, pages = 2, 8, 128, 64, 70000
    nq, nk, wide = H * dh, hkv * dh, (H + 2 * hkv) * dh
    step = R.steps(R.frequencies(128, 1e4))
    plan = _plan(step, R.HALF)
    X, P = to_dev(rng.standard_normal((70, wide)).astype(np.float16)), dev(np.arange(5, 75, dtype=np.int32))
    k, v = (torch.zeros((pages, hkv * bs * dh), dtype=torch.uint8, device="cuda") for _ in "kv")
    ks, vs = (torch.zeros((pages, hkv), device="cuda") for _ in "kv")
    q = torch.zeros((70, nq), dtype=torch.float16, device="cuda")
    c = shops.kv_cache(A(k), A(v), A(ks), A(vs), pages, hkv, dh, bs, shops.SH_INT8)
    torch.cuda.synchronize()
    for first in (0, pages - 2):
        S = dev((first * bs + np.arange(70)).astype(np.int32))
        assert lib.sh_kv_append_rope(C.byref(c), plan, A(q), A(X), A(X, nq), A(X, nq + nk), A(P), A(S), 70, H, nq, wide, wide, wide) == 0, shops.last_error()
    for t in (k, v, ks, vs):
        assert torch.equal(t[:2], t[pages - 2:]) and bool((t[:2] != 0).any())
        assert not bool((t[2: pages - 2: 997] != 0).any())
