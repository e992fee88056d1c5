"""The 8-bit paged key / value cache on the GPU against its 64-bit definition (oracle/kv_refs.py): the step's tables and the
written codes exactly, attention within a bound derived from its roundings."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from conftest import _KEEP, to_dev, to_np
from oracle import kv_refs as R
from softhier_mlir_amd import shops

pytestmark = pytest.mark.gpu
A = shops.addr
INT8, FP8 = shops.SH_INT8, shops.SH_FP8


def dev(a):
    """A numpy array of any type on the GPU, kept alive for the test."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    _KEEP.append(t)
    return t


# ---- sh_kv_slots ----------------------------------------------------------------------------------------------------
def _slots_case(rng, B, ld, bs, pages, longest, ended, fill=0.5):
    """Requests with their pages in the table, the other pages in the ring from a random first entry."""
    cap = ld * bs
    lens = rng.integers(0, int(cap * fill) + 1, B).astype(np.int32)
    perm = rng.permutation(pages).astype(np.int32)
    table = np.full((B, ld), -1, np.int32)
    used = 0
    for b in range(B):
        n = -(-int(lens[b]) // bs)
        if used + n > pages:
            lens[b], n = 0, 0
        table[b, :n] = perm[used:used + n]
        used += n
    add = rng.integers(0, longest + 1, B).astype(np.int32)
    add[rng.random(B) < ended] = -1
    head, count = int(rng.integers(pages)), pages - used
    pool = np.full(pages, -1, np.int32)
    pool[(head + np.arange(count)) % pages] = perm[used:]
    return table, lens, add, pool, np.array([head, count, 0], np.int32)


def _run_slots(lib, table, lens, add, pool, state, bs, rows, in_place=False):
    t, le, ad, po, st = (dev(x) for x in (table, lens, add, pool, state))
    B, ld = table.shape
    lo, so = (le, st) if in_place else (dev(np.full(B, -9, np.int32)), dev(np.full(3, -9, np.int32)))
    rs, sl, ps, kl = (dev(np.full(n, -9, np.int32)) for n in (B + 1, rows + 3, rows + 3, B))
    assert lib.sh_kv_slots(A(t), ld, A(le), A(lo), A(ad), A(po), A(st), A(so), A(rs), A(sl), A(ps), A(kl), B, bs, len(pool), rows) == 0, shops.last_error()
    got = dict(table=t, pool=po, lens_out=lo, state_out=so, row_start=rs, slots=sl, pos=ps, kv_len=kl)
    got = {k: to_np(x) for k, x in got.items()}
    for k in ("slots", "pos"):
        assert (got[k][rows:] == -9).all()                           # nothing behind `rows`
        got[k] = got[k][:rows]
    if not in_place:
        assert np.array_equal(to_np(le), lens) and np.array_equal(to_np(st), state)
    return got


def _check_slots(got, want):
    for k, w in want.items():
        assert np.array_equal(got[k], w), k


@pytest.mark.parametrize("B,ld,bs,longest,ended,spare,in_place", [
    (1, 4, 16, 1, 0.0, 8, False), (1, 40, 16, 500, 0.0, 100, True), (7, 9, 64, 70, 0.3, 20, True), (64, 256, 16, 1, 0.0, 100, False),
    (64, 256, 16, 1, 0.2, 2, True), (1024, 8, 16, 2, 0.1, 300, True), (1025, 6, 32, 3, 0.1, 40, False), (3000, 5, 16, 9, 0.2, 900, True),
    (200, 300, 16, 2000, 0.1, 20000, False), (200, 300, 16, 2000, 0.1, 3000, True), (1300, 64, 64, 300, 0.2, 6000, True)])
@pytest.mark.parametrize("short", [0, 37])
def test_slots_exact(lib, gpu, B, ld, bs, longest, ended, spare, in_place, short):
    """Served, refused (pages, table width, rows) and ended requests, in one workgroup and in many; `short`: fewer row places
    than rows, or more."""
    rng = np.random.default_rng(B * 7 + ld + short)
    case = _slots_case(rng, B, ld, bs, pages := B * ld // 4 + spare, longest, ended)
    total = int(np.maximum(case[2], 0).sum())
    rows = total + 5 if not short else max(1, total - short)
    want = R.slots(*case, bs, rows)
    assert pages == len(case[3])
    _check_slots(_run_slots(lib, *case, bs, rows, in_place), want)


def test_slots_over_a_serving_run(lib, gpu):
    """Sixty steps in place on one set of arrays: prompts arrive, decode, end; their pages come round the ring again. After
    each step no page is owned twice."""
    rng = np.random.default_rng(5)
    B, ld, bs, pages, rows = 12, 8, 16, 40, 128
    table, lens = np.full((B, ld), -1, np.int32), np.zeros(B, np.int32)
    pool, state = np.arange(pages, dtype=np.int32), np.array([0, pages, 0], np.int32)
    refused = 0
    for step in range(60):
        add = np.where(lens == 0, np.where(rng.random(B) < 0.4, rng.integers(1, 60, B), 0), 1).astype(np.int32)
        add[(lens > 0) & (rng.random(B) < 0.15)] = -1
        want = R.slots(table, lens, add, pool, state, bs, rows)
        _check_slots(_run_slots(lib, table, lens, add, pool, state, bs, rows, True), want)
        table, pool, lens, state = (want[k] for k in ("table", "pool", "lens_out", "state_out"))
        refused += int(state[2])
        owned = [int(p) for b in range(B) for p in table[b, :-(-int(lens[b]) // bs)]]
        free = [int(pool[(state[0] + i) % pages]) for i in range(state[1])]
        assert sorted(owned + free) == list(range(pages))
    assert refused                                                   # the pool was too small at times


# ---- sh_kv_append ---------------------------------------------------------------------------------------------------
class Cache:
    """A cache on the GPU with its numpy copy; `pad` bytes / floats lie between pages."""

    def __init__(self, rng, pages, hkv, dh, bs, fmt, pad=0, values=False):
        self.pages, self.hkv, self.dh, self.bs, self.fmt = pages, hkv, dh, bs, fmt
        n = hkv * bs * dh
        self.pg, self.pgs = n + 16 * pad, hkv + pad
        raw = rng.integers(0, 256, (2, pages, self.pg)).astype(np.uint8)
        if fmt == FP8 and values:
            raw[(raw & 127) == 127] = 1
        sc = np.exp2(rng.integers(-9, -4, (2, pages, self.pgs))).astype(np.float32)
        self.raw, self.sc = raw, sc
        self.dk, self.dv, self.dks, self.dvs = dev(raw[0]), dev(raw[1]), dev(sc[0]), dev(sc[1])
        self.c = shops.kv_cache(A(self.dk), A(self.dv), A(self.dks), A(self.dvs), pages, hkv, dh, bs, fmt, self.pg if pad else 0,
                                self.pg if pad else 0, self.pgs if pad else 0)

    def host(self, raw, sc):
        n = self.hkv * self.bs * self.dh
        k = raw[0][:, :n].reshape(self.pages, self.hkv, self.bs, self.dh).copy()
        v = raw[1][:, :n].reshape(self.pages, self.hkv, self.dh, self.bs).copy()
        return k, v, sc[0][:, :self.hkv].copy(), sc[1][:, :self.hkv].copy()

    def before(self):
        return self.host(self.raw, self.sc)

    def now(self):
        raw, sc = [to_np(self.dk), to_np(self.dv)], [to_np(self.dks), to_np(self.dvs)]
        n = self.hkv * self.bs * self.dh
        for i in range(2):                                           # between the pages nothing is written
            assert np.array_equal(raw[i][:, n:], self.raw[i][:, n:]) and np.array_equal(sc[i][:, self.hkv:], self.sc[i][:, self.hkv:])
        return self.host(raw, sc)


def _slots_of(rng, runs, pages, bs):
    """Rows of requests that begin at offset `held` of a page of their own and add n tokens; -1 rows between some."""
    perm, at, out = rng.permutation(pages), 0, []
    for held, n in runs:
        if n < 0:
            out += [-1] * -n
            continue
        need = (held + n - 1) // bs + 1
        pg = perm[at:at + need]
        at += need
        out += [int(pg[p // bs]) * bs + p % bs for p in range(held, held + n)]
    return np.array(out, np.int32)


APPENDS = [
    dict(hkv=1, dh=16, bs=16, runs=[(0, 1)]),
    dict(hkv=8, dh=128, bs=16, runs=[(i % 16, 1) for i in range(33)]),
    dict(hkv=5, dh=64, bs=16, runs=[(0, 100), (-1, -1), (15, 1), (3, 13), (3, 14), (-2, -2), (0, 16), (8, 40)]),
    dict(hkv=2, dh=80, bs=32, runs=[(31, 2), (0, 64), (5, 3), (0, 33), (1, 31)]),
    dict(hkv=3, dh=96, bs=64, runs=[(0, 64), (63, 130), (10, 5), (0, 1)]),
    dict(hkv=2, dh=256, bs=64, runs=[(0, 150), (7, 64)]),
    dict(hkv=1, dh=32, bs=64, runs=[(64 * 0 + 33, 3000), (0, 700)]),
    dict(hkv=8, dh=64, bs=32, runs=[(0, 2500), (5, 2600), (0, 31)]),
]


@pytest.mark.parametrize("fmt", [INT8, FP8])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{c['hkv']}x{c['dh']}_bs{c['bs']}")
def test_append_exact(lib, gpu, case, fmt):
    """Codes and scales bit for bit, older tokens rounded again where a scale grew, everything else as it was; NaN,
    infinities, zero rows and the smallest halves among the values; odd leading dims and bases."""
    rng = np.random.default_rng(case["dh"] + case["bs"])
    hkv, dh, bs, runs = (case[k] for k in ("hkv", "dh", "bs", "runs"))
    pages = sum((h + n - 1) // bs + 1 for h, n in runs if n > 0) + 4
    slot = _slots_of(rng, runs, pages, bs)
    rows, n = len(slot), hkv * dh
    ld = n + 3
    buf = rng.standard_normal((2, rows, ld)) * np.exp2(rng.integers(-10, 6, (2, rows, 1)))
    buf = buf.astype(np.float16)
    buf[:, rows // 2, : dh // 2] = 0
    if rows > 4:
        buf[0, 1, :3] = [np.nan, np.inf, -np.inf]
        buf[1, 2, :2] = [6e-8, -6e-8]
        buf[1, 3, :n] = 0
        buf[0, rows - 1, :2] = [65504, -65504]
    c = Cache(rng, pages, hkv, dh, bs, fmt, pad=1, values=True)
    x = np.concatenate([np.zeros(1, np.float16), buf.ravel()])      # a base off the 16-byte grid
    X = to_dev(x)
    S = dev(slot)
    assert lib.sh_kv_append(C.byref(c.c), A(X, 1), A(X, 1 + rows * ld), ld, ld, A(S), rows) == 0, shops.last_error()
    want = R.append(*c.before(), buf[0][:, :n], buf[1][:, :n], slot, fmt)
    for name, g, w in zip(("k", "v", "ks", "vs"), c.now(), want):
        if fmt == FP8 and g.dtype == np.uint8:                       # a zero may carry either sign
            g, w = (np.where(t == 128, 0, t) for t in (g, w))
        assert np.array_equal(g, w), (name, np.argwhere(g != w)[:4])
    # the same rows at the same slots again: the same codes
    assert lib.sh_kv_append(C.byref(c.c), A(X, 1), A(X, 1 + rows * ld), ld, ld, A(S), rows) == 0
    for g, w in zip(c.now(), want):
        if fmt == FP8 and g.dtype == np.uint8:
            g, w = (np.where(t == 128, 0, t) for t in (g, w))
        assert np.array_equal(g, w)


@pytest.mark.parametrize("fmt", [INT8, FP8])
def test_append_to_scales_of_another_kind(lib, gpu, fmt):
    """Pages whose scales are no powers of two: new codes are the correctly rounded quotients, and the scale stays where it suffices."""
    rng = np.random.default_rng(37)
    hkv, dh, bs, pages = 4, 64, 16, 40
    c = Cache(rng, pages, hkv, dh, bs, fmt, values=True)
    host = list(c.before())
    host[2], host[3] = (rng.uniform(0.004, 0.2, (pages, hkv)).astype(np.float32) for _ in "kv")
    c.dks.copy_(dev(host[2])); c.dvs.copy_(dev(host[3]))             # noqa: E702
    c.sc = np.stack(host[2:])
    slot = np.concatenate([p * bs + np.arange(int(rng.integers(1, bs)), bs) for p in rng.permutation(pages)]).astype(np.int32)
    x = rng.standard_normal((2, len(slot), hkv * dh)).astype(np.float16)
    X, S = to_dev(x), dev(slot)
    want = R.append(*host, x[0], x[1], slot, fmt)
    assert (want[2] == host[2]).any() and (want[2] != host[2]).any()
    assert lib.sh_kv_append(C.byref(c.c), A(X), A(X, x[0].size), hkv * dh, hkv * dh, A(S), len(slot)) == 0
    for name, g, w in zip(("k", "v", "ks", "vs"), c.now(), want):
        if fmt == FP8 and g.dtype == np.uint8:
            g, w = (np.where(t == 128, 0, t) for t in (g, w))
        bad = g != w
        # the quotient is rounded to fp32 before it is rounded to a code: a value next to a code's border may fall on it
        assert bad.mean() <= 1e-4, (name, int(bad.sum()))


@pytest.mark.parametrize("fmt", [INT8, FP8])
def test_append_skips_slots_outside_the_cache(lib, gpu, fmt):
    rng = np.random.default_rng(3)
    c = Cache(rng, 3, 2, 32, 16, fmt, values=True)
    slot = np.array([-1, 48, 2 ** 31 - 1, -(2 ** 31), 5, 47, 100], np.int32)
    x = rng.standard_normal((2, 7, 64)).astype(np.float16)
    X, S = to_dev(x), dev(slot)
    assert lib.sh_kv_append(C.byref(c.c), A(X), A(X, 7 * 64), 64, 64, A(S), 7) == 0
    for g, w in zip(c.now(), R.append(*c.before(), x[0], x[1], slot, fmt)):
        assert np.array_equal(np.where(g == 128, 0, g) if g.dtype == np.uint8 else g, np.where(w == 128, 0, w) if w.dtype == np.uint8 else w)


# ---- sh_attention_kv -------------------------------------------------------------------------------------------------
def bound(o, reach, spread, dh, L, vmax):
    """Largest error of an fp16 result: its own rounding (half a step, 2^-11); a probability's rounding to fp16 (2^-11 of it);
    an error d of a score changes its probability by the factor e^d, twice where the sum's is counted: fp32 sums of dh
    exact products and four more fp32 operations, 2^-23 of sum |q||k| each; exp2 (2^-22); the fp16 floor 2^-25, and 2^-25 of
    2^-13 of the value scales for each key."""
    d = (dh + 8) * 2.0 ** -23 * spread + 2.0 ** -21
    return 2.0 ** -11 * np.abs(o) + reach * (2.0 ** -11 + 2 * d + L * 2.0 ** -24) + 2.0 ** -24 + L * 2.0 ** -37 * vmax


def _attend(lib, c, q, table, kv_len, row_start, H, scale, window=0, max_q=None, ldq=None, rows=None, host=None, off=0):
    import torch
    rows = q.shape[0] if rows is None else rows
    D = H * c.dh
    ldq = ldq or D
    Q = np.full((q.shape[0], ldq), np.nan, np.float16)
    Q[:, :D] = q
    Qd = to_dev(np.concatenate([np.zeros(off, np.float16), Q.ravel()]))
    O = torch.full((q.shape[0], ldq), 7.0, dtype=torch.float16, device="cuda")
    T, Ln = dev(table), dev(np.asarray(kv_len, np.int32))
    Rs = dev(np.asarray(row_start, np.int32)) if row_start is not None else None
    if max_q is None:
        max_q = 1 if row_start is None else max(1, int(np.diff(row_start).max()))
    B, ld = table.shape
    need = lib.sh_attention_kv_ws_bytes(C.byref(c.c), B, rows, max_q, H, ld)
    ws = torch.full((int(need) + 64,), 255, dtype=torch.uint8, device="cuda")     # NaN wherever it is read before written
    rc = lib.sh_attention_kv(A(Qd, off), A(O), C.byref(c.c), A(T), ld, A(Ln), A(Rs) if Rs is not None else 0, B, rows, max_q, H, ldq, ldq, scale,
                             window, A(ws), need)
    assert rc == 0, shops.last_error()
    o = to_np(O).astype(np.float64)
    assert (to_np(ws)[int(need):] == 255).all()
    k, v, ks, vs = host or c.before()
    want, reach, spread = R.attention(q, k, v, ks, vs, table, kv_len, row_start, H, scale, c.fmt, window, max_q)
    none = np.isnan(want).all(1)
    assert (o[none] == 7.0).all() and (o[:, D:] == 7.0).all()               # rows of no request and other columns: untouched
    vmax = 127 * vs.max() if c.fmt == INT8 else 448 * vs.max()
    tol = bound(want, reach, spread, c.dh, int(max(kv_len)), vmax)
    err = np.abs(o[:, :D] - want)
    bad = ~none[:, None] & ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float(err[bad].max()), float(tol[bad].min()), np.argwhere(bad)[:5].tolist())
    return o[:, :D]


def _table(rng, kv_len, bs, pages, ld=None):
    need = [-(-n // bs) for n in kv_len]
    ld = ld or max(1, max(need))
    perm = rng.permutation(pages)[: sum(need)]
    t = np.full((len(kv_len), ld), -7, np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = perm[at:at + n]
        at += n
    return t


ATTNS = [   # H, hkv, dh, bs, lengths, new rows
    (1, 1, 16, 16, [1], None),
    (15, 5, 64, 16, [937], None),
    (8, 8, 128, 16, [1, 2, 15, 16, 17, 63, 64, 65, 0, 127], None),
    (32, 8, 128, 16, [3000, 5, 700], None),
    (16, 1, 64, 64, [129, 64, 1], None),
    (7, 1, 80, 32, [400, 33], None),
    (24, 1, 64, 32, [300, 31], None),                       # more than 16 heads on one
    (64, 2, 32, 16, [77], None),
    (4, 2, 256, 16, [513, 90], None),
    (6, 2, 96, 64, [200, 1000], None),
    (8, 2, 128, 32, [50, 300, 4, 64], [4, 4, 4, 4]),          # drafts: sixteen rows exactly
    (6, 2, 64, 16, [50, 300, 4], [5, 1, 3]),
    (4, 4, 128, 16, [200, 90, 64], [70, 0, 64]),              # chunks, a request without rows
    (8, 2, 64, 16, [333, 7, 130], [100, 7, 130]),             # prompts from their first token
    (15, 5, 64, 32, [260], [51]),
    (2, 1, 256, 32, [150], [33]),
    (3, 3, 48, 16, [40, 10], [3, 12]),                        # more rows than keys: the first two see none
    (16, 2, 128, 16, [150, 600, 20], [150, 1, 3]),
    (4, 1, 64, 16, [6000, 3], [20, 1]),                       # few rows over a long context: its keys in parts
    (8, 1, 128, 64, [2600, 900], [9, 17]),
    (4, 2, 112, 32, [1500], [40]),
    (12, 1, 256, 16, [900, 1], [30, 1]),
    (1, 1, 16, 16, [700], [700]),
]


@pytest.mark.parametrize("fmt", [INT8, FP8])
@pytest.mark.parametrize("case", ATTNS, ids=lambda c: f"h{c[0]}k{c[1]}d{c[2]}bs{c[3]}L{c[4][0]}" + (f"q{c[5][0]}" if c[5] else ""))
def test_attention(lib, gpu, case, fmt):
    H, hkv, dh, bs, L, new = case
    rng = np.random.default_rng(H * dh + sum(L))
    pages = sum(-(-n // bs) for n in L) + 3
    c = Cache(rng, pages, hkv, dh, bs, fmt, pad=1, values=True)
    start = None if new is None else np.concatenate([[0], np.cumsum(new)])
    rows = len(L) if new is None else int(start[-1])
    q = rng.standard_normal((rows, H * dh)).astype(np.float16)
    _attend(lib, c, q, _table(rng, L, bs, pages), L, start, H, dh ** -0.5, ldq=H * dh + 5, off=1)


@pytest.mark.parametrize("window", [1, 15, 64, 100, 5000])
@pytest.mark.parametrize("new", [None, [1, 4, 3], [1, 40, 3]])
def test_attention_window(lib, gpu, window, new):
    """Pages before every window hold NaN codes and scales and have table entries outside the cache: nothing of them is seen."""
    rng = np.random.default_rng(window)
    L, bs, dh, H, hkv = [400, 130, 64], 16, 64, 4, 2
    pages = sum(-(-n // bs) for n in L) + 3
    c = Cache(rng, pages, hkv, dh, bs, FP8, values=True)
    table = _table(rng, L, bs, pages)
    host = c.before()
    for b, n in enumerate(L):
        first = n - (new[b] if new else 1) + 1 - window
        for j in range(max(0, first) // bs):
            pg = table[b, j]
            host[0][pg], host[1][pg], host[2][pg], host[3][pg] = 0x7F, 0xFF, np.nan, np.nan
            if j % 2:
                table[b, j] = -1 if j % 4 == 1 else pages + 5
    c.dk.copy_(dev(host[0].reshape(pages, -1))); c.dv.copy_(dev(host[1].reshape(pages, -1)))   # noqa: E702
    c.dks.copy_(dev(host[2])); c.dvs.copy_(dev(host[3]))                                       # noqa: E702
    clean = [np.where((h & 127) == 127, 0, h).astype(np.uint8) if h.dtype == np.uint8 else np.nan_to_num(h) for h in host]
    start = None if new is None else np.concatenate([[0], np.cumsum(new)])
    q = rng.standard_normal((3 if new is None else sum(new), H * dh)).astype(np.float16)
    _attend(lib, c, q, table, L, start, H, 0.125, window=window, host=clean)


@pytest.mark.parametrize("fmt", [INT8, FP8])
def test_attention_behind_the_last_key(lib, gpu, fmt):
    """The rest of the last page and pages the table names by mistake hold NaN codes and infinite scales: left out."""
    rng = np.random.default_rng(11)
    L, bs, dh, H, hkv = [37, 5, 64, 200], 16, 128, 8, 2
    pages = sum(-(-n // bs) for n in L) + 3
    c = Cache(rng, pages, hkv, dh, bs, fmt, values=True)
    table = _table(rng, L, bs, pages, ld=16)
    host = c.before()
    clean = [h.copy() for h in host]
    for b, n in enumerate(L):
        if n % bs:
            host[0][table[b, n // bs], :, n % bs:], host[1][table[b, n // bs], :, :, n % bs:] = 0x7F, 0xFF
    gone = table[3, 3]
    host[0][gone], host[1][gone], host[2][gone], host[3][gone] = 0x7F, 0x7F, np.inf, np.nan
    table[3, 3], table[3, 9] = -5, 2 ** 31 - 1
    c.dk.copy_(dev(host[0].reshape(pages, -1))); c.dv.copy_(dev(host[1].reshape(pages, -1)))   # noqa: E702
    c.dks.copy_(dev(host[2])); c.dvs.copy_(dev(host[3]))                                       # noqa: E702
    q = rng.standard_normal((4, H * dh)).astype(np.float16)
    _attend(lib, c, q, table, L, None, H, dh ** -0.5, host=clean)


def test_attention_lengths_out_of_range(lib, gpu):
    """Negative lengths are 0 (zeros), lengths beyond the table end at it; every page outside the cache: zeros."""
    rng = np.random.default_rng(13)
    c = Cache(rng, 8, 2, 64, 16, INT8)
    table = _table(rng, [48, 48], 16, 8, ld=3)
    table = np.concatenate([table, np.full((1, 3), 8, np.int32)])
    q = rng.standard_normal((3, 4 * 64)).astype(np.float16)
    o = _attend(lib, c, q, table, [-4, 1000, 40], None, 4, 0.125)
    assert (o[0] == 0).all() and (o[2] == 0).all()


def test_attention_max_q_and_rows_bound_what_is_written(lib, gpu):
    """A request with more rows than max_q: its first max_q rows, at their own positions. Rows at and behind `rows` stay."""
    rng = np.random.default_rng(17)
    c = Cache(rng, 20, 2, 64, 16, INT8)
    table = _table(rng, [100, 90], 16, 20)
    q = rng.standard_normal((60, 4 * 64)).astype(np.float16)
    _attend(lib, c, q, table, [100, 90], np.array([0, 40, 60]), 4, 0.125, max_q=7)
    _attend(lib, c, q, table, [100, 90], np.array([0, 40, 60]), 4, 0.125, max_q=0xFFFFFFFF)
    _attend(lib, c, q[:5], table, [100, 90], np.array([0, 3, 5]), 4, 0.125, max_q=0xFFFFFFFF, window=0xFFFFFFFF)
    import torch
    O = torch.full((60, 256), 7.0, dtype=torch.float16, device="cuda")
    Q, T, Ln, Rs = to_dev(q), dev(table), dev(np.array([100, 90], np.int32)), dev(np.array([0, 40, 60], np.int32))
    need = lib.sh_attention_kv_ws_bytes(C.byref(c.c), 2, 50, 40, 4, table.shape[1])
    ws = torch.empty(int(need), dtype=torch.uint8, device="cuda")
    assert lib.sh_attention_kv(A(Q), A(O), C.byref(c.c), A(T), table.shape[1], A(Ln), A(Rs), 2, 50, 40, 4, 256, 256, 0.125, 0, A(ws), need) == 0
    o = to_np(O)
    assert (o[50:] == 7.0).all() and (o[:50] != 7.0).any(1).all()


@pytest.mark.parametrize("fmt", [INT8, FP8])
def test_attention_scales_far_apart(lib, gpu, fmt):
    """Value scales from 2^-30 to 2^9 from page to page, key scales that make scores of hundreds."""
    rng = np.random.default_rng(19)
    L, bs, dh, H, hkv = [700, 64], 16, 64, 8, 2
    pages = sum(-(-n // bs) for n in L) + 1
    c = Cache(rng, pages, hkv, dh, bs, fmt, values=True)
    host = list(c.before())
    host[3] = np.exp2(rng.integers(-30, 5 if fmt == FP8 else 9, host[3].shape)).astype(np.float32)
    host[3][::7] = 0.0
    host[2] = np.exp2(rng.integers(-9, 0, host[2].shape)).astype(np.float32)
    c.dks.copy_(dev(host[2])); c.dvs.copy_(dev(host[3]))             # noqa: E702
    q = rng.standard_normal((2, H * dh)).astype(np.float16)
    o = _attend(lib, c, q, _table(rng, L, bs, pages), L, None, H, 0.125, host=host)
    assert np.isfinite(o).all()


@pytest.mark.parametrize("fmt", [INT8, FP8])
@pytest.mark.parametrize("H,hkv,dh", [(4, 2, 32), (15, 5, 64), (4, 4, 80), (7, 1, 112), (8, 1, 128), (2, 1, 256), (16, 1, 64), (24, 2, 80)])
def test_attention_probabilities_keep_their_precision(lib, gpu, fmt, H, hkv, dh):
    """Values of +-1 by turns and nearly equal scores: outputs near 0 whose terms are not, so that a probability held in fp16 (off by
    up to 2^-11 of it) shows. The bound: the result's rounding; scores as in `bound`; 2^-19 for a page's log2 weight (one step of
    2^-20 at 14), its difference to the maximum and the exponential's argument (2^-21 each); exp2 and the two halves, 2^-21; fp32
    sums, 2^-24 of reach a key."""
    import torch
    rng = np.random.default_rng(dh)
    L, bs = [2, 3, 17, 40], 16
    pages = sum(-(-n // bs) for n in L)
    c = Cache(rng, pages, hkv, dh, bs, fmt, values=True)
    one = 64 if fmt == INT8 else 0x38                               # 64 x 2^-6, 1.0 x 2^0
    v = np.where(np.arange(bs) % 2, (-one & 255) if fmt == INT8 else one | 128, one).astype(np.uint8)
    host = list(c.before())
    host[1] = np.broadcast_to(v, host[1].shape).copy()
    host[2], host[3] = np.full_like(host[2], 2.0 ** -7), np.full_like(host[3], 2.0 ** -6 if fmt == INT8 else 1.0)
    c.dv.copy_(dev(host[1].reshape(pages, -1)))
    c.dks.copy_(dev(host[2])); c.dvs.copy_(dev(host[3]))             # noqa: E702
    q = (rng.standard_normal((4, H * dh)) * 0.02).astype(np.float16)
    table = _table(rng, L, bs, pages)
    Q, T, Ln = to_dev(q), dev(table), dev(np.array(L, np.int32))
    O = torch.zeros(4, H * dh, dtype=torch.float16, device="cuda")
    need = int(lib.sh_attention_kv_ws_bytes(C.byref(c.c), 4, 4, 1, H, table.shape[1]))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert lib.sh_attention_kv(A(Q), A(O), C.byref(c.c), A(T), table.shape[1], A(Ln), 0, 4, 4, 1, H, H * dh, H * dh, dh ** -0.5, 0, A(ws), need) == 0
    o, reach, spread = R.attention(q, *host, table, L, None, H, dh ** -0.5, fmt)
    d = (dh + 8) * 2.0 ** -23 * spread + 2.0 ** -19 + 2.0 ** -21
    err = np.abs(to_np(O) - o)
    assert (err <= 2.0 ** -11 * np.abs(o) + reach * (2 * d + max(L) * 2.0 ** -24) + 2.0 ** -24).all(), float((err / reach).max())


def _call(lib, c, q, table, kv_len, row_start, H, scale, window=0, max_q=1):
    import torch
    rows, D = q.shape
    Q, T, Ln = to_dev(q), dev(table), dev(np.asarray(kv_len, np.int32))
    Rs = dev(np.asarray(row_start, np.int32)) if row_start is not None else None
    O = torch.full((rows, D), 7.0, dtype=torch.float16, device="cuda")
    need = int(lib.sh_attention_kv_ws_bytes(C.byref(c.c), len(kv_len), rows, max_q, H, table.shape[1]))
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    rc = lib.sh_attention_kv(A(Q), A(O), C.byref(c.c), A(T), table.shape[1], A(Ln), A(Rs) if Rs is not None else 0, len(kv_len), rows, max_q, H, D, D,
                             scale, window, A(ws), need)
    assert rc == 0, shops.last_error()
    return to_np(O).astype(np.float64)


FEW_AND_MANY = [(4, 2, 64, [40, 0, 700], None), (2, 1, 128, [6000, 3, 90], None), (16, 1, 64, [5000, 100, 2], None),       # single tokens, whole and cut
                (4, 2, 80, [60, 300, 5], [40, 2, 9]), (4, 1, 64, [2500, 90, 31], [30, 90, 1])]                             # chunks, whole and cut


@pytest.mark.parametrize("fmt", [INT8, FP8])
@pytest.mark.parametrize("H,hkv,dh,L,new", FEW_AND_MANY)
def test_attention_rows_with_infinities(lib, gpu, fmt, H, hkv, dh, L, new):
    """An infinity or NaN in a head's row of q makes that head's output NaN wherever it sees a key, also where all of its scores are -inf
    (every code of that channel has one sign); heads that see none give zeros, and the others their own values."""
    rng = np.random.default_rng(dh + len(L))
    bs = 16
    pages = sum(-(-n // bs) for n in L) + 1
    c = Cache(rng, pages, hkv, dh, bs, fmt, values=True)
    host = list(c.before())
    host[0][..., 0] = 0x30                                          # positive in both formats
    c.dk.copy_(dev(host[0].reshape(pages, -1)))
    start = None if new is None else np.concatenate([[0], np.cumsum(new)])
    rows = 3 if new is None else sum(new)
    q = rng.standard_normal((rows, H, dh)).astype(np.float16)
    clean = q.copy()
    bad = np.zeros((rows, H), bool)
    for i, x in enumerate((-np.inf, np.inf, np.nan, -np.inf)):
        r, h = (i * 7) % rows, i % H
        q[r, h, 0 if i != 3 else dh - 1] = x
        bad[r, h] = True
    table = _table(rng, L, bs, pages)
    o = _call(lib, c, q.reshape(rows, -1), table, L, start, H, dh ** -0.5, max_q=1 if new is None else max(new)).reshape(rows, H, dh)
    want, reach, spread = (x.reshape(rows, H, dh) for x in R.attention(clean.reshape(rows, -1), *host, table, L, start, H, dh ** -0.5, fmt))
    sees = reach.any(2) > 0
    assert np.isnan(o[bad & sees]).all() and (o[bad & ~sees] == 0).all() and (bad & sees).any()
    tol = bound(want, reach, spread, dh, max(L), (127 if fmt == INT8 else 448) * host[3].max())
    assert (np.abs(o - want) <= tol)[~bad].all()


@pytest.mark.parametrize("fmt", [INT8, FP8])
@pytest.mark.parametrize("top", [3e6, -3e6, 1e9, -1e9, -4e30, 1e36, -1e36])
@pytest.mark.parametrize("H,hkv,dh,L,new", FEW_AND_MANY)
def test_attention_scores_of_any_size(lib, gpu, fmt, top, H, hkv, dh, L, new):
    """Scores of one channel, -1/16 to 1 times or 1 to 16 times `top`, far enough apart that the largest alone counts; where several keys share it
    (in pages of other value scales, too) their values are averaged. Bound: result and probability to fp16, 2^-11 each, log2 of a weight
    (2^-19), sums (2^-24 a key)."""
    rng = np.random.default_rng(dh + len(L))
    bs = 16
    pages = sum(-(-n // bs) for n in L) + 1
    c = Cache(rng, pages, hkv, dh, bs, fmt, values=True)
    host = list(c.before())
    codes = np.array([8, 32, 64, 127]) if fmt == INT8 else np.array([0x20, 0x38, 0x40, 0x48])        # 8 .. 127; 1/8, 1, 2, 4
    if top < 0:
        codes = (-codes) & 255 if fmt == INT8 else codes | 128
    host[0][..., 0] = codes[rng.integers(0, 4, host[0].shape[:3])]
    host[2] = np.full_like(host[2], abs(top) / (127 if fmt == INT8 else 4))
    c.dk.copy_(dev(host[0].reshape(pages, -1)))
    c.dks.copy_(dev(host[2]))
    start = None if new is None else np.concatenate([[0], np.cumsum(new)])
    rows = 3 if new is None else sum(new)
    q = np.zeros((rows, H, dh), np.float16)
    q[..., 0] = 1
    table = _table(rng, L, bs, pages)
    o = _call(lib, c, q.reshape(rows, -1), table, L, start, H, 1.0, max_q=1 if new is None else max(new))
    want, reach, _ = R.attention(q.reshape(rows, -1), *host, table, L, start, H, 1.0, fmt)
    err = np.abs(o - want)
    assert (err <= 2.0 ** -11 * np.abs(want) + reach * (2.0 ** -11 + 2.0 ** -19 + max(L) * 2.0 ** -24) + 2.0 ** -24).all(), float(err.max())


@pytest.mark.parametrize("B,dh", [(65, 64), (300, 32), (512, 128), (700, 32), (256, 256), (257, 256), (600, 80)])
@pytest.mark.parametrize("longest", [500, 5000])
def test_attention_many_requests(lib, gpu, B, dh, longest):
    """More requests than a wave has lanes, or a workgroup threads, most without keys or rows; items that are cut and that are not."""
    rng = np.random.default_rng(B)
    bs = 16
    L = np.where(rng.random(B) < 0.7, 0, rng.integers(1, 60, B))
    L[B // 3], L[B - 1] = longest, 90
    new = np.where(rng.random(B) < 0.5, 0, rng.integers(1, 4, B))
    new[B // 3] = new[B - 1] = 2
    start = np.concatenate([[0], np.cumsum(new)])
    pages = int(sum(-(-n // bs) for n in L)) + 1
    c = Cache(rng, pages, 1, dh, bs, INT8)
    q = rng.standard_normal((int(start[-1]), 2 * dh)).astype(np.float16)
    _attend(lib, c, q, _table(rng, L.tolist(), bs, pages), L.tolist(), start, 2, 0.2)


@pytest.mark.parametrize("B", [65, 200])
def test_attention_many_chunks(lib, gpu, B):
    """Chunks of more requests than a wave has lanes, one of them long enough to be cut."""
    rng = np.random.default_rng(B)
    bs, dh = 16, 32
    new = np.where(rng.random(B) < 0.3, 0, rng.integers(1, 12, B))
    new[3], new[B - 1] = 40, 50
    L = new + np.where(rng.random(B) < 0.5, 0, rng.integers(0, 200, B))
    L[B - 1] = 4000
    start = np.concatenate([[0], np.cumsum(new)])
    pages = int(sum(-(-n // bs) for n in L)) + 1
    c = Cache(rng, pages, 1, dh, bs, FP8, values=True)
    q = rng.standard_normal((int(start[-1]), 2 * dh)).astype(np.float16)
    _attend(lib, c, q, _table(rng, L.tolist(), bs, pages), L.tolist(), start, 2, 0.2)


def test_attention_row_ranges_that_decrease(lib, gpu):
    """150 requests over the same 512 rows (row_start 0, 512, 0, 512, ...): more units than a call of 512 rows has, one of them a request
    that is cut and of whose parts only some exist. What is written is some request's result, and nothing else is written."""
    import torch
    rng = np.random.default_rng(41)
    R_, H, hkv, dh, bs, B, long = 512, 4, 2, 32, 16, 300, 2 * 83
    c = Cache(rng, 200, hkv, dh, bs, INT8)
    kv_len = np.full(B, 64, np.int32)
    kv_len[long] = 3000
    table = np.tile(np.arange(188, dtype=np.int32), (B, 1))
    start = np.where(np.arange(B + 1) % 2, R_, 0).astype(np.int32)
    q = rng.standard_normal((R_, H * dh)).astype(np.float16)
    need = int(lib.sh_attention_kv_ws_bytes(C.byref(c.c), B, R_, R_, H, 188))
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    O = torch.full((R_ + 64, H * dh), 7.0, dtype=torch.float16, device="cuda")
    Q, T, Ln, Rs = to_dev(q), dev(table), dev(kv_len), dev(start)
    for _ in range(3):
        rc = lib.sh_attention_kv(A(Q), A(O, 32 * H * dh), C.byref(c.c), A(T), 188, A(Ln), A(Rs), B, R_, R_, H, H * dh, H * dh, 0.2, 0, A(ws), need)
        assert rc == 0, shops.last_error()
    o = to_np(O).astype(np.float64)
    assert (o[:32] == 7.0).all() and (o[-32:] == 7.0).all() and (to_np(ws)[need:] == 255).all()
    o = o[32:-32].reshape(R_, H, dh)
    ok = np.zeros((R_, H), bool)
    for n in (64, 3000):
        want, reach, spread = (x.reshape(R_, H, dh) for x in R.attention(q, *c.before(), table[:1], [n], np.array([0, R_]), H, 0.2, INT8))
        ok |= (np.abs(o - want) <= bound(want, reach, spread, dh, n, 127 * c.sc.max())).all(2)
    assert ok.all()


@pytest.mark.parametrize("fmt", [INT8, FP8])
def test_pages_shared_in_a_table_of_the_callers(lib, gpu, fmt):
    """Three requests over the same two pages of a prefix, each with pages of its own behind: new tokens go into those, the shared pages keep
    their bytes, and attention gives the bits of a table with a copy of the prefix for each."""
    rng = np.random.default_rng(43)
    H, hkv, dh, bs = 6, 2, 64, 16
    c = Cache(rng, 14, hkv, dh, bs, fmt, values=True)
    table = np.array([[3, 9, 0, 1], [3, 9, 2, 4], [3, 9, 5, 0]], np.int32)
    held, new = [40, 48, 32], [3, 9, 1]
    slot = np.array([table[b, p // bs] * bs + p % bs for b in range(3) for p in range(held[b], held[b] + new[b])], np.int32)
    x = rng.standard_normal((2, len(slot), hkv * dh)).astype(np.float16)
    X, S = to_dev(x), dev(slot)
    assert lib.sh_kv_append(C.byref(c.c), A(X), A(X, x[0].size), hkv * dh, hkv * dh, A(S), len(slot)) == 0
    now = c.now()
    for g, w, old in zip(now, R.append(*c.before(), x[0], x[1], slot, fmt), c.before()):
        assert np.array_equal(*(np.where(t == 128, 0, t) if t.dtype == np.uint8 else t for t in (g, w)))
        assert np.array_equal(g[[3, 9]], old[[3, 9]])
    q = rng.standard_normal((len(slot), H * dh)).astype(np.float16)
    start, L = np.concatenate([[0], np.cumsum(new)]), [h + n for h, n in zip(held, new)]
    one = _call(lib, c, q, table, L, start, H, 0.125, max_q=max(new))
    apart = table.copy()
    for b, (i, j) in ((1, (10, 11)), (2, (12, 13))):
        apart[b, :2] = i, j
        for t in (c.dk, c.dv, c.dks, c.dvs):
            t[[i, j]] = t[[3, 9]]
    assert np.array_equal(one, _call(lib, c, q, apart, L, start, H, 0.125, max_q=max(new)))
    want, reach, spread = R.attention(q, *now, table, L, start, H, 0.125, fmt)
    assert (np.abs(one - want) <= bound(want, reach, spread, dh, max(L), 448 * now[3].max())).all()


WINDOWS = [   # H, hkv, dh, bs, lengths, new rows, window
    (4, 2, 128, 16, [6500, 3000, 40, 2600], None, 2500),            # single tokens, cut between workgroups: 40 key tiles each
    (8, 1, 64, 64, [9000, 2501, 2499], None, 2500),
    (16, 1, 64, 16, [7000, 64], None, 4000),                        # sixteen rows a tile
    (2, 1, 80, 32, [6100, 5000], [4, 3], 2500),                     # drafts
    (4, 1, 256, 16, [6000], [3], 2600),
    (4, 1, 48, 16, [6500, 2600], [1, 4], 2500),
    (8, 2, 64, 16, [6000, 700, 3000], [40, 20, 1], 2500),           # chunks whose keys are cut into parts
    (4, 1, 128, 32, [5000, 300], [90, 300], 1000),
    (2, 1, 32, 16, [3000], [700], 600),                             # row tiles that see few of the request's key tiles: empty parts
    (4, 1, 256, 16, [2800], [50], 2000),
]


@pytest.mark.parametrize("fmt", [INT8, FP8])
@pytest.mark.parametrize("H,hkv,dh,bs,L,new,window", WINDOWS)
def test_attention_window_over_long_contexts(lib, gpu, fmt, H, hkv, dh, bs, L, new, window):
    """A first key tile behind 0 with keys that are shared between workgroups and joined. Pages before every window hold NaN codes and
    scales."""
    rng = np.random.default_rng(window + sum(L))
    pages = sum(-(-n // bs) for n in L) + 3
    c = Cache(rng, pages, hkv, dh, bs, fmt, values=True)
    table = _table(rng, L, bs, pages)
    host = c.before()
    clean = [h.copy() for h in host]
    for b, n in enumerate(L):
        for pg in table[b, : max(0, n - (new[b] if new else 1) + 1 - window) // bs]:
            host[0][pg], host[1][pg], host[2][pg], host[3][pg] = 0x7F, 0xFF, np.nan, np.nan
            clean[2][pg], clean[3][pg] = 0, 0
    c.dk.copy_(dev(host[0].reshape(pages, -1))); c.dv.copy_(dev(host[1].reshape(pages, -1)))   # noqa: E702
    c.dks.copy_(dev(host[2])); c.dvs.copy_(dev(host[3]))                                       # noqa: E702
    start = None if new is None else np.concatenate([[0], np.cumsum(new)])
    q = rng.standard_normal((len(L) if new is None else sum(new), H * dh)).astype(np.float16)
    _attend(lib, c, q, table, L, start, H, dh ** -0.5, window=window, host=clean)


@pytest.mark.parametrize("B", [65, 300, 600, 1500])
@pytest.mark.parametrize("window,longest,rows", [(100, 900, 3), (2500, 6000, 3), (1000, 4000, 90)])
def test_attention_window_of_many_requests(lib, gpu, B, window, longest, rows):
    """More requests than a wave has lanes or a workgroup threads, runs of idle ones between them, under a window; single tokens, drafts and
    (90 rows) chunks."""
    rng = np.random.default_rng(B + window)
    bs, dh = 16, 32
    new = np.where(rng.random(B) < 0.6, 0, rng.integers(1, 4, B))
    new[B // 4:B // 2] = 0
    new[B // 3], new[B - 1] = rows, 2
    L = np.where(rng.random(B) < 0.5, 0, rng.integers(1, 60, B))
    L[B // 3], L[B - 1], L[7] = longest, longest // 2, window + 1
    start = np.concatenate([[0], np.cumsum(new)])
    pages = int(sum(-(-n // bs) for n in L)) + 1
    c = Cache(rng, pages, 1, dh, bs, FP8, values=True)
    q = rng.standard_normal((int(start[-1]), 2 * dh)).astype(np.float16)
    _attend(lib, c, q, _table(rng, L.tolist(), bs, pages), L.tolist(), start, 2, 0.2, window=window)


@pytest.mark.parametrize("B,active", [(65536, [0, 1, 63, 64, 20000, 20128, 65535]), (513, [512]), (2000, [700]), (4096, list(range(0, 4096, 129)))])
def test_attention_slots_mostly_idle(lib, gpu, B, active):
    """A batch of fixed slots of which few have a request; the others add no row (and some hold keys all the same)."""
    rng = np.random.default_rng(B)
    bs, ld, dh = 16, 64, 64
    L, new = np.zeros(B, np.int32), np.zeros(B, np.int64)
    L[::97] = 100
    L[active], new[active] = rng.integers(1, ld * bs + 1, len(active)), rng.integers(1, 4, len(active))
    c = Cache(rng, 200, 1, dh, bs, INT8)
    table = rng.integers(0, 200, (B, ld)).astype(np.int32)
    start = np.concatenate([[0], np.cumsum(new)])
    q = rng.standard_normal((int(start[-1]), 2 * dh)).astype(np.float16)
    o = _call(lib, c, q, table, L, start, 2, 0.125, max_q=3)
    some = np.array(active)
    want, reach, spread = R.attention(q, *c.before(), table[some], L[some], np.concatenate([start[some], start[-1:]]), 2, 0.125, INT8)
    assert (np.abs(o - want) <= bound(want, reach, spread, dh, ld * bs, 127 * c.sc.max())).all()


@pytest.mark.parametrize("window", [0, 200])
def test_tokens_and_chunks_of_a_step_in_two_calls(lib, gpu, window):
    """The requests of a step in two calls over the same rows: single tokens first, then the chunks, whose row_start begins behind them."""
    import torch
    rng = np.random.default_rng(47)
    H, hkv, dh, bs, nd = 8, 2, 64, 16, 5
    L, new = [300, 1, 77, 900, 16, 150, 400, 90], [1, 1, 1, 1, 1, 150, 33, 1]
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    rows, D = int(start[-1]), H * dh
    pages = sum(-(-n // bs) for n in L) + 1
    c = Cache(rng, pages, hkv, dh, bs, FP8, values=True)
    table = _table(rng, L, bs, pages)
    ld, B = table.shape[1], len(L)
    q = rng.standard_normal((rows, D)).astype(np.float16)
    Q, T, Ln, Rs = to_dev(q), dev(table), dev(np.array(L, np.int32)), dev(start)
    O = torch.full((rows, D), 7.0, dtype=torch.float16, device="cuda")
    need = int(lib.sh_attention_kv_ws_bytes(C.byref(c.c), B, rows, max(new), H, ld))
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    for first, n, max_q in ((0, nd, 1), (nd, B - nd, max(new))):
        rc = lib.sh_attention_kv(A(Q), A(O), C.byref(c.c), A(T, first * ld), ld, A(Ln, first), A(Rs, first), n, rows, max_q, H, D, D, 0.125, window, A(ws), need)
        assert rc == 0, shops.last_error()
        if first == 0:
            assert (to_np(O)[nd:] == 7.0).all()
    want, reach, spread = R.attention(q, *c.before(), table, L, start, H, 0.125, FP8, window)
    assert (np.abs(to_np(O) - want) <= bound(want, reach, spread, dh, max(L), 448 * c.sc.max())).all()


def test_attention_repeats_its_bits(lib, gpu):
    rng = np.random.default_rng(29)
    L = [5000, 40, 900]
    c = Cache(rng, 400, 2, 128, 16, FP8, values=True)
    t = _table(rng, L, 16, 400)
    q = rng.standard_normal((3, 8 * 128)).astype(np.float16)
    a = _attend(lib, c, q, t, L, None, 8, 0.09)
    assert np.array_equal(a, _attend(lib, c, q, t, L, None, 8, 0.09))


def test_cache_beyond_4_gib(lib, gpu):
    """Pages whose byte offsets pass 2^32: written and read back at both ends of a 5 GiB cache."""
    import torch
    bs, hkv, dh = 64, 8, 128
    pg = hkv * bs * dh
    pages = (5 << 30) // pg
    k, v = (torch.zeros(pages * pg, dtype=torch.uint8, device="cuda") for _ in "kv")
    ks, vs = (torch.ones(pages, hkv, device="cuda") for _ in "kv")
    cc = shops.kv_cache(A(k), A(v), A(ks), A(vs), pages, hkv, dh, bs, INT8)
    rng = np.random.default_rng(31)
    ends = np.array([pages - 1, 0, pages - 2, pages // 2 + 7])
    L = 4 * bs - 3
    slot = np.array([int(ends[p // bs]) * bs + p % bs for p in range(L)], np.int32)
    x = rng.standard_normal((2, L, hkv * dh)).astype(np.float16)
    X, S = to_dev(x), dev(slot)
    assert lib.sh_kv_append(C.byref(cc), A(X), A(X, L * hkv * dh), hkv * dh, hkv * dh, A(S), L) == 0
    take = torch.from_numpy(ends).cuda()
    small = [t.view(pages, -1)[take].cpu().numpy() for t in (k, v, ks, vs)]
    small = [small[0].reshape(4, hkv, bs, dh), small[1].reshape(4, hkv, dh, bs), small[2], small[3]]
    zero = [np.zeros_like(s) for s in small[:2]] + [np.ones_like(s) for s in small[2:]]
    want = R.append(*zero, x[0], x[1], np.arange(L), INT8)
    for g, w in zip(small, want):
        assert np.array_equal(g, w)
    q = rng.standard_normal((1, 16 * dh)).astype(np.float16)
    Q, O = to_dev(q), torch.zeros(1, 16 * dh, dtype=torch.float16, device="cuda")
    T, Ln = dev(ends.astype(np.int32)[None]), dev(np.array([L], np.int32))
    need = lib.sh_attention_kv_ws_bytes(C.byref(cc), 1, 1, 1, 16, 4)
    ws = torch.empty(int(need), dtype=torch.uint8, device="cuda")
    assert lib.sh_attention_kv(A(Q), A(O), C.byref(cc), A(T), 4, A(Ln), 0, 1, 1, 1, 16, 16 * dh, 16 * dh, 0.09, 0, A(ws), need) == 0
    o, reach, spread = R.attention(q, *small, np.arange(4)[None], [L], None, 16, 0.09, INT8)
    assert (np.abs(to_np(O) - o) <= bound(o, reach, spread, dh, L, 127 * small[3].max())).all()
    del k, v
    torch.cuda.empty_cache()
