"""What sh_kv_slots, sh_kv_append, sh_attention_kv and sh_gemm_w4 refuse, without a GPU: every check comes before any GPU
work, with its code and message."""
from __future__ import annotations

import ctypes as C

import pytest

from softhier_mlir_amd import shops

ONE = 1 << 20                                   # never dereferenced: the checks fail first


def _cache(**kw):
    d = dict(k=ONE, v=ONE, ks=ONE, vs=ONE, pages=8, hkv=2, dh=64, bs=16, fmt=shops.SH_INT8)
    d.update(kw)
    return shops.kv_cache(**d)


BAD_CACHES = [dict(k=0), dict(v=0), dict(ks=0), dict(vs=0), dict(k=ONE + 8), dict(v=ONE + 4), dict(ks=ONE + 2), dict(bs=8), dict(bs=48),
              dict(bs=128), dict(dh=0), dict(dh=8), dict(dh=72), dict(dh=272), dict(hkv=0), dict(hkv=1025), dict(fmt=shops.SH_FP16), dict(fmt=9),
              dict(pages=0), dict(pages=1 << 27), dict(pgk=2 * 16 * 64 - 16), dict(pgv=2 * 16 * 64 + 8), dict(pgs=1)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_caches_refused(lib, bad):
    c = C.byref(_cache(**bad))
    assert lib.sh_kv_append(c, ONE, ONE, 128, 128, ONE, 4) == -1
    assert shops.last_error()[0] == -1
    assert lib.sh_attention_kv(ONE, ONE, c, ONE, 4, ONE, 0, 2, 2, 1, 4, 1 << 20, 1 << 20, 0.125, 0, ONE, 1 << 40) == -1
    assert "[sh_attention_kv]" in shops.last_error()[1]


def test_append_refusals(lib):
    c = C.byref(_cache())
    good = [c, ONE, ONE, 128, 128, ONE, 4]
    for i, v in ((0, None), (1, 0), (2, 0), (3, 127), (4, 100), (5, 0), (1, ONE + 1), (5, ONE + 2), (6, 1 << 31)):
        a = list(good)
        a[i] = v
        assert lib.sh_kv_append(*a) == -1, (i, v)
        assert shops.last_error()[0] == -1
    assert lib.sh_kv_append(c, 0, 0, 128, 128, 0, 0) == 0                   # no rows: nothing to do


def test_attention_refusals(lib):
    c = C.byref(_cache())
    need = lib.sh_attention_kv_ws_bytes(c, 2, 2, 1, 4, 4)
    assert need > 0
    good = [ONE, ONE, c, ONE, 4, ONE, 0, 2, 2, 1, 4, 256, 256, 0.125, 0, ONE, need]
    for i, v in ((0, 0), (1, 0), (2, None), (3, 0), (5, 0), (4, 0), (4, 1 << 27), (7, 65537), (8, 1 << 31), (10, 0), (10, 3), (11, 255), (12, 255),
                 (13, float("nan")), (13, float("inf")), (13, 0.0), (13, -0.125), (15, 0), (15, ONE + 8), (0, ONE + 1), (6, ONE + 2)):
        a = list(good)
        a[i] = v
        assert lib.sh_attention_kv(*a) == -1, (i, v)
        assert shops.last_error()[0] == -1
    a = list(good)
    a[16] = need - 1
    assert lib.sh_attention_kv(*a) == -2
    assert shops.last_error()[0] == -2
    for i in (7, 8, 9):                                                     # no request, row or row bound: nothing to do
        a = list(good)
        a[i] = 0
        assert lib.sh_attention_kv(*a) == 0


@pytest.mark.parametrize("B,rows,max_q,ld,window", [(1, 1 << 29, 1 << 29, 4, 0),       # chunk units: rows H / 128 = 2^24
                                                    (65536, 65536, 1, 1 << 20, 0),      # tiles: 2^16 requests x 2^18 x 2 heads or more
                                                    (65536, 65536, 1, 1 << 20, 64)])    # and a window leaves the bound as it is
def test_attention_sizes_refused(lib, B, rows, max_q, ld, window):
    c = C.byref(_cache())
    assert lib.sh_attention_kv(ONE, ONE, c, ONE, ld, ONE, ONE, B, rows, max_q, 4, 256, 256, 0.125, window, ONE, 1 << 62) == -1
    assert "of 4 heads" in shops.last_error()[1] or "and 4 heads" in shops.last_error()[1]


def test_attention_workspace_grows_with_the_rows_and_heads(lib):
    c = C.byref(_cache())
    n = [lib.sh_attention_kv_ws_bytes(c, 64, 64, q, h, 64) for q, h in ((1, 2), (1, 8), (4, 8), (100, 8))]
    assert n[0] < n[1] < n[2] <= n[3]
    assert lib.sh_attention_kv_ws_bytes(None, 1, 1, 1, 2, 1) == 0
    for rows in (1, 64, 5000):                                              # no bound on a request's rows: theirs
        assert lib.sh_attention_kv_ws_bytes(c, 64, rows, 0xFFFFFFFF, 8, 64) == lib.sh_attention_kv_ws_bytes(c, 64, rows, rows, 8, 64)


def test_slots_refusals(lib):
    good = [ONE, 4, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, 3, 16, 8, 5]
    bad = [(i, 0) for i in (0, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11)] + [(i, ONE + 2) for i in (0, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11)]
    bad += [(1, 0), (1, 1 << 30), (12, 0), (12, 65537), (13, 24), (13, 128), (14, 0), (14, 1 << 28), (15, 1 << 31)]
    for i, v in bad:
        a = list(good)
        a[i] = v
        assert lib.sh_kv_slots(*a) == -1, (i, v)
        assert shops.last_error()[0] == -1


def test_w4_refusals(lib):
    e = lambda **kw: C.byref(shops.epi(**kw))  # noqa: E731
    good = [ONE, ONE, ONE, 0, ONE, 2, 64, 128, 32, 128, 64, 64, 64, None]
    bad = [(0, 0), (1, 0), (2, 0), (4, 0), (7, 0), (7, 100), (8, 0), (8, 16), (8, 48), (9, 127), (10, 63), (11, 63), (12, 63), (0, ONE + 1),
           (1, ONE + 2), (2, ONE + 1), (4, ONE + 1), (5, (1 << 19) + 1), (13, e(act=2)), (13, e(bias=ONE, bias_fmt=2)), (13, e(bias=ONE + 1)),
           (13, e(bias=ONE + 2, bias_fmt=shops.SH_BIAS_FP32)), (13, e(residual=ONE, ldr=63)), (13, e(residual=ONE + 1, ldr=64)), (13, e(splits=2)),
           (13, e(ln_stats=ONE)), (13, e(ln_c=ONE)), (13, e(stats_out=ONE)), (13, e(ln_parts=4))]
    for i, v in bad:
        a = list(good)
        a[i] = v
        assert lib.sh_gemm_w4(*a) == -1, (i, v)
        assert shops.last_error()[0] == -1
    for i in (5, 6):                                                        # no rows or columns: nothing to do
        a = list(good)
        a[i] = 0
        assert lib.sh_gemm_w4(*a) == 0


def test_attention_scale_times_log2_e_is_finite(lib):
    c = C.byref(_cache())
    need = lib.sh_attention_kv_ws_bytes(c, 2, 2, 1, 4, 4)
    assert lib.sh_attention_kv(ONE, ONE, c, ONE, 4, ONE, 0, 2, 2, 1, 4, 256, 256, 3e38, 0, ONE, need) == -1
    assert "scale" in shops.last_error()[1]


def test_attention_workspace_of_chunks_follows_the_table(lib):
    """A call of chunks holds parts only where keys can be cut: 104 MB at most here, a few where the table is short; and the size for the
    largest call is enough for every smaller one."""
    c = C.byref(_cache(hkv=8, dh=128))
    n = [lib.sh_attention_kv_ws_bytes(c, 8, 4096, 2048, 32, ld) for ld in (1, 32, 33, 64, 1 << 20)]
    few = lib.sh_attention_kv_ws_bytes(c, 8, 4096, 4, 32, 1)
    assert n[0] == n[1] == few < n[2] <= n[3] <= n[4] == 1536 * (128 * 130 * 4 + 32) + 16
    assert lib.sh_attention_kv_ws_bytes(c, 1, 20, 20, 32, 64) < n[4] // 16
    steps = dict(B=(1, 2, 9, 300), rows=(1, 17, 64, 1000), max_q=(1, 2, 16, 17, 900), ld=(1, 40, 5000))
    at = lambda B, rows, max_q, ld: lib.sh_attention_kv_ws_bytes(c, B, rows, max_q, 32, ld)  # noqa: E731
    for name, v in steps.items():
        for lo, hi in zip(v, v[1:]):
            for B in steps["B"]:
                for rows in steps["rows"]:
                    for q in steps["max_q"]:
                        for ld in steps["ld"]:
                            a = dict(B=B, rows=rows, max_q=q, ld=ld)
                            assert at(**{**a, name: lo}) <= at(**{**a, name: hi}), (a, name, lo, hi)
