"""sh_rope_pos, sh_kv_append_rope, sh_mx4_quant and sh_gemm_mx4 at the ends of their offsets: the largest leading dims of the products' tiles, rows far apart in
the build for many columns, and more rows than one launch takes."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from conftest import _KEEP
from oracle import rope_mx4_refs as R
from softhier_mlir_amd import shops
from test_gpu_mx4_tiles import ROWS, T64, T256, _operand, _put, _value, tile
from test_gpu_rope import _check, _plan

pytestmark = pytest.mark.gpu
A = shops.addr


def _far(t, ld):
    """The rows of t with a leading dim of ld bytes, in the upper half of a buffer."""
    import torch
    buf = torch.empty(2 * len(t) * ld, dtype=torch.uint8, device="cuda")
    rows = buf[len(t) * ld:].view(len(t), ld)
    rows[:, : t.shape[1]] = t
    _KEEP.append(buf)
    return rows


@pytest.mark.parametrize("scales", [False, True])
@pytest.mark.parametrize("t,M,N,far", [(T256, 300, 30000, "x"), (T256, 30000, 300, "w"), (T64, 300, 515, "xw")])
def test_tiles_of_the_largest_leading_dims(lib, gpu, t, M, N, far, scales):
    """2^24 bytes from row to row, 255 rows of a tile: offsets up to 2^32 from its first row. The bits of the compact rows."""
    import torch
    assert tile(M, N) == t
    rng = np.random.default_rng(M)
    K = 1100
    ops = [*_put(*_operand(rng, M, K), True), *_put(*_operand(rng, N, K, -9, -4), True)]

    def run():
        z = torch.zeros((M, N), dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        assert lib.sh_gemm_mx4(*(A(o) for o in ops), A(z), M, N, K, *(o.stride(0) for o in ops), N, None) == 0, shops.last_error()
        return z
    want = run()
    for c in far:
        i = 2 * (c == "w") + scales
        ops[i] = _far(ops[i], 1 << 24)
    assert torch.equal(run(), want)
    assert bool((want != 0).any())


def test_many_rows_of_a_far_weight(lib, gpu):
    """A weight whose rows are more than 2^24 bytes apart takes the kernel for few rows however many there are, here in two launches. Exact sums."""
    import torch
    rng = np.random.default_rng(1)
    M, N, K = 65535 * 64 + 131, 9, 70
    assert tile(M, N, near=False) is ROWS
    x, w = _operand(rng, 1000, K, 0, 2), _operand(rng, N, K, -1, 1)
    (xc, xs), (wc, ws) = _put(*x, False), _put(*w, False)
    pick = torch.randint(0, 1000, (M,), device="cuda")
    xc, xs, wf = xc[pick], xs[pick], _far(wc, (1 << 24) + 16)
    res = torch.randint(-4, 5, (M, N), device="cuda").half()
    z = torch.zeros((M, N), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    assert lib.sh_gemm_mx4(A(xc), A(xs), A(wf), A(ws), A(z), M, N, K, xc.shape[1], xs.shape[1], (1 << 24) + 16, ws.shape[1], N,
                           C.byref(shops.epi(residual=A(res), ldr=N))) == 0, shops.last_error()
    want = ((_value(*x) @ _value(*w).T).half()[pick].float() + res.float()).half()          # (sums of multiples of 1/8 are exact in fp32)
    assert torch.equal(z, want)


def test_quantised_rows_past_a_launch(lib, gpu):
    import torch
    rows = (1 << 28) + 77                                        # a launch takes 2^28 rows of one block
    x = torch.randint(0, 1 << 16, (rows, 2), device="cuda", dtype=torch.int32).to(torch.int16).view(torch.float16)
    c, s = torch.full((rows, 16), 0xA5, dtype=torch.uint8, device="cuda"), torch.full((rows, 4), 0xA5, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert lib.sh_mx4_quant(A(c), A(s), A(x), rows, 2, 16, 4, 2) == 0, shops.last_error()
    assert bool((s[:, 1:] == 0xA5).all())
    for first in (0, (1 << 28) - 500, rows - 500):
        wc, ws = R.quant(x[first: first + 500].cpu().numpy())
        assert np.array_equal(R.unpack(c[first: first + 500].cpu().numpy()), wc) and np.array_equal(s[first: first + 500, :1].cpu().numpy(), ws)
    half = rows // 2                                             # and all of it against two calls
    c2, s2 = torch.full_like(c, 0xA5), torch.full_like(s, 0xA5)
    torch.cuda.synchronize()
    for r, n in ((0, half), (half, rows - half)):
        assert lib.sh_mx4_quant(A(c2, 16 * r), A(s2, 4 * r), A(x, 2 * r), n, 2, 16, 4, 2) == 0
    assert torch.equal(c, c2) and torch.equal(s, s2)


@pytest.mark.parametrize("in_place", [False, True])
def test_many_turned_columns_of_rows_far_apart(lib, gpu, in_place):
    """The build for many columns (2^22 halves and more) with offsets past 32 bits."""
    import torch
    rows, heads, dh, far = 600, 56, 128, (1 << 32) // 500
    assert rows * heads * dh >= 1 << 22 and rows * far > 1 << 32
    rng = np.random.default_rng(8)
    x = rng.standard_normal((rows, heads * dh)).astype(np.float16)
    step, pos = R.steps(R.frequencies(64, 1e4)), np.arange(rows, dtype=np.int32) * 100 - 50
    X = torch.empty((rows, far), dtype=torch.float16, device="cuda")
    Y = X if in_place else torch.empty((rows, far), dtype=torch.float16, device="cuda")
    Y[:, : heads * dh] = 9.0
    X[:, : heads * dh] = torch.from_numpy(x).cuda()
    P = torch.from_numpy(pos).cuda()
    torch.cuda.synchronize()
    assert lib.sh_rope_pos(A(Y), A(X), A(P), _plan(step, R.HALF), rows, heads, dh, far, far) == 0, shops.last_error()
    y = Y[:, : heads * dh].contiguous().cpu().numpy()
    _check(y, x, step, pos, heads, dh, R.HALF)
    assert (y[0] == (x[0] if in_place else 9.0)).all()


def test_turned_rows_past_a_launch(lib, gpu):
    """2^31 chunks and more are two launches: the bits of calls that are one."""
    import torch
    rows = (1 << 30) + 1001
    X = torch.randn((rows, 4), device="cuda", dtype=torch.float16)
    Y, Z = (torch.zeros((rows, 4), dtype=torch.float16, device="cuda") for _ in "yz")
    pos = torch.arange(rows, device="cuda", dtype=torch.int32) - 5
    plan = _plan(R.steps(R.frequencies(4, 1e4)), R.PAIRS)
    torch.cuda.synchronize()
    assert lib.sh_rope_pos(A(Y), A(X), A(pos), plan, rows, 1, 4, 4, 4) == 0, shops.last_error()
    half = rows // 2
    for r, n in ((0, half), (half, rows - half)):
        assert lib.sh_rope_pos(A(Z, 4 * r), A(X, 4 * r), A(pos, r), plan, n, 1, 4, 4, 4) == 0
    assert torch.equal(Y.view(torch.int32), Z.view(torch.int32))
    assert bool((Y[:5] == 0).all()) and bool((Y[-1001:].view(torch.int32) != 0).any())


@pytest.mark.parametrize("fmt", [shops.SH_INT8, shops.SH_FP8])
def test_appended_rows_past_a_launch(lib, gpu, fmt):
    """More rows than one launch appends, a page over the border between two: the bits of two calls that meet at another page."""
    import torch
    H = hkv = 1
    dh = bs = 16
    rows, border = (1 << 23) * 16 + 1000, (1 << 23) * 16        # 2^30 threads: two workgroups of 64 for 16 rows
    pages = rows // bs + 2
    X = torch.randn((rows, 16), device="cuda", dtype=torch.float16)
    first = 7                                                   # (the first page's offset, so that pages lie over the borders of the groups of rows)
    slots = torch.arange(first, first + rows, device="cuda", dtype=torch.int32)
    pos = torch.arange(rows, device="cuda", dtype=torch.int32)
    step = R.steps(R.frequencies(16, 1e4))
    plan = _plan(step, R.HALF)

    def run(cuts):
        k, v = (torch.zeros(pages * bs * dh, dtype=torch.uint8, device="cuda") for _ in "kv")
        ks, vs = (torch.zeros((pages, 1), device="cuda") for _ in "kv")
        q = torch.zeros((rows, 16), dtype=torch.float16, device="cuda")
        c = shops.kv_cache(A(k), A(v), A(ks), A(vs), pages, hkv, dh, bs, fmt)
        torch.cuda.synchronize()
        for a, b in zip(cuts, cuts[1:]):
            assert lib.sh_kv_append_rope(C.byref(c), plan, A(q, 16 * a), A(X, 16 * a), A(X, 16 * a), A(X, 16 * a), A(pos, a), A(slots, a), b - a, H, 16, 16, 16, 16) == 0, shops.last_error()
        torch.cuda.synchronize()
        return k, v, ks, vs, q
    cut = rows // 2 // 16 * 16 - first                          # (a page's first slot)
    assert (cut + first) % 16 == 0 and border > cut
    one, two = run([0, rows]), run([0, cut, rows])
    for a, b in zip(one[:4], two[:4]):
        assert torch.equal(a, b)
    assert torch.equal(one[4].view(torch.int16), two[4].view(torch.int16))
    pick = [0, 1, border - 1, border, border + 1, rows - 1]
    _check(one[4][pick].cpu().numpy(), X[pick].cpu().numpy(), step, pos[pick].cpu().numpy(), 1, 16, R.HALF)
