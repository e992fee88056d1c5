"""sh_mx4_quant, sh_gemm_mx4 and sh_gemm_mx4_f16 on the GPU against 64 bits (oracle/rope_mx4_refs.py)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from conftest import _KEEP, codes, to_dev, to_np
from oracle import rope_mx4_refs as R
from softhier_mlir_amd import shops

pytestmark = pytest.mark.gpu
A = shops.addr


def dev(a):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    _KEEP.append(t)
    return t


def up(n, m):
    return -(-n // m) * m


def _quant(lib, x, pad=0, off=0, cpad=0, spad=0):
    import torch
    rows, cols = x.shape
    nb = -(-cols // 32)
    xp = np.full(off + rows * (cols + pad), np.nan, np.float16)
    xp[off:].reshape(rows, cols + pad)[:, :cols] = x
    X = to_dev(xp)
    ldc, lds = 16 * nb + 16 * cpad, up(nb, 4) + 4 * spad
    c, s = (torch.full((rows, n), 0xA5, dtype=torch.uint8, device="cuda") for n in (ldc, lds))
    assert lib.sh_mx4_quant(A(c), A(s), A(X, off), rows, cols, ldc, lds, cols + pad) == 0, shops.last_error()
    c, s = to_np(c), to_np(s)
    assert (c[:, 16 * nb:] == 0xA5).all() and (s[:, nb:] == 0xA5).all()
    return R.unpack(c[:, : 16 * nb]), s[:, :nb]


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 8), (2, 31), (1, 32), (5, 33), (64, 720), (50, 4096), (7, 1001), (300, 65), (2, 14336)])
@pytest.mark.parametrize("pad,off", [(0, 0), (1, 1), (8, 3)])
def test_quant(lib, gpu, rows, cols, pad, off):
    rng = np.random.default_rng(rows + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 8, (rows, 1)))).astype(np.float16)
    c, s = _quant(lib, x, pad, off, cpad=pad, spad=off)
    wc, ws = R.quant(x)
    assert np.array_equal(s, ws) and np.array_equal(c, wc)


def test_quant_every_half(lib, gpu):
    """Every finite half beside each of several largest values of its block: the code and the scale, ties and subnormals among them."""
    h = np.arange(65536, dtype=np.uint16).view(np.float16)
    h = h[np.isfinite(h)]
    for top in (0.0, 6e-8, 1e-5, 0.375, 1.0, 5.9, 6.0, 6.004, 7.0, 11.99, 12.0, 4000.0, 65504.0):
        v = h[np.abs(h) <= np.float16(top)] if top else h[h == 0]
        v = np.concatenate([v, np.zeros(-len(v) % 31, np.float16)]).reshape(-1, 31)
        x = np.concatenate([np.full((len(v), 1), top, np.float16), v], 1)
        x[::2] = x[::2, ::-1]
        c, s = _quant(lib, x)
        e = -32
        while float(np.float16(top)) > 6 * 2.0 ** e:
            e += 1
        assert (s == e + 127).all(), top
        assert np.array_equal(c, R.code(x.astype(np.float64) / 2.0 ** e)), top


def test_quant_specials(lib, gpu):
    """A NaN or an infinity makes its block's scale NaN and its codes 0, and no other block's."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 100)).astype(np.float16)
    x[0, 5], x[1, 40], x[2, 99], x[3, 32], x[3, 64] = np.nan, np.inf, -np.inf, np.nan, np.nan
    x[4] = 0
    x[5, :32] = -0.0
    c, s = _quant(lib, x)
    wc, ws = R.quant(x)
    assert np.array_equal(s, ws) and np.array_equal(c, wc)
    assert np.argwhere(s == 255).tolist() == [[0, 0], [1, 1], [2, 3], [3, 1], [3, 2]]


def _operand(rng, rows, K, lo=-3, hi=2):
    nb = -(-K // 32)
    c = rng.integers(0, 16, (rows, 32 * nb)).astype(np.uint8)
    c[:, K:] = 0
    return c, rng.integers(127 + lo, 127 + hi, (rows, nb)).astype(np.uint8)


def _put(c, s, cpad=0, spad=0):
    """Codes and scales on the GPU, leading dims wider than they need be; the bytes behind are not to be used."""
    nb = s.shape[1]
    cp, sp = np.full((len(c), 16 * nb + 16 * cpad), 0x77, np.uint8), np.full((len(s), up(nb, 4) + 4 * spad), 255, np.uint8)
    cp[:, : 16 * nb], sp[:, :nb] = R.pack(c), s
    return dev(cp), dev(sp)


def _epi(N, bias, bias32, act, residual):
    if bias is None and not act and residual is None:
        return None
    Bi = 0 if bias is None else A(dev(bias.astype(np.float32))) if bias32 else A(to_dev(bias))
    Re = 0 if residual is None else A(to_dev(residual))
    return C.byref(shops.epi(bias=Bi, bias_fmt=int(bias32), act=act, residual=Re, ldr=N if residual is not None else 0))


def _run(lib, x, w, M, N, K, bias=None, bias32=False, act=0, residual=None, cpad=0, spad=0, zpad=0, zoff=0, f16=None):
    import torch
    (wc, ws) = _put(*w, cpad, spad)
    Z = torch.full((zoff + M * (N + zpad),), 9.0, dtype=torch.float16, device="cuda")
    e = _epi(N, bias, bias32, act, residual)
    if f16 is not None:
        rc = lib.sh_gemm_mx4_f16(A(f16[0], f16[2]), A(wc), A(ws), A(Z, zoff), M, N, K, f16[1], wc.shape[1], ws.shape[1], N + zpad, e)
    else:
        xc, xs = _put(*x, cpad, spad)
        rc = lib.sh_gemm_mx4(A(xc), A(xs), A(wc), A(ws), A(Z, zoff), M, N, K, xc.shape[1], xs.shape[1], wc.shape[1], ws.shape[1], N + zpad, e)
    assert rc == 0, shops.last_error()
    z = to_np(Z)
    assert (z[:zoff] == 9.0).all()
    z = z[zoff:].reshape(M, N + zpad)
    assert (z[:, N:] == 9.0).all()
    return z[:, :N].astype(np.float64)


def _check(got, x, w, bias=None, gelu=False, residual=None):
    """Rounding to fp16 (half a step, 2^-11, twice with a residual). Sums of exact products in fp32: within an instruction up to 128 terms, then a chain of
    an instruction's sums (K / 64 at most), up to 16 waves' and eight more operations, each at most 2^-23 of sum |x w| (the matrix pipe may cut
    instead of rounding); GELU's slope is below 1.13, and its hardware exp2 and reciprocal add 2^-20 of the result."""
    xv, wv = R.value(*x), R.value(*w)
    z, s = R.gemm(xv, wv, bias, gelu)
    d = (128 + xv.shape[1] / 64 + 16 + 8) * 2.0 ** -23 * (s + (0 if bias is None else np.abs(bias.astype(np.float64))))
    tol = 2.0 ** -11 * np.abs(z) + (1.13 if gelu else 1.0) * d + 2.0 ** -25 + (2.0 ** -19 * np.abs(z) + 2.0 ** -22 if gelu else 0)
    if residual is not None:
        z = z + residual.astype(np.float64)
        tol = tol * (1 + 2.0 ** -11) + 2.0 ** -11 * np.abs(z) + 2.0 ** -25
    err = np.abs(got - z)
    assert (err <= tol).all(), (float((err - tol).max()), np.argwhere(~(err <= tol))[:4].tolist())


SHAPES = [(1, 1, 1), (1, 16, 32), (1, 17, 33), (1, 64, 128), (1, 2048, 720), (1, 100, 4096), (2, 33, 200), (5, 68, 1032), (16, 256, 512), (17, 132, 968), (31, 960, 960),
          (33, 40, 136), (50, 720, 2048), (64, 260, 1608), (65, 48, 320), (200, 72, 264), (3, 5000, 64), (64, 64, 16384), (128, 128, 256), (129, 127, 255), (256, 256, 512),
          (257, 300, 700), (300, 1000, 1000), (511, 513, 96), (700, 640, 2880), (1000, 260, 4100), (70, 2100, 31), (2048, 512, 512), (4100, 4200, 200), (4097, 4096, 33), (2500, 8200, 1200),
          (20, 5000, 600), (32, 8300, 1100), (40, 5000, 300), (64, 4096, 4128), (1000, 2048, 300), (2048, 4096, 288), (700, 5000, 1000), (9, 9000, 520)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(lib, gpu, M, N, K):
    rng = np.random.default_rng(M + N + K)
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -4)
    _check(_run(lib, x, w, M, N, K), x, w)


@pytest.mark.parametrize("M,N,K", [(1, 132, 712), (20, 64, 256), (64, 97, 344), (300, 257, 515), (200, 1100, 2100)])
@pytest.mark.parametrize("pads", [dict(cpad=1, spad=1, zpad=1, zoff=1), dict(cpad=3, spad=2, zpad=8, zoff=3)], ids=str)
def test_strides(lib, gpu, M, N, K, pads):
    rng = np.random.default_rng(M)
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -4)
    _check(_run(lib, x, w, M, N, K, **pads), x, w)


@pytest.mark.parametrize("M,N,K", [(1, 960, 720), (50, 200, 512), (7, 33, 96), (300, 515, 320), (600, 1029, 800)])
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("bias32", [False, True])
def test_epilogue(lib, gpu, M, N, K, gelu, bias32):
    rng = np.random.default_rng(M)
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -5)
    b, r = rng.standard_normal(N).astype(np.float16), rng.standard_normal((M, N)).astype(np.float16)
    _check(_run(lib, x, w, M, N, K, b, bias32, int(gelu), r), x, w, b, gelu, r)
    _check(_run(lib, x, w, M, N, K, b, bias32, int(gelu)), x, w, b, gelu)
    _check(_run(lib, x, w, M, N, K, residual=r, zpad=1), x, w, residual=r)


@pytest.mark.parametrize("M,N,K", [(3, 80, 256), (40, 100, 1100), (260, 300, 520), (520, 1100, 600)])
def test_exact_on_small_sums(lib, gpu, M, N, K):
    """Codes of whole and half numbers with scales of 1, 2 and 4: every sum is exact, so are the results; every code meets every code."""
    rng = np.random.default_rng(1)
    x, w = _operand(rng, M, K, 0, 2), _operand(rng, N, K, -1, 1)
    for c in (x[0], w[0]):
        c[(np.abs(R.VALUES[c]) > 1.0) & (rng.random(c.shape) < 0.97)] = 0
    z = R.gemm(R.value(*x), R.value(*w))[0]
    keep = np.abs(z) <= 512
    assert keep.mean() > 0.8
    assert np.array_equal(_run(lib, x, w, M, N, K)[keep], z.astype(np.float16).astype(np.float64)[keep])


@pytest.mark.parametrize("M,N,K", [(2, 40, 700), (300, 330, 700)])
def test_scales_over_the_range(lib, gpu, M, N, K):
    """Scales far from 1 that meet again near it, the smallest and the largest byte among them, and zeros under any scale."""
    rng = np.random.default_rng(7)
    x, w = _operand(rng, M, K), _operand(rng, N, K)
    nb = x[1].shape[1]
    e = rng.integers(-100, 100, nb)
    e[:4] = (-120, 120, -127 + 4, 127 - 3)
    x[1][:] = np.clip(127 + e + rng.integers(-2, 2, (M, nb)), 0, 254)
    w[1][:] = np.clip(127 - e - rng.integers(6, 9, (N, nb)), 0, 254)
    x[0][:, 32 * 5: 32 * 6] = 0
    x[1][:, 5], w[1][:, 5] = 254, 100
    _check(_run(lib, x, w, M, N, K), x, w)


@pytest.mark.parametrize("M,N", [(5, 70), (300, 333)])
def test_nan_scales(lib, gpu, M, N):
    """A scale of 255 makes its row (of x) or column (of W) NaN, though its codes are 0, and nothing else."""
    rng = np.random.default_rng(9)
    x, w = _operand(rng, M, 300), _operand(rng, N, 300, -9, -5)
    x[1][3, 9], w[1][44, 0] = 255, 255
    x[0][3, 288:], w[0][44, :32] = 0, 0
    z = _run(lib, x, w, M, N, 300)
    bad = np.zeros((M, N), bool)
    bad[3], bad[:, 44] = True, True
    assert np.array_equal(np.isnan(z), bad)


@pytest.mark.parametrize("M,N,K", [(1, 64, 1), (1, 2048, 720), (1, 200, 4096), (2, 33, 5), (7, 100, 1000), (16, 300, 2080), (5, 40, 31), (16, 50, 9000), (3, 1024, 260), (1, 8300, 700), (13, 8193, 1100), (7, 5000, 600), (2, 17000, 300)])
@pytest.mark.parametrize("pad,off", [(0, 0), (1, 1), (8, 3)])
def test_f16_rows(lib, gpu, M, N, K, pad, off):
    """The bits of sh_mx4_quant and sh_gemm_mx4, and the product within its bound."""
    rng = np.random.default_rng(M + K)
    h = (rng.standard_normal((M, K)) * np.exp2(rng.integers(-3, 3, (M, 1)))).astype(np.float16)
    w = _operand(rng, N, K, -9, -4)
    b, r = rng.standard_normal(N).astype(np.float16), rng.standard_normal((M, N)).astype(np.float16)
    xp = np.full(off + M * (K + pad), np.nan, np.float16)
    xp[off:].reshape(M, K + pad)[:, :K] = h
    X = to_dev(xp)
    x = R.quant(h)
    for kw in (dict(), dict(bias=b, act=1, residual=r)):
        got = _run(lib, None, w, M, N, K, f16=(X, K + pad, off), **kw)
        _check(got, x, w, kw.get("bias"), "act" in kw, kw.get("residual"))
        assert np.array_equal(got, _run(lib, x, w, M, N, K, **kw))


def test_f16_rows_specials(lib, gpu):
    """Rows with a NaN or an infinity are NaN, the others are as they are alone."""
    rng = np.random.default_rng(2)
    h, w = rng.standard_normal((6, 500)).astype(np.float16), _operand(rng, 90, 500, -9, -5)
    clean = _run(lib, None, w, 6, 90, 500, f16=(to_dev(h), 500, 0))
    h[1, 499], h[4, 0] = np.nan, np.inf
    z = _run(lib, None, w, 6, 90, 500, f16=(to_dev(h), 500, 0))
    assert np.isnan(z[[1, 4]]).all() and np.array_equal(np.delete(z, [1, 4], 0), np.delete(clean, [1, 4], 0))


def test_quantised_weight(lib, gpu):
    """A weight as the rows of W^T through sh_mx4_quant, activations likewise: the product of their values, on one stream and without waits between."""
    import torch
    rng = np.random.default_rng(5)
    M, N, K = 70, 200, 300
    x, wt = rng.standard_normal((M, K)).astype(np.float16), (rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float16)
    X, W = to_dev(x), to_dev(wt)
    bufs = []
    s, prev = torch.cuda.Stream(), lib.sh_get_stream()
    torch.cuda.synchronize()
    try:
        lib.sh_set_stream(s.cuda_stream)
        with torch.cuda.stream(s):
            for t, n in ((X, M), (W, N)):
                c, q = torch.empty((n, 160), dtype=torch.uint8, device="cuda"), torch.empty((n, 12), dtype=torch.uint8, device="cuda")
                assert lib.sh_mx4_quant(A(c), A(q), A(t), n, K, 160, 12, K) == 0
                bufs += [c, q]
            z = torch.zeros((M, N), dtype=torch.float16, device="cuda")
            assert lib.sh_gemm_mx4(*(A(t) for t in bufs), A(z), M, N, K, 160, 12, 160, 12, N, None) == 0
        s.synchronize()
    finally:
        lib.sh_set_stream(prev)
    _check(to_np(z).astype(np.float64), R.quant(x), R.quant(wt))


@pytest.mark.parametrize("M", [1, 40, 300, 1000])
def test_in_a_graph(lib, gpu, M):
    """Captured (rows to codes, then the product) and replayed on other rows: the eager bits of every replay."""
    import torch
    rng = np.random.default_rng(M)
    N, K = 520, 448
    w = _operand(rng, N, K, -9, -5)
    wc, ws = _put(*w)
    X = torch.zeros((M, K), dtype=torch.float16, device="cuda")
    out = [torch.zeros((M, N), dtype=torch.float16, device="cuda") for _ in "abc"]
    bufs = [(torch.zeros((M, 224), dtype=torch.uint8, device="cuda"), torch.zeros((M, 16), dtype=torch.uint8, device="cuda")) for _ in "ab"]

    def call(b, z):
        assert lib.sh_mx4_quant(A(b[0]), A(b[1]), A(X), M, K, 224, 16, K) == 0
        assert lib.sh_gemm_mx4(A(b[0]), A(b[1]), A(wc), A(ws), A(z), M, N, K, 224, 16, wc.shape[1], ws.shape[1], N, None) == 0, shops.last_error()
    torch.cuda.synchronize()
    s, g, prev = torch.cuda.Stream(), torch.cuda.CUDAGraph(), lib.sh_get_stream()
    with torch.cuda.graph(g, stream=s):
        lib.sh_set_stream(s.cuda_stream)
        call(bufs[0], out[0])
        if M <= 16:
            assert lib.sh_gemm_mx4_f16(A(X), A(wc), A(ws), A(out[2]), M, N, K, K, wc.shape[1], ws.shape[1], N, None) == 0
    lib.sh_set_stream(prev)
    for i in range(4):
        X.copy_(torch.from_numpy(rng.standard_normal((M, K)).astype(np.float16)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        call(bufs[1], out[1])
        assert np.array_equal(codes(out[0]), codes(out[1])), i
        if M <= 16:
            assert np.array_equal(codes(out[2]), codes(out[1])), i


def test_calls_give_the_same_bits_again(lib, gpu):
    rng = np.random.default_rng(8)
    for M, N, K in ((30, 500, 3000), (900, 700, 1500)):
        x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -4)
        first = _run(lib, x, w, M, N, K)
        for _ in range(3):
            assert np.array_equal(_run(lib, x, w, M, N, K), first)


@pytest.mark.parametrize("M,N", [(70, 90), (40, 200), (300, 40)])
def test_rows_far_apart(lib, gpu, M, N):
    """Leading dims so large that offsets pass 32 bits, of x, of W and of z."""
    import torch
    rng = np.random.default_rng(M)
    K, far = 700, (1 << 32) // 30 // 128 * 128
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -5)
    nb = x[1].shape[1]
    want = _run(lib, x, w, M, N, K)
    ops, lds = [], []
    for (c, s), n, big in ((x, M, M > 60), (w, N, N > 60)):
        ldc = far if big else 16 * nb
        buf = torch.zeros((n, ldc), dtype=torch.uint8, device="cuda")
        buf[:, : 16 * nb] = dev(R.pack(c))
        ops += [buf, _put(c, s)[1]]
        lds += [ldc, ops[-1].shape[1]]
    z = torch.zeros((M, far // 2), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    assert lib.sh_gemm_mx4(*(A(t) for t in ops), A(z), M, N, K, *lds, far // 2, None) == 0, shops.last_error()
    got = to_np(z[:, :N]).astype(np.float64)
    if M <= 64:                                              # (the same kernel: for more rows it is the one whose offsets hold)
        assert np.array_equal(got, want)
    _check(got, x, w)


def test_quant_rows_far_apart(lib, gpu):
    import torch
    rng = np.random.default_rng(6)
    rows, cols, far = 40, 300, (1 << 32) // 36 // 16 * 16
    x = rng.standard_normal((rows, cols)).astype(np.float16)
    X = torch.zeros((rows, far), dtype=torch.float16, device="cuda")
    X[:, :cols] = to_dev(x)
    c, s = torch.zeros((rows, far), dtype=torch.uint8, device="cuda"), torch.zeros((rows, 12), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert lib.sh_mx4_quant(A(c), A(s), A(X), rows, cols, far, 12, far) == 0, shops.last_error()
    wc, ws = R.quant(x)
    assert np.array_equal(to_np(s[:, :10]), ws) and np.array_equal(R.unpack(to_np(c[:, :160].contiguous())), wc)
