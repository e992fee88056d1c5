"""sh_gemm_mx4's tiles, each build of them: the five shapes, scales by 16 bytes and by words, one to sixteen slices of 128 k, ragged edges,
every part of the epilogue. Which tile a shape takes is worked out here from the table of the source, and every row of CASES says which
one it is for, so that a change of the rule that moves a shape elsewhere is seen without a GPU."""
from __future__ import annotations

import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest

from conftest import _KEEP, to_dev
from oracle import rope_mx4_refs as R
from softhier_mlir_amd import shops

A = shops.addr
SOURCE = Path(__file__).resolve().parents[1] / "softhier_mlir_amd" / "csrc" / "sh_mx4.hip"
ROWS = None                                                 # (the kernel for few rows)
T64, T64x128, T128, T128x256, T256 = (64, 64), (64, 128), (128, 128), (128, 256), (256, 256)


def tile(M: int, N: int, near: bool = True):
    """The tile of a product, or ROWS: the rule of sh_gemm_mx4 with the shapes' times that its source holds."""
    table = re.search(r"static const Shape shapes\[\] = \{(.*)\};", SOURCE.read_text()).group(1)
    shapes = [tuple(float(v) for v in t.split(",")) for t in re.findall(r"\{([^{}]*)\}", table)]
    assert len(shapes) == 5
    if M <= 64 and (M <= 32 or N <= 4096) or not near:
        return ROWS
    cost = [first + more * ((-(-M // int(bm)) * -(-N // int(bn)) - 1) // 256) for bm, bn, first, more in shapes]
    return tuple(int(v) for v in shapes[cost.index(min(cost))][:2])


# a small and a skinny shape of each tile, ragged in both directions
CASES = [(T64, 300, 515), (T64, 65, 1000), (T64x128, 600, 1900), (T64x128, 50, 17000), (T128, 1000, 2200), (T128, 300, 9001), (T128x256, 1300, 3300),
         (T128x256, 4000, 1100), (T256, 300, 30000), (T256, 30000, 300)]
ONE = [(T64, 300, 515), (T64x128, 600, 1900), (T128, 1000, 2200), (T128x256, 1300, 3300), (T256, 2201, 3901)]


def test_the_rule_in_the_source():
    """The words of the source that `tile` repeats."""
    text = SOURCE.read_text()
    for words in ("if (M <= 16) ok = launch_rows<1, false>", "else if (M <= 32) ok = launch_rows<2, false>", "else if ((M <= 64 && N <= 4096) || !near) ok = launch_rows<4, false>",
                  "const double c = shapes[i].first + shapes[i].more * (double)((tiles - 1) / 256);", "if (!i || c < least) { pick = i; least = c; }"):
        assert words in text, words


def test_cases_reach_their_tiles():
    for t, M, N in CASES + ONE:
        assert tile(M, N) == t, (t, M, N, tile(M, N))
    assert {t for t, _, _ in ONE} == {T64, T64x128, T128, T128x256, T256}


def _operand(rng, rows, K, lo=-3, hi=2):
    nb = -(-K // 32)
    c = rng.integers(0, 16, (rows, 32 * nb), dtype=np.uint8)
    c[:, K:] = 0
    return c, rng.integers(127 + lo, 127 + hi, (rows, nb), dtype=np.uint8)


def _dev(a):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    _KEEP.append(t)
    return t


def _put(c, s, wide: bool, cpad=0):
    """Codes, and scales in rows of whole 16 bytes (`wide`) or 4 bytes more; what lies behind the blocks is not to be used."""
    nb = s.shape[1]
    lds = -(-nb // 16) * 16 + (0 if wide else 4)
    cp, sp = np.full((len(c), 16 * nb + 16 * cpad), 0x77, np.uint8), np.full((len(s), lds), 255, np.uint8)
    cp[:, : 16 * nb], sp[:, :nb] = R.pack(c), s
    return _dev(cp), _dev(sp)


def _value(c, s):
    """The numbers that the codes stand for, in 64 bits on the GPU."""
    import torch
    v = torch.from_numpy(R.VALUES).cuda()[torch.from_numpy(c).cuda().int()]
    e = torch.exp2(torch.from_numpy(s).cuda().double() - 127)
    return v * torch.where(torch.from_numpy(s).cuda() == 255, float("nan"), e).repeat_interleave(32, 1)


def _run(lib, x, w, K, wide, bias=None, bias32=False, act=0, residual=None, cpad=0, zpad=0, zoff=0):
    import torch
    M, N = len(x[0]), len(w[0])
    (xc, xs), (wc, ws) = _put(*x, wide, cpad), _put(*w, wide, cpad)
    Z = torch.full((zoff + M * (N + zpad),), 9.0, dtype=torch.float16, device="cuda")
    e = None
    if bias is not None or act or residual is not None:
        b = 0 if bias is None else A(_dev(bias.astype(np.float32))) if bias32 else A(to_dev(bias))
        e = C.byref(shops.epi(bias=b, bias_fmt=int(bias32), act=act, residual=0 if residual is None else A(to_dev(residual)), ldr=N if residual is not None else 0))
    torch.cuda.synchronize()
    rc = lib.sh_gemm_mx4(A(xc), A(xs), A(wc), A(ws), A(Z, zoff), M, N, K, xc.shape[1], xs.shape[1], wc.shape[1], ws.shape[1], N + zpad, e)
    assert rc == 0, shops.last_error()
    assert bool((Z[:zoff] == 9.0).all())
    z = Z[zoff:].view(M, N + zpad)
    assert bool((z[:, N:] == 9.0).all())
    return z[:, :N].clone()


def _check(got, x, w, bias=None, gelu=False, residual=None):
    """Rounding to fp16 (half a step, 2^-11, twice with a residual). Sums of exact products in fp32: within an instruction up to 128 terms (few rows; 64
    in tiles), a chain of an instruction's sums (K / 64 at most), eight waves' (few rows) and eight more operations, each at most 2^-23 of sum |x w| (the matrix pipe may cut instead of rounding);
    GELU's slope is below 1.13, and its hardware exp2 and reciprocal add 2^-19 of the result and 2^-22."""
    import torch
    xv, wv = _value(*x), _value(*w)
    z, s = xv @ wv.T, xv.abs() @ wv.abs().T
    if bias is not None:
        b = torch.from_numpy(bias).cuda().double()
        z, s = z + b, s + b.abs()
    d = (128 + xv.shape[1] / 64 + 16) * 2.0 ** -23 * s
    if gelu:
        z = 0.5 * z * (1 + torch.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
        d = 1.13 * d + 2.0 ** -19 * z.abs() + 2.0 ** -22
    tol = 2.0 ** -11 * z.abs() + d + 2.0 ** -25
    if residual is not None:
        z = z + torch.from_numpy(residual).cuda().double()
        tol = tol * (1 + 2.0 ** -11) + 2.0 ** -11 * z.abs() + 2.0 ** -25
    bad = ~((got.double() - z).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


SLICES = [33, 250, 330, 500, 640, 700, 800, 1000, 1100, 1400, 1536, 2040]              # 1 to 9, 11, 12 and 16 slices of 128 k


@pytest.mark.gpu
@pytest.mark.parametrize("t,M,N,K", [(*c, K) for c in ONE for K in SLICES] + [(*c, K) for c in CASES if c not in ONE for K in (250, 700, 1400)], ids=str)
def test_slices(lib, gpu, t, M, N, K):
    """Within the bound, with scales by 16 bytes; by words the same bits."""
    import torch
    assert tile(M, N) == t
    rng = np.random.default_rng(M + N + K)
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -4)
    got = _run(lib, x, w, K, True)
    _check(got, x, w)
    assert torch.equal(_run(lib, x, w, K, False), got)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [200, 1200])
@pytest.mark.parametrize("bias32", [False, True])
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("t,M,N", ONE, ids=str)
def test_epilogue(lib, gpu, t, M, N, gelu, bias32, K):
    rng = np.random.default_rng(M)
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -5)
    b, r = rng.standard_normal(N).astype(np.float16), rng.standard_normal((M, N)).astype(np.float16)
    _check(_run(lib, x, w, K, True, b, bias32, int(gelu), r, zpad=1, zoff=1), x, w, b, gelu, r)
    _check(_run(lib, x, w, K, False, b, bias32, int(gelu), cpad=1, zpad=8, zoff=3), x, w, b, gelu)
    _check(_run(lib, x, w, K, bias32, residual=r, cpad=3), x, w, residual=r)


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("K", [300, 1290])
@pytest.mark.parametrize("t,M,N", ONE, ids=str)
def test_exact_sums(lib, gpu, t, M, N, K, wide):
    """Codes of whole and half numbers with scales of 1, 2 and 1/2: sums of multiples of 1/8, far fewer than 2^24 of them, are exact in fp32, so the
    results are the sums' nearest halves."""
    rng = np.random.default_rng(1)
    x, w = _operand(rng, M, K, 0, 2), _operand(rng, N, K, -1, 1)
    for c in (x[0], w[0]):
        c[(np.abs(R.VALUES[c]) > 1.0) & (rng.random(c.shape) < 0.97)] = 0
    z = _value(*x) @ _value(*w).T
    got = _run(lib, x, w, K, wide)
    assert bool((got == z.half()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("t,M,N", ONE, ids=str)
def test_scales_over_the_range(lib, gpu, t, M, N, wide):
    """Scales far from 1 that meet again near it, the smallest and the largest byte among them, and zeros under any scale."""
    rng = np.random.default_rng(7)
    K = 1400
    x, w = _operand(rng, M, K), _operand(rng, N, K)
    nb = x[1].shape[1]
    e = rng.integers(-100, 100, nb)
    e[:4] = (-120, 120, -127 + 4, 127 - 3)
    x[1][:] = np.clip(127 + e + rng.integers(-2, 2, (M, nb)), 0, 254)
    w[1][:] = np.clip(127 - e - rng.integers(6, 9, (N, nb)), 0, 254)
    x[0][:, 32 * 5: 32 * 6] = 0
    x[1][:, 5], w[1][:, 5] = 254, 100
    _check(_run(lib, x, w, K, wide), x, w)


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("K", [300, 1500])
@pytest.mark.parametrize("t,M,N", ONE, ids=str)
def test_nan_scales(lib, gpu, t, M, N, K, wide):
    """A scale of 255 in any block makes its row (of x) or column (of W) NaN, though its codes are 0, and nothing else."""
    import torch
    rng = np.random.default_rng(9)
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -5)
    nb = x[1].shape[1]
    bad = torch.zeros((M, N), dtype=torch.bool, device="cuda")
    for i, b in enumerate((0, 3, 5, nb - 2, nb - 1)):
        m, n = (M * (i + 1)) // 6 + i, (N * (i + 1)) // 7 + i
        x[1][m, b], w[1][n, nb - 1 - b] = 255, 255
        x[0][m, 32 * b: 32 * b + 32], w[0][n, 32 * (nb - 1 - b): 32 * (nb - b)] = 0, 0
        bad[m], bad[:, n] = True, True
    assert torch.equal(torch.isnan(_run(lib, x, w, K, wide)), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("t,M,N", ONE, ids=str)
def test_one_operand_by_words(lib, gpu, t, M, N):
    """Scales in whole 16 bytes on one side alone, or from an address that is not: the bits of both in whole 16 bytes."""
    import torch
    rng = np.random.default_rng(4)
    K = 1100
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -4)
    want = _run(lib, x, w, K, True)
    nb = x[1].shape[1]
    off = torch.full((M * 48 + 4,), 255, dtype=torch.uint8, device="cuda")
    off[4:].view(M, 48)[:, :nb] = _dev(x[1])
    for (xc, xs), (wc, ws), xo in ((_put(*x, True), _put(*w, False), 0), (_put(*x, False), _put(*w, True), 0), ((_put(*x, True)[0], off.view(-1)), _put(*w, True), 4)):
        z = torch.zeros((M, N), dtype=torch.float16, device="cuda")
        ldxs = 48 if xo else xs.shape[1]
        torch.cuda.synchronize()
        assert lib.sh_gemm_mx4(A(xc), A(xs) + xo, A(wc), A(ws), A(z), M, N, K, xc.shape[1], ldxs, wc.shape[1], ws.shape[1], N, None) == 0, shops.last_error()
        assert torch.equal(z, want)


@pytest.mark.gpu
@pytest.mark.parametrize("t,M,N", ONE, ids=str)
def test_again_and_in_a_graph(lib, gpu, t, M, N):
    """The same bits from call to call, and from replays between eager calls on other rows."""
    import torch
    rng = np.random.default_rng(5)
    K = 1100
    w = _operand(rng, N, K, -9, -4)
    (wc, ws), rows = _put(*w, True), [_put(*_operand(rng, M, K), True) for _ in "abc"]
    xc, xs = (t.clone() for t in rows[0])
    z, g0 = (torch.zeros((M, N), dtype=torch.float16, device="cuda") for _ in "zg")

    def call(a, s, out):
        assert lib.sh_gemm_mx4(A(a), A(s), A(wc), A(ws), A(out), M, N, K, a.shape[1], s.shape[1], wc.shape[1], ws.shape[1], N, None) == 0, shops.last_error()
    torch.cuda.synchronize()
    s, g, prev = torch.cuda.Stream(), torch.cuda.CUDAGraph(), lib.sh_get_stream()
    with torch.cuda.graph(g, stream=s):
        lib.sh_set_stream(s.cuda_stream)
        call(xc, xs, g0)
    lib.sh_set_stream(prev)
    for i in (0, 1, 2, 0):
        xc.copy_(rows[i][0])
        xs.copy_(rows[i][1])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for _ in range(2):
            z.fill_(9.0)
            torch.cuda.synchronize()
            call(*rows[i], z)
            assert torch.equal(z, g0), i
            torch.cuda.synchronize()
