"""sh_gemm_w4 on the GPU against the product in 64 bits (oracle/kv_refs.py)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from conftest import _KEEP, to_dev, to_np
from oracle import kv_refs as R
from softhier_mlir_amd import shops

pytestmark = pytest.mark.gpu
A = shops.addr


def dev(a):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    _KEEP.append(t)
    return t


def _weights(rng, K, N, group, zero):
    G = -(-K // group)
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    scale = (rng.uniform(0.5, 1.5, (G, N)) / np.sqrt(K)).astype(np.float16)
    return codes, scale, rng.integers(0, 16, (G, N)).astype(np.uint8) if zero else None


def _run(lib, x, codes, scale, zero, group, bias=None, bias32=False, act=0, residual=None, pad=0, off=0):
    """The call with every leading dim `pad` wider than it need be and bases `off` elements off the allocation."""
    import torch
    (M, K), N = x.shape, codes.shape[1]
    wide = lambda a, n, fill: np.concatenate([np.full(off, fill, a.dtype), np.pad(a, ((0, 0), (0, n)), constant_values=fill).ravel()])  # noqa: E731
    X, W, S = to_dev(wide(x, pad, np.nan)), dev(wide(R.w4_pack(codes).view(np.int32), pad, -1)), to_dev(wide(scale, pad, np.nan))
    Zp = dev(wide(zero, pad, 255)) if zero is not None else None
    Z = torch.full((off + M * (N + pad),), 9.0, dtype=torch.float16, device="cuda")
    e = None
    if bias is not None or act or residual is not None:
        Bi = 0 if bias is None else dev(bias.astype(np.float32)) if bias32 else to_dev(bias)
        Re = 0 if residual is None else to_dev(residual)
        e = C.byref(shops.epi(bias=A(Bi) if bias is not None else 0, bias_fmt=int(bias32), act=act,
                              residual=A(Re) if residual is not None else 0, ldr=N))
    rc = lib.sh_gemm_w4(A(X, off), A(W, off), A(S, off), A(Zp, off) if zero is not None else 0, A(Z, off), M, N, K, group, K + pad, N + pad, N + pad,
                        N + pad, e)
    assert rc == 0, shops.last_error()
    z = to_np(Z)
    assert (z[:off] == 9.0).all()
    z = z[off:].reshape(M, N + pad)
    assert (z[:, N:] == 9.0).all()
    return z[:, :N].astype(np.float64)


def _check(got, x, codes, scale, zero, group, bias=None, gelu=False, residual=None):
    """Rounding to fp16 (half a step, 2^-11, twice with a residual); sums of x code and of x zero, exact products in fp32: a chain
    of at most 128 within a group, one term for each group of the chain's wave, then the waves, and up to eight more operations,
    each 2^-23 of sum |x| (code + zero) scale at most; GELU's slope is below 1.13, and its hardware exp2 and reciprocal add
    2^-20 of the result."""
    z, _ = R.gemm_w4(x, codes, scale, zero, group, bias, gelu)
    of = np.arange(codes.shape[0]) // group
    s = np.abs(x.astype(np.float64)) @ ((codes + (8.0 if zero is None else zero.astype(np.float64)[of])) * np.abs(scale.astype(np.float64))[of])
    d = (128 + 8 + 8 + codes.shape[0] / 256) * 2.0 ** -23 * (s + (0 if bias is None else np.abs(bias)))
    tol = 2.0 ** -11 * np.abs(z) + (1.13 if gelu else 1.0) * d + 2.0 ** -25 + (2.0 ** -19 * np.abs(z) + 2.0 ** -22 if gelu else 0)
    if residual is not None:
        z = z + residual.astype(np.float64)
        tol = tol * (1 + 2.0 ** -11) + 2.0 ** -11 * np.abs(z) + 2.0 ** -25
    err = np.abs(got - z)
    assert (err <= tol).all(), (float((err - tol).max()), np.argwhere(~(err <= tol))[:4].tolist())


SHAPES = [(1, 1, 8, 32), (1, 16, 32, 32), (1, 64, 128, 128), (1, 2048, 720, 32), (1, 100, 4096, 128), (1, 4096, 1024, 64), (2, 33, 200, 64),
          (5, 68, 1032, 128), (16, 256, 512, 96), (17, 132, 968, 256), (31, 960, 960, 64), (33, 40, 136, 32), (50, 720, 2048, 128), (64, 260, 1608, 128),
          (65, 48, 320, 32), (200, 72, 264, 128), (3, 5000, 64, 32), (64, 64, 16384, 128)]


@pytest.mark.parametrize("zero", [True, False])
@pytest.mark.parametrize("M,N,K,group", SHAPES)
def test_w4(lib, gpu, M, N, K, group, zero):
    rng = np.random.default_rng(M + N + K)
    w = _weights(rng, K, N, group, zero)
    x = rng.standard_normal((M, K)).astype(np.float16)
    _check(_run(lib, x, *w, group), x, *w, group)


@pytest.mark.parametrize("pad,off", [(1, 1), (4, 4), (3, 2)])
@pytest.mark.parametrize("M,N,K,group", [(1, 132, 712, 64), (20, 64, 256, 128), (64, 97, 344, 32)])
def test_w4_strides_and_alignment(lib, gpu, M, N, K, group, pad, off):
    rng = np.random.default_rng(pad + M)
    w = _weights(rng, K, N, group, True)
    x = rng.standard_normal((M, K)).astype(np.float16)
    _check(_run(lib, x, *w, group, pad=pad, off=off), x, *w, group)


@pytest.mark.parametrize("M,N,K", [(1, 960, 720), (50, 200, 512), (7, 33, 96)])
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("bias32", [False, True])
def test_w4_epilogue(lib, gpu, M, N, K, gelu, bias32):
    rng = np.random.default_rng(M)
    w = _weights(rng, K, N, 32, True)
    x, b, r = rng.standard_normal((M, K)).astype(np.float16), rng.standard_normal(N).astype(np.float16), rng.standard_normal((M, N)).astype(np.float16)
    got = _run(lib, x, *w, 32, bias=b, bias32=bias32, act=int(gelu), residual=r)
    _check(got, x, *w, 32, bias=b.astype(np.float64), gelu=gelu, residual=r)


def test_w4_subnormal_and_large_rows(lib, gpu):
    """Rows of the smallest halves and of large ones: the code's own subnormals are exact beside them."""
    rng = np.random.default_rng(4)
    w = _weights(rng, 512, 64, 128, True)
    x = (rng.standard_normal((4, 512)) * np.array([[6e-8], [1e-4], [1.0], [3000.0]])).astype(np.float16)
    w = (w[0], (w[1].astype(np.float32) * 16).astype(np.float16), w[2])
    x[3] = np.clip(x[3], -60, 60)
    _check(_run(lib, x, *w, 128), x, *w, 128)


def test_w4_exact_on_integers(lib, gpu):
    """Small integers throughout: every sum is exact, so are the results."""
    rng = np.random.default_rng(1)
    codes, zero = rng.integers(0, 16, (256, 80)).astype(np.uint8), rng.integers(0, 16, (2, 80)).astype(np.uint8)
    scale = np.exp2(rng.integers(-3, 1, (2, 80))).astype(np.float16)
    x = rng.integers(-1, 2, (9, 256)).astype(np.float16)
    z, _ = R.gemm_w4(x, codes, scale, zero, 128)
    assert np.array_equal(_run(lib, x, codes, scale, zero, 128), z.astype(np.float16).astype(np.float64))


def test_w4_rows_do_not_depend_on_each_other(lib, gpu):
    """A row's bits are the same alone and among 64, and a row of NaN stays in its row."""
    rng = np.random.default_rng(2)
    w = _weights(rng, 1024, 192, 128, True)
    x = rng.standard_normal((64, 1024)).astype(np.float16)
    all_rows = _run(lib, x, *w, 128)
    for m in (0, 17, 40, 63):
        assert np.array_equal(_run(lib, x[m:m + 1], *w, 128)[0], all_rows[m])
    x[5] = np.nan
    z = _run(lib, x, *w, 128)
    assert np.isnan(z[5]).all() and np.array_equal(np.delete(z, 5, 0), np.delete(all_rows, 5, 0))


@pytest.mark.parametrize("N,K,group", [(72, 8200, 128), (700, 12248, 64), (1024, 8192, 128), (1025, 8200, 128), (40, 16384, 32), (2048, 2048, 128)])
def test_w4_long_chains_of_few_columns(lib, gpu, N, K, group):
    """Either side of where sixteen waves share a chain: the product, and a row's bits alone and among others."""
    rng = np.random.default_rng(N + K)
    w = _weights(rng, K, N, group, True)
    x = rng.standard_normal((35, K)).astype(np.float16)
    all_rows = _run(lib, x, *w, group)
    _check(all_rows, x, *w, group)
    for m in (0, 33):
        assert np.array_equal(_run(lib, x[m:m + 1], *w, group)[0], all_rows[m])
    assert np.array_equal(_run(lib, x[:20], *w, group), all_rows[:20])
