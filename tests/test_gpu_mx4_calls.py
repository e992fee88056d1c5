"""Calls of sh_gemm_mx4 and sh_gemm_mx4_f16 that their header allows: the residual that is the result's own memory, a few columns of many rows, addresses and
leading dims of any alignment that is allowed, work on two streams at once."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from oracle import rope_mx4_refs as R
from softhier_mlir_amd import shops
from test_gpu_mx4_tiles import ONE, _check, _dev, _operand, _put

pytestmark = pytest.mark.gpu
A = shops.addr

# the kernel for few rows with 16, 32 and 64 of them, then the tiles
FEW = [(1, 515), (16, 1029), (30, 5003), (31, 515), (40, 517), (64, 1031)]
ALL = FEW + [(M, N) for _, M, N in ONE]


def _call(lib, x, w, K, z, ldz, epi=None, off=0):
    (xc, xs), (wc, ws) = x, w
    return lib.sh_gemm_mx4(A(xc), A(xs), A(wc), A(ws), A(z, off), len(xc), len(wc), K, xc.shape[1], xs.shape[1], wc.shape[1], ws.shape[1], ldz, epi)


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("pad,off", [(0, 0), (5, 3)])
@pytest.mark.parametrize("M,N", ALL)
def test_residual_in_place(lib, gpu, M, N, pad, off, gelu):
    """z on its way through a decoder's layers: each result takes the place of the residual that was added."""
    import torch
    rng = np.random.default_rng(M + N)
    K = 1000
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -5)
    b, r = rng.standard_normal(N).astype(np.float16), rng.standard_normal((M, N)).astype(np.float16)
    B = torch.zeros(N + 1, dtype=torch.float16, device="cuda")
    B[1:] = _dev(b)                                                      # (a bias at an odd place)
    Z = torch.full((off + M * (N + pad),), 9.0, dtype=torch.float16, device="cuda")
    z = Z[off:].view(M, N + pad)
    z[:, :N] = _dev(r)
    e = shops.epi(bias=A(B, 1), act=int(gelu), residual=A(Z, off), ldr=N + pad, splits=1)
    ops = _put(*x, True), _put(*w, True)
    torch.cuda.synchronize()
    assert _call(lib, *ops, K, Z, N + pad, C.byref(e), off) == 0, shops.last_error()
    _check(z[:, :N], x, w, b, gelu, r)
    assert bool((Z[:off] == 9.0).all()) and bool((z[:, N:] == 9.0).all())
    if M <= 16:
        h = rng.standard_normal((M, K)).astype(np.float16)
        H = _dev(h)
        z[:, :N] = _dev(r)
        torch.cuda.synchronize()
        wc, ws = ops[1]
        assert lib.sh_gemm_mx4_f16(A(H), A(wc), A(ws), A(Z, off), M, N, K, K, wc.shape[1], ws.shape[1], N + pad, C.byref(e)) == 0, shops.last_error()
        _check(z[:, :N], R.quant(h), w, b, gelu, r)


@pytest.mark.parametrize("K", [31, 700])
@pytest.mark.parametrize("N", [1, 2, 3, 7, 8, 9])
@pytest.mark.parametrize("M", [1, 20, 64, 65, 300, 20000, 70001])
def test_few_columns(lib, gpu, M, N, K):
    """Rows of fewer than eight columns, whose residual and result are not read or written past them."""
    import torch
    rng = np.random.default_rng(M + N + K)
    x, w = _operand(rng, M, K), _operand(rng, N, K, -9, -4)
    b, r = rng.standard_normal(N).astype(np.float16), rng.standard_normal((M, N)).astype(np.float16)
    B, z = _dev(b.astype(np.float32)), _dev(r)
    ops = _put(*x, False), _put(*w, True)
    Z = torch.full((3 + M * N + 3,), 9.0, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    assert _call(lib, *ops, K, Z, N, C.byref(shops.epi(bias=A(B), bias_fmt=shops.SH_BIAS_FP32, residual=A(z), ldr=N)), 3) == 0, shops.last_error()
    _check(Z[3:3 + M * N].view(M, N), x, w, b, False, r)
    assert bool((Z[:3] == 9.0).all()) and bool((Z[3 + M * N:] == 9.0).all())


def test_two_streams_at_once(lib, gpu):
    """Products of each kernel on two streams, neither waiting for the other: the bits that each has alone."""
    import torch
    rng = np.random.default_rng(3)
    K, jobs = 1100, []
    for M, N in ALL:
        ops = _put(*_operand(rng, M, K), True), _put(*_operand(rng, N, K, -9, -4), True)
        jobs.append((ops, *(torch.zeros((M, N), dtype=torch.float16, device="cuda") for _ in "abc")))
    torch.cuda.synchronize()
    for ops, z, _, _ in jobs:
        assert _call(lib, *ops, K, z, z.shape[1]) == 0, shops.last_error()
    torch.cuda.synchronize()
    streams, prev = [torch.cuda.Stream() for _ in "ab"], lib.sh_get_stream()
    try:
        for i in range(len(jobs)):
            for s, j, k in ((streams[0], jobs[i], 2), (streams[1], jobs[-1 - i], 3)):
                lib.sh_set_stream(s.cuda_stream)
                assert _call(lib, *j[0], K, j[k], j[k].shape[1]) == 0, shops.last_error()
    finally:
        lib.sh_set_stream(prev)
    torch.cuda.synchronize()
    for _, z, a, b in jobs:
        assert torch.equal(a, z) and torch.equal(b, z)
