"""sh_rope_pos and sh_kv_append_rope where a thread turns several heads by the angles it has: how many follows from the rows, so a call of all rows
is compared with calls of few rows, whose threads have one head each, and some rows with 64 bits."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from conftest import _KEEP
from oracle import rope_mx4_refs as R
from softhier_mlir_amd import shops
from test_gpu_rope import _both, _check, _plan

pytestmark = pytest.mark.gpu
A = shops.addr

# rows, heads, dh, rot, the columns of a group in the kernel (8, 4 or 1), the heads of a thread not in place: rows heads (dh / 2 columns) >> 20
MANY = [(10000, 37, 256, 240, 8, 5), (6000, 37, 256, 248, 4, 6), (3000, 37, 128, 126, 1, 6), (16001, 40, 128, 64, 8, 4), (9000, 40, 128, 128, 8, 2), (20000, 7, 512, 512, 8, 4),
        (9000, 9, 512, 504, 4, 4), (30000, 1, 512, 512, 8, 1), (3000, 41, 72, 72, 4, 1), (5000, 21, 80, 20, 1, 4), (12000, 19, 256, 256, 8, 3), (15000, 13, 200, 200, 4, 4)]


def _heads(rows, heads, chunks, shift=20):
    return min(heads, max(1, rows * heads * chunks >> shift))


@pytest.mark.parametrize("layout", [R.HALF, R.PAIRS])
@pytest.mark.parametrize("in_place,pad,off", [(False, 0, 0), (False, 3, 1), (True, 0, 0), (True, 1, 3)])
@pytest.mark.parametrize("rows,heads,dh,rot,P,hs", MANY)
def test_rows_of_many_heads(lib, gpu, rows, heads, dh, rot, P, hs, in_place, pad, off, layout):
    import torch
    assert P == (8 if dh % 16 == rot % 16 == 0 else 4 if dh % 8 == rot % 8 == 0 else 1) and hs == _heads(rows, heads, dh // (2 * P))
    g = torch.Generator(device="cuda")
    g.manual_seed(rows + rot)
    wide = heads * dh
    ldx, ldy = (wide + pad, wide + pad) if in_place else (wide + pad, wide + 2 * pad)
    X = torch.randn(off + rows * ldx, generator=g, device="cuda", dtype=torch.float32).half()
    Y, Z = (X.clone() if in_place else torch.full((off + rows * ldy,), 9.0, dtype=torch.float16, device="cuda") for _ in "yz")
    pos = torch.randint(-2000, 131072, (rows,), generator=g, device="cuda", dtype=torch.int32)
    step = R.steps(R.frequencies(rot, 1e4))
    plan = _plan(step, layout, 1.25)
    torch.cuda.synchronize()
    assert lib.sh_rope_pos(A(Y, off), A(Y if in_place else X, off), A(pos), plan, rows, heads, dh, ldy, ldx) == 0, shops.last_error()
    few = max(1, (1 << 21) // (heads * (dh // (2 * P))) - 1)                 # rows whose threads have a head each
    assert _heads(few, heads, dh // (2 * P)) == 1
    for r in range(0, rows, few):
        n = min(few, rows - r)
        assert lib.sh_rope_pos(A(Z, off + r * ldy), A(Z if in_place else X, off + r * (ldy if in_place else ldx)), A(pos, r), plan, n, heads, dh, ldy, ldx) == 0
    assert torch.equal(Y.view(torch.int16), Z.view(torch.int16))
    pick = sorted({0, 1, rows // 3, rows // 2, rows - 2, rows - 1} | {int(v) for v in (pos < 0).nonzero()[:3, 0]})
    x = torch.stack([X[off + r * ldx: off + r * ldx + wide] for r in pick]).cpu().numpy()
    y = torch.stack([Y[off + r * ldy: off + r * ldy + wide] for r in pick]).cpu().numpy()
    p = pos[pick].cpu().numpy()
    _check(y, x, step, p, heads, dh, layout, 1.25)
    assert np.array_equal(y[p < 0], x[p < 0] if in_place else np.full_like(y[p < 0], 9.0))


# counts, H, hkv, dh, bs, rot, the heads of a thread of queries
QUERIES = [([8000, 1000], 37, 1, 128, 16, 128, 10), ([7001, 30, 2000], 36, 4, 128, 32, 64, 9), ([6000], 14, 2, 256, 64, 256, 5), ([20000], 6, 1, 80, 16, 24, 2), ([9000, 2], 33, 11, 64, 16, 64, 4)]


@pytest.mark.parametrize("layout", [R.HALF, R.PAIRS])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("counts,H,hkv,dh,bs,rot,hs", QUERIES)
def test_queries_of_many_heads(lib, gpu, counts, H, hkv, dh, bs, rot, hs, in_place, layout):
    """The one call's bits are those of the three, and its queries within their bound of 64 bits."""
    idle = 37
    assert hs == _heads(sum(counts) + idle, H, dh // 8, 19)
    r = _both(lib, 5 + H, counts, H, hkv, dh, bs, shops.SH_FP8, rot, layout, idle=idle, in_place=in_place)
    import torch
    rows, wide = r["x"].shape
    X, q = torch.from_numpy(r["x"]).cuda(), torch.zeros((rows, H * dh), dtype=torch.float16, device="cuda")
    P, S = torch.from_numpy(r["pos"]).cuda(), torch.full((rows,), -1, dtype=torch.int32, device="cuda")      # (no row is stored)
    _KEEP.extend([X, q, P, S])
    torch.cuda.synchronize()
    assert lib.sh_kv_append_rope(C.byref(r["cache"].c), _plan(r["step"], layout), A(q), A(X), A(X, H * dh), A(X, (H + hkv) * dh), A(P), A(S), rows, H, H * dh, wide, wide, wide) == 0
    pick = [0, 1, rows // 3, rows // 2, rows - idle - 1, rows - 1]
    y = q[pick].cpu().numpy()
    assert (y[-1] == 0).all()
    _check(y, r["x"][pick, : H * dh], r["step"], r["pos"][pick], H, dh, layout)


def test_many_heads_in_a_graph(lib, gpu):
    """Captured and replayed at other positions, the eager bits of every replay."""
    import torch
    rows, heads, dh = 9000, 37, 128
    X = torch.randn((rows, heads * dh), device="cuda").half()
    Y, Z = (torch.zeros_like(X) for _ in "yz")
    pos = torch.zeros(rows, dtype=torch.int32, device="cuda")
    plan = _plan(R.steps(R.frequencies(64, 1e4)), R.HALF)

    def call(y):
        assert lib.sh_rope_pos(A(y), A(X), A(pos), plan, rows, heads, dh, heads * dh, heads * dh) == 0, shops.last_error()
    torch.cuda.synchronize()
    s, g, prev = torch.cuda.Stream(), torch.cuda.CUDAGraph(), lib.sh_get_stream()
    with torch.cuda.graph(g, stream=s):
        lib.sh_set_stream(s.cuda_stream)
        call(Y)
    lib.sh_set_stream(prev)
    for i in range(3):
        pos.copy_(torch.randint(0, 131072, (rows,), dtype=torch.int32))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        call(Z)
        torch.cuda.synchronize()
        assert torch.equal(Y.view(torch.int16), Z.view(torch.int16)), i
