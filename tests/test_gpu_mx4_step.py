"""Rotary positions and the 4-bit products together with the cache, as a decoder's step uses them: tables, norm, rows to codes, the
projection, queries turned and keys turned into the cache, attention, codes again, the output projection with its residual. Each call's result against 64 bits
on what it read; single tokens through the products that take fp16 rows; a step captured into a HIP graph and replayed beside an eager one."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from conftest import to_np
from oracle import kv_refs as K
from oracle import refs
from oracle import rope_mx4_refs as R
from softhier_mlir_amd import shops

pytestmark = pytest.mark.gpu
A, ALL = shops.addr, shops.SH_ALL


class Layer:
    def __init__(self, lib, seed, B, H, hkv, dh, D, bs, ld, pages, rows, fmt, rot, layout):
        import torch
        rng = np.random.default_rng(seed)
        self.lib, self.B, self.H, self.hkv, self.dh, self.D, self.bs, self.ld, self.pages, self.rows, self.fmt, self.rot, self.layout = \
            lib, B, H, hkv, dh, D, bs, ld, pages, rows, fmt, rot, layout
        self.N = (H + 2 * hkv) * dh
        u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")  # noqa: E731
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        f16 = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
        up = lambda n, m: -(-n // m) * m  # noqa: E731
        self.ldc = {k: 16 * -(-k // 32) for k in (D, H * dh)}
        self.lds = {k: up(-(-k // 32), 16) for k in (D, H * dh)}
        self.gamma = torch.from_numpy((1 + 0.1 * rng.standard_normal((1, D))).astype(np.float16)).cuda()
        self.w = {}
        for name, k, n in (("qkv", D, self.N), ("out", H * dh, D)):           # the rows of W^T, by the library's own quantisation
            wt = torch.from_numpy((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float16)).cuda()
            c, s = u8(n, self.ldc[k]), u8(n, self.lds[k])
            assert lib.sh_mx4_quant(A(c), A(s), A(wt), n, k, self.ldc[k], self.lds[k], k) == 0, shops.last_error()
            torch.cuda.synchronize()
            self.w[name] = (c, s)
        self.step = torch.zeros(rot // 2, dtype=torch.int64, device="cuda")
        assert lib.sh_rope_steps(A(self.step), rot, 1e4, shops.SH_ROPE_BANDS, 4.0, 1.0, 4.0, 64) == 0
        self.plan = shops.rope_plan(A(self.step), rot, layout)
        self.g = dict(table=i32(B, ld), lens=i32(B), pool=torch.from_numpy(rng.permutation(pages).astype(np.int32)).cuda(),
                      state=torch.tensor([0, pages, 0], dtype=torch.int32, device="cuda"))
        self.kv = [u8(pages, hkv, bs, dh), u8(pages, hkv, dh, bs)] + [torch.ones(pages, hkv, device="cuda") for _ in "kv"]
        self.c = shops.kv_cache(*(A(t) for t in self.kv), pages, hkv, dh, bs, fmt)
        self.b = dict(add=i32(B), row_start=i32(B + 1), slots=i32(rows), pos=i32(rows), kv_len=i32(B), x=f16(rows, D), n=f16(rows, D), nc=u8(rows, self.ldc[D]),
                      ns=u8(rows, self.lds[D]), qkv=f16(rows, self.N), q=f16(rows, H * dh), o=f16(rows, H * dh), oc=u8(rows, self.ldc[H * dh]),
                      os=u8(rows, self.lds[H * dh]), y=f16(rows, D))
        self.ws = torch.empty(int(lib.sh_attention_kv_ws_bytes(C.byref(self.c), B, rows, rows, H, ld)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

    def run(self, max_q, few):
        """The step's calls; few: the products take the fp16 rows."""
        lib, b, g, D, N, rows, HD = self.lib, self.b, self.g, self.D, self.N, self.rows, self.H * self.dh
        rc = [lib.sh_kv_slots(A(g["table"]), self.ld, A(g["lens"]), A(g["lens"]), A(b["add"]), A(g["pool"]), A(g["state"]), A(g["state"]), A(b["row_start"]),
                              A(b["slots"]), A(b["pos"]), A(b["kv_len"]), self.B, self.bs, self.pages, rows)]
        lib.sh_rmsnorm(A(b["n"]), A(b["x"]), A(self.gamma), rows, D, D, 1e-5, ALL)
        epi = shops.epi(residual=A(b["x"]), ldr=D)
        for src, c, s, w, dst, k, n, e in (("n", "nc", "ns", "qkv", "qkv", D, N, None), ("o", "oc", "os", "out", "y", HD, D, C.byref(epi))):
            wc, ws = (A(t) for t in self.w[w])
            if few:
                rc.append(lib.sh_gemm_mx4_f16(A(b[src]), wc, ws, A(b[dst]), rows, n, k, k, self.ldc[k], self.lds[k], n, e))
            else:
                rc.append(lib.sh_mx4_quant(A(b[c]), A(b[s]), A(b[src]), rows, k, self.ldc[k], self.lds[k], k))
                rc.append(lib.sh_gemm_mx4(A(b[c]), A(b[s]), wc, ws, A(b[dst]), rows, n, k, self.ldc[k], self.lds[k], self.ldc[k], self.lds[k], n, e))
            if src == "n":
                rc.append(lib.sh_kv_append_rope(C.byref(self.c), C.byref(self.plan), A(b["q"]), A(b["qkv"]), A(b["qkv"], HD), A(b["qkv"], HD + self.hkv * self.dh),
                                                A(b["pos"]), A(b["slots"]), rows, self.H, HD, N, N, N))
                rc.append(lib.sh_attention_kv(A(b["q"]), A(b["o"]), C.byref(self.c), A(g["table"]), self.ld, A(b["kv_len"]), A(b["row_start"]), self.B, rows, max_q,
                                              self.H, HD, HD, self.dh ** -0.5, 0, A(self.ws), self.ws.numel()))
        assert not any(rc), (rc, shops.last_error())

    def put(self, x, add):
        import torch
        self.b["x"].copy_(torch.from_numpy(x))
        self.b["add"].copy_(torch.from_numpy(np.asarray(add, np.int32)))
        self.before = [to_np(t).copy() for t in self.kv]

    def weight(self, name, k):
        c, s = (to_np(t) for t in self.w[name])
        return R.value(R.unpack(c), s[:, : -(-k // 32)])

    def check(self, few):
        b = {k: to_np(v) for k, v in self.b.items()}
        H, hkv, dh, D, HD = self.H, self.hkv, self.dh, self.D, self.H * self.dh
        live = b["pos"] >= 0
        bad, err, _ = refs.close(b["n"], refs.rmsnorm(b["x"], to_np(self.gamma), 1e-5))
        assert bad == 0, ("norm", err)
        for src, c, s, w, dst, k, res in (("n", "nc", "ns", "qkv", "qkv", D, None), ("o", "oc", "os", "out", "y", HD, "x")):
            xc, xs = R.quant(b[src])
            if not few:
                assert np.array_equal(R.unpack(b[c]), xc) and np.array_equal(b[s][:, : xs.shape[1]], xs), src
            z = R.gemm(R.value(xc, xs), self.weight(w, k))[0].astype(np.float16).astype(np.float64)
            if res:
                z = z + b[res].astype(np.float64)
            bad, err, _ = refs.close(b[dst], z)
            assert bad == 0, (dst, err)
        t = R.turn(b["qkv"][:, : (H + hkv) * dh], to_np(self.step).view(np.uint64), b["pos"], H + hkv, dh, self.layout)
        bad, err, _ = refs.close(b["q"][live], t[live, :HD])
        assert bad == 0, ("queries", err)
        # the cache: of the turned keys, of which one in thousands rounds to the next half; so codes are compared as values, to a code's step
        want = K.append(*self.before, np.nan_to_num(t[:, HD:]).astype(np.float16), b["qkv"][:, HD + hkv * dh:], b["slots"], self.fmt)
        got = [to_np(x) for x in self.kv]
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[3], want[3]) and np.array_equal(got[2], want[2])
        assert np.mean(got[0] != want[0]) < 0.01
        d = np.abs(K.value(got[0], self.fmt) - K.value(want[0], self.fmt))
        assert (d <= np.maximum(1.0, 2.0 ** -3 * np.abs(K.value(want[0], self.fmt)))).all()
        o = K.attention(b["q"], *got, to_np(self.g["table"]), b["kv_len"], b["row_start"], H, dh ** -0.5, self.fmt)[0]
        rows = ~np.isnan(o).all(1)
        bad, err, _ = refs.close(b["o"][rows], o[rows])
        assert bad == 0, ("attention", err)


@pytest.mark.parametrize("fmt,H,hkv,dh,rot,layout,bs", [(shops.SH_INT8, 15, 5, 64, 64, R.HALF, 16), (shops.SH_FP8, 8, 2, 128, 64, R.PAIRS, 32)])
def test_prompts_then_tokens(lib, gpu, fmt, H, hkv, dh, rot, layout, bs):
    rng = np.random.default_rng(dh)
    layer = Layer(lib, 3, B=3, H=H, hkv=hkv, dh=dh, D=320, bs=bs, ld=12, pages=26, rows=64, fmt=fmt, rot=rot, layout=layout)
    for add in ([40, 5, 0], [13, 0, 30], [1, 1, 1], [1, -1, 1], [1, 20, 1], [1, 1, 1]):
        x = rng.standard_normal((64, 320)).astype(np.float16)
        layer.put(x, add)
        layer.run(max(1, max(add)), False)
        layer.check(False)


def test_many_rows(lib, gpu):
    """Chunks of prompts: the products in tiles, pages shared out in groups of rows."""
    rng = np.random.default_rng(2)
    layer = Layer(lib, 4, B=4, H=4, hkv=2, dh=64, D=256, bs=16, ld=24, pages=110, rows=640, fmt=shops.SH_FP8, rot=48, layout=R.HALF)
    for add in ([200, 150, 33, 1], [1, 1, 100, 300]):
        layer.put(rng.standard_normal((640, 256)).astype(np.float16), add)
        layer.run(max(add), False)
        layer.check(False)


def test_single_tokens_in_a_graph(lib, gpu):
    """A step of single tokens with fp16 rows into the products, captured once and replayed: lengths, pages and positions go on from replay to replay,
    requests end; the eager steps on other buffers give the same bits, and each is checked."""
    import torch
    kw = dict(B=6, H=12, hkv=3, dh=96, D=256, bs=16, ld=8, pages=60, rows=6, fmt=shops.SH_FP8, rot=96, layout=R.HALF)
    eager, graph = Layer(lib, 5, **kw), Layer(lib, 5, **kw)
    rng = np.random.default_rng(1)
    xs = rng.standard_normal((14, 6, 256)).astype(np.float16)
    one = np.ones(6, np.int32)
    for la in (eager, graph):
        la.put(xs[0], one)
    torch.cuda.synchronize()
    s, g, prev = torch.cuda.Stream(), torch.cuda.CUDAGraph(), lib.sh_get_stream()
    with torch.cuda.graph(g, stream=s):
        lib.sh_set_stream(s.cuda_stream)
        graph.run(1, True)
    lib.sh_set_stream(prev)
    for i in range(14):
        add = one if i % 5 else np.array([1, -1, 1, 0, 1, 1], np.int32)
        for la in (eager, graph):
            la.put(xs[i], add)
        g.replay()
        torch.cuda.synchronize()
        eager.run(1, True)
        torch.cuda.synchronize()
        for k in ("slots", "pos", "kv_len", "qkv", "q", "o", "y"):
            assert torch.equal(eager.b[k].view(torch.uint8), graph.b[k].view(torch.uint8)), (i, k)
        for a, b in zip(eager.kv, graph.kv):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i
        eager.check(True)
