"""The serving operators together, as a decoder's step uses them: tables, norm, 4-bit projections, RoPE, the cache's write,
attention over it, the output projection with its residual. A prompt in two chunks, then single tokens, against the same steps
in numpy with the stored intermediates rounded to fp16; captured into a HIP graph and replayed; on a stream of its own."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from conftest import to_np
from oracle import kv_refs as R
from oracle import refs
from softhier_mlir_amd import shops

pytestmark = pytest.mark.gpu
A, ALL = shops.addr, shops.SH_ALL
f16 = lambda x: np.asarray(x, np.float64).astype(np.float16)  # noqa: E731


class Layer:
    """One layer's attention half with its cache, on the GPU and (the same arrays) in numpy."""

    def __init__(self, seed, B, H, hkv, dh, D, bs, ld, pages, rows, fmt, group=32):
        import torch
        rng = np.random.default_rng(seed)
        self.B, self.H, self.hkv, self.dh, self.D, self.bs, self.ld, self.pages, self.rows, self.fmt, self.group = \
            B, H, hkv, dh, D, bs, ld, pages, rows, fmt, group
        self.N, self.KV = (H + 2 * hkv) * dh, hkv * dh
        self.w = {}
        for name, (K, N) in dict(qkv=(D, self.N), out=(H * dh, D)).items():
            codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
            scale = (rng.uniform(0.5, 1.5, (-(-K // group), N)) * 0.25 / np.sqrt(K)).astype(np.float16)
            zero = rng.integers(6, 10, scale.shape).astype(np.uint8)
            self.w[name] = (codes, scale, zero)
        self.gamma = (1 + 0.1 * rng.standard_normal((1, D))).astype(np.float16)
        pos = np.arange(ld * bs)
        th = pos[:, None] * 10000.0 ** (-np.arange(dh // 2) / (dh // 2))[None]
        self.tab = np.concatenate([np.cos(th), np.sin(th)], 1).astype(np.float16)
        # numpy state
        self.table, self.lens = np.zeros((B, ld), np.int32), np.zeros(B, np.int32)
        self.pool, self.state = rng.permutation(pages).astype(np.int32), np.array([0, pages, 0], np.int32)
        self.cache = [np.zeros((pages, hkv, bs, dh), np.uint8), np.zeros((pages, hkv, dh, bs), np.uint8), np.ones((pages, hkv), np.float32),
                      np.ones((pages, hkv), np.float32)]
        # GPU state
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.g = {k: t(getattr(self, k)) for k in ("table", "lens", "pool", "state", "gamma", "tab")}
        self.gc = [t(c) for c in self.cache]
        self.c = shops.kv_cache(*(A(x) for x in self.gc), pages, hkv, dh, bs, fmt)
        self.gw = {k: (t(R.w4_pack(w[0]).view(np.int32)), t(w[1]), t(w[2])) for k, w in self.w.items()}
        i = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        h = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
        self.b = dict(add=i(B), row_start=i(B + 1), slots=i(rows), pos=i(rows), kv_len=i(B), x=h(rows, D), n=h(rows, D), qkv=h(rows, self.N),
                      q=h(rows, H * dh), k=h(rows, self.KV), rows_tab=h(rows, dh), o=h(rows, H * dh), y=h(rows, D))
        torch.cuda.synchronize()

    def step_gpu(self, lib, max_q):
        """The step's calls, on the buffers; the RoPE rows are gathered by position."""
        import torch
        b, g, rows, D, N, H, dh, KV = self.b, self.g, self.rows, self.D, self.N, self.H, self.dh, self.KV
        if not hasattr(self, "ws"):
            self.ws = torch.empty(int(lib.sh_attention_kv_ws_bytes(C.byref(self.c), self.B, rows, rows, H, self.ld)), dtype=torch.uint8, device="cuda")
            self.ws_dec = torch.empty(int(lib.sh_attention_kv_ws_bytes(C.byref(self.c), self.B, rows, 1, H, self.ld)), dtype=torch.uint8, device="cuda")
        ws = self.ws if max_q > 1 else self.ws_dec
        rc = [lib.sh_kv_slots(A(g["table"]), self.ld, A(g["lens"]), A(g["lens"]), A(b["add"]), A(g["pool"]), A(g["state"]), A(g["state"]), A(b["row_start"]),
                              A(b["slots"]), A(b["pos"]), A(b["kv_len"]), self.B, self.bs, self.pages, rows)]
        lib.sh_rmsnorm(A(b["n"]), A(b["x"]), A(g["gamma"]), rows, D, D, 1e-5, ALL)
        w, s, z = self.gw["qkv"]
        rc.append(lib.sh_gemm_w4(A(b["n"]), A(w), A(s), A(z), A(b["qkv"]), rows, N, D, self.group, D, N, N, N, None))
        torch.index_select(g["tab"], 0, b["pos"].clamp_min(0), out=b["rows_tab"])
        b["q"].copy_(b["qkv"][:, : H * dh])
        b["k"].copy_(b["qkv"][:, H * dh: H * dh + KV])
        lib.sh_rope(A(b["q"]), A(b["q"]), A(b["rows_tab"]), rows, H * dh, H * dh, dh, dh, ALL)
        lib.sh_rope(A(b["k"]), A(b["k"]), A(b["rows_tab"]), rows, KV, KV, dh, dh, ALL)
        rc.append(lib.sh_kv_append(C.byref(self.c), A(b["k"]), A(b["qkv"], H * dh + KV), KV, N, A(b["slots"]), rows))
        rc.append(lib.sh_attention_kv(A(b["q"]), A(b["o"]), C.byref(self.c), A(g["table"]), self.ld, A(b["kv_len"]), A(b["row_start"]), self.B, rows,
                                      max_q, H, H * dh, H * dh, dh ** -0.5, 0, A(ws), ws.numel()))
        w, s, z = self.gw["out"]
        e = shops.epi(residual=A(b["x"]), ldr=D)
        rc.append(lib.sh_gemm_w4(A(b["o"]), A(w), A(s), A(z), A(b["y"]), rows, D, H * dh, self.group, H * dh, D, D, D, C.byref(e)))
        assert rc == [0] * 5, (rc, shops.last_error())

    def step_numpy(self, x, add):
        r = R.slots(self.table, self.lens, add, self.pool, self.state, self.bs, self.rows)
        self.table, self.pool, self.lens, self.state = (r[k] for k in ("table", "pool", "lens_out", "state_out"))
        H, dh, KV = self.H, self.dh, self.KV
        qkv = f16(R.gemm_w4(f16(refs.rmsnorm(x, self.gamma, 1e-5)), *self.w["qkv"], self.group)[0])
        tab = self.tab[np.maximum(r["pos"], 0)]
        q, k = (f16(refs.rope(m, tab, dh)) for m in (qkv[:, : H * dh], qkv[:, H * dh: H * dh + KV]))
        self.cache = list(R.append(*self.cache, k, qkv[:, H * dh + KV:], r["slots"], self.fmt))
        o = R.attention(q, *self.cache, self.table, r["kv_len"], r["row_start"], H, dh ** -0.5, self.fmt)[0]
        none = np.isnan(o).all(1)
        y = f16(f16(R.gemm_w4(f16(np.where(none[:, None], 0, o)), *self.w["out"], self.group)[0]).astype(np.float64) + x.astype(np.float64))
        return r, y, none

    def put(self, x, add):
        import torch
        self.b["x"].copy_(torch.from_numpy(x))
        self.b["add"].copy_(torch.from_numpy(np.asarray(add, np.int32)))


def _check(layer, r, y, none):
    for k in ("slots", "pos", "row_start", "kv_len"):
        assert np.array_equal(to_np(layer.b[k]), r[k]), k
    for k in ("table", "lens", "state"):
        assert np.array_equal(to_np(layer.g[k]), getattr(layer, k)), k
    bad, err, _ = refs.close(to_np(layer.b["y"])[~none], y[~none])
    assert bad == 0, err


@pytest.mark.parametrize("fmt,H,hkv,dh,bs", [(shops.SH_INT8, 15, 5, 64, 16), (shops.SH_FP8, 8, 2, 128, 32)])
def test_prompts_then_tokens(lib, gpu, fmt, H, hkv, dh, bs):
    rng = np.random.default_rng(dh)
    layer = Layer(3, B=3, H=H, hkv=hkv, dh=dh, D=320, bs=bs, ld=12, pages=26, rows=64, fmt=fmt)
    steps = [[40, 5, 0], [13, 0, 30], [1, 1, 1], [1, 1, 1], [1, -1, 1], [1, 20, 1], [1, 1, -1], [1, 1, 1]]
    for add in steps:
        x = rng.standard_normal((64, 320)).astype(np.float16)
        layer.put(x, add)
        layer.step_gpu(lib, max(1, max(add)))
        _check(layer, *layer.step_numpy(x, np.array(add, np.int32)))


def test_step_in_a_graph(lib, gpu):
    """A decode step captured once and replayed: lengths, pages and codes go on from replay to replay. The same steps run
    eagerly on other buffers give the same bits, with work of both kinds between."""
    import torch
    kw = dict(B=4, H=12, hkv=3, dh=96, D=256, bs=16, ld=8, pages=40, rows=4, fmt=shops.SH_FP8)
    eager, graph = Layer(5, **kw), Layer(5, **kw)
    rng = np.random.default_rng(1)
    xs = rng.standard_normal((12, 4, 256)).astype(np.float16)
    add = np.array([1, 1, 1, 1], np.int32)
    for la in (eager, graph):
        la.put(xs[0], add)
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    prev = lib.sh_get_stream()
    with torch.cuda.stream(s):
        lib.sh_set_stream(s.cuda_stream)
        graph.step_gpu(lib, 1)                                       # (torch's own allocations)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            graph.step_gpu(lib, 1)
    lib.sh_set_stream(prev)
    torch.cuda.synchronize()
    eager.step_gpu(lib, 1)
    for i in range(1, 12):
        for la in (eager, graph):
            la.put(xs[i], add if i % 5 else np.array([1, -1, 1, 0], np.int32))
        g.replay()
        torch.cuda.synchronize()
        eager.step_gpu(lib, 1)
        torch.cuda.synchronize()
        for k in ("slots", "pos", "row_start", "kv_len", "o", "y"):
            assert torch.equal(eager.b[k].view(torch.uint8), graph.b[k].view(torch.uint8)), (i, k)
        for k in ("table", "lens", "pool", "state"):
            assert torch.equal(eager.g[k], graph.g[k]), (i, k)
        for a, b in zip(eager.gc, graph.gc):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


def test_two_graphs_beside_each_other(lib, gpu):
    """Attention captured twice, each with its own workspace, replayed on two streams at a time: the eager bits of both."""
    import torch
    rng = np.random.default_rng(2)
    kw = dict(B=6, H=16, hkv=4, dh=128, D=64, bs=16, ld=200, pages=1300, rows=6, fmt=shops.SH_INT8)
    one, two = Layer(7, **kw), Layer(8, **kw)
    prev = lib.sh_get_stream()
    runs = []
    for la in (one, two):
        for c in la.gc[:2]:
            c.copy_(torch.from_numpy(rng.integers(0, 256, c.shape).astype(np.uint8)))
        la.b["q"].copy_(torch.from_numpy(rng.standard_normal((6, 16 * 128)).astype(np.float16)))
        la.g["table"].copy_(torch.from_numpy(np.arange(1200, dtype=np.int32).reshape(6, 200)))
        la.b["kv_len"].copy_(torch.from_numpy(np.array([3200, 1, 700, 2048, 0, 999], np.int32)))
        need = int(lib.sh_attention_kv_ws_bytes(C.byref(la.c), 6, 6, 1, 16, 200))
        ws, o = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.zeros(6, 16 * 128, dtype=torch.float16, device="cuda")
        args = (A(la.b["q"]), A(o), C.byref(la.c), A(la.g["table"]), 200, A(la.b["kv_len"]), 0, 6, 6, 1, 16, 2048, 2048, 0.09, 0, A(ws), need)
        torch.cuda.synchronize()
        assert lib.sh_attention_kv(*args) == 0
        torch.cuda.synchronize()
        want = o.clone()
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            lib.sh_set_stream(s.cuda_stream)
            assert lib.sh_attention_kv(*args) == 0
        lib.sh_set_stream(prev)
        runs.append((g, torch.cuda.Stream(), o, want, ws))
    for _ in range(5):
        for g, s, o, _, _ in runs:
            with torch.cuda.stream(s):
                o.zero_()
                g.replay()
        torch.cuda.synchronize()
        for _, _, o, want, _ in runs:
            assert torch.equal(o, want)


def test_first_call_under_capture(lib, gpu):
    """A graph whose capture is the first call of its kernels (a head width nothing else here decodes with)."""
    import torch
    rng = np.random.default_rng(4)
    la = Layer(13, B=3, H=4, hkv=2, dh=112, D=64, bs=32, ld=4, pages=12, rows=3, fmt=shops.SH_INT8)
    la.gc[0].copy_(torch.from_numpy(rng.integers(0, 256, la.gc[0].shape).astype(np.uint8)))
    la.gc[1].copy_(torch.from_numpy(rng.integers(0, 256, la.gc[1].shape).astype(np.uint8)))
    la.b["q"].copy_(torch.from_numpy(rng.standard_normal((3, 4 * 112)).astype(np.float16)))
    table = rng.permutation(12).astype(np.int32).reshape(3, 4)
    la.g["table"].copy_(torch.from_numpy(table))
    la.b["kv_len"].copy_(torch.from_numpy(np.array([128, 5, 77], np.int32)))
    need = int(lib.sh_attention_kv_ws_bytes(C.byref(la.c), 3, 3, 1, 4, 4))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    s, g, prev = torch.cuda.Stream(), torch.cuda.CUDAGraph(), lib.sh_get_stream()
    with torch.cuda.graph(g, stream=s):
        lib.sh_set_stream(s.cuda_stream)
        assert lib.sh_attention_kv(A(la.b["q"]), A(la.b["o"]), C.byref(la.c), A(la.g["table"]), 4, A(la.b["kv_len"]), 0, 3, 3, 1, 4, 448, 448, 0.1, 0,
                                   A(ws), need) == 0, shops.last_error()
    lib.sh_set_stream(prev)
    k, v, ks, vs = (to_np(c) for c in la.gc)
    want = R.attention(to_np(la.b["q"]), k, v, ks, vs, table, [128, 5, 77], None, 4, 0.1, shops.SH_INT8)[0]
    for _ in range(3):
        la.b["o"].zero_()
        g.replay()
        torch.cuda.synchronize()
        bad, err, _ = refs.close(to_np(la.b["o"]), want)
        assert bad == 0, err


@pytest.mark.parametrize("H,hkv,dh,longest,window", [(8, 1, 64, 1, 0), (16, 1, 128, 1, 3000), (4, 2, 96, 4, 0), (8, 1, 128, 20, 0), (4, 1, 64, 40, 2000)])
def test_lengths_that_move_between_replays(lib, gpu, H, hkv, dh, longest, window):
    """Tables, the cache's write and attention in one graph, with a table wide enough that keys are shared between workgroups (8192
    tokens). From replay to replay lengths grow by tokens and by thousands, pass page ends, and requests end and begin; every replay gives the bits
    of the same calls made eagerly on other buffers."""
    import torch
    rng = np.random.default_rng(H + dh + longest)
    B, bs, ld, rows = 4, 16, 512, 4 * longest
    pages = 4 * ld
    kw = dict(B=B, H=H, hkv=hkv, dh=dh, D=32, bs=bs, ld=ld, pages=pages, rows=rows, fmt=shops.SH_FP8)
    both = [Layer(21, **kw), Layer(21, **kw)]
    codes = [rng.integers(0, 256, c.shape).astype(np.uint8) for c in both[0].gc[:2]]
    for c in codes:
        c[(c & 127) == 127] = 1
    kv = rng.standard_normal((rows, H * dh + 2 * hkv * dh)).astype(np.float16)
    stride = kv.shape[1]
    prev, calls = lib.sh_get_stream(), []
    for la in both:
        for t, c in zip(la.gc, codes):
            t.copy_(torch.from_numpy(c))
        la.gc[2].fill_(2.0 ** -7)
        la.gc[3].fill_(2.0 ** -6)
        la.qkv = torch.from_numpy(kv).cuda()
        need = int(lib.sh_attention_kv_ws_bytes(C.byref(la.c), B, rows, longest, H, ld))
        la.ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        la.o = torch.zeros(rows, H * dh, dtype=torch.float16, device="cuda")

        def call(la=la, need=need):
            b, g = la.b, la.g
            rc = [lib.sh_kv_slots(A(g["table"]), ld, A(g["lens"]), A(g["lens"]), A(b["add"]), A(g["pool"]), A(g["state"]), A(g["state"]),
                                  A(b["row_start"]), A(b["slots"]), A(b["pos"]), A(b["kv_len"]), B, bs, pages, rows),
                  lib.sh_kv_append(C.byref(la.c), A(la.qkv, H * dh), A(la.qkv, (H + hkv) * dh), stride, stride, A(b["slots"]), rows),
                  lib.sh_attention_kv(A(la.qkv), A(la.o), C.byref(la.c), A(g["table"]), ld, A(b["kv_len"]), A(b["row_start"]), B, rows, longest, H,
                                      stride, H * dh, dh ** -0.5, window, A(la.ws), need)]
            assert rc == [0, 0, 0], (rc, shops.last_error())
        calls.append(call)
    # the requests' tables for the longest lengths, so that lengths can be set from outside: request b has pages b ld .. (b + 1) ld - 1
    for la in both:
        la.g["table"].copy_(torch.arange(pages, dtype=torch.int32).view(B, ld))
        la.g["state"].copy_(torch.tensor([0, 0, 0], dtype=torch.int32))
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        lib.sh_set_stream(s.cuda_stream)
        calls[1]()
    lib.sh_set_stream(prev)
    lens = [[15, 0, 6000, 31], None, [47, 16, 8000, 4000], None, [8192 - longest, 1, 100, 3200], [0, 0, 0, 0], None, [5000, 5000, 5000, 5000]]
    for i, at in enumerate(lens):
        add = [longest, max(1, longest // 2), 1, 0 if i % 3 == 1 else longest]
        for la in both:
            if at is not None:
                la.g["lens"].copy_(torch.tensor(at, dtype=torch.int32))
            head = la.g["lens"].cpu()
            # the step's new pages come from the ring: it is given those of the table's next entries, in order
            fresh = [int(la.g["table"][b, j]) for b in range(B) for j in range(-(-int(head[b]) // bs), -(-(int(head[b]) + add[b]) // bs))]
            la.g["pool"][: len(fresh)] = torch.tensor(fresh, dtype=torch.int32, device="cuda")
            la.g["state"].copy_(torch.tensor([0, len(fresh), 0], dtype=torch.int32))
            la.b["add"].copy_(torch.tensor(add, dtype=torch.int32))
            la.o.fill_(7.0)
        torch.cuda.synchronize()
        calls[0]()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        one, two = both
        assert int(one.g["state"][2]) == 0 and int(one.b["kv_len"].min()) > 0
        for x, y in [(one.g[k], two.g[k]) for k in ("table", "lens", "pool", "state")] + [(one.b[k], two.b[k]) for k in ("slots", "pos", "row_start", "kv_len")]:
            assert torch.equal(x, y), i
        for x, y in list(zip(one.gc, two.gc)) + [(one.o, two.o)]:
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), i
        n = int(one.b["row_start"][-1])
        want = R.attention(kv[:n, : H * dh], *(to_np(t) for t in one.gc), to_np(one.g["table"]), to_np(one.b["kv_len"]), to_np(one.b["row_start"]), H,
                           dh ** -0.5, shops.SH_FP8, window)[0]
        bad, err, _ = refs.close(to_np(one.o)[:n], want)
        assert bad == 0, (i, err)


def test_on_a_stream_of_its_own(lib, gpu):
    import torch
    rng = np.random.default_rng(9)
    layer = Layer(11, B=2, H=4, hkv=4, dh=32, D=128, bs=64, ld=3, pages=6, rows=40, fmt=shops.SH_INT8)
    s, prev = torch.cuda.Stream(), lib.sh_get_stream()
    try:
        with torch.cuda.stream(s):
            lib.sh_set_stream(s.cuda_stream)
            for add in ([30, 10], [1, 1]):
                x = rng.standard_normal((40, 128)).astype(np.float16)
                layer.put(x, add)
                layer.step_gpu(lib, max(add))
                s.synchronize()
                _check(layer, *layer.step_numpy(x, np.array(add, np.int32)))
    finally:
        lib.sh_set_stream(prev)
