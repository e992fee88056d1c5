"""The operators of a decoder's serving step, as they are measured: the 8-bit paged key/value cache (its tables, its
writes, the attention that reads it) and the products with 4-bit weights.

A case is a dict of plain values. `prepare` makes what a serving program holds before the call; `run` is one pass, through
the library's entry points where `own` is true and in elementary torch operations (fp32, rounded once at the end) where it
is false; `exact` computes the same outputs in 64 bits, written apart from both; `work` is what a pass cannot do without.

  slots   sh_kv_slots: from the requests' lengths and what each adds, the block table's new pages (from a ring of free
          pages, which ended requests refill), row offsets, slots, positions and key counts
  append  sh_kv_append: new key and value rows into the pages at those slots, in 8 bits with one power-of-two scale for
          each page and head; a page whose scale grows has its older tokens rescaled
  attn    sh_attention_kv: causal attention of the new rows over the cached keys, ragged, grouped heads, optional window
  w4      sh_gemm_w4: z = x . ((code - zero) scale) + bias [+ residual] for few rows, scales per group of k

Every pass leaves its state so that the next one computes the same outputs: `slots` writes its new lengths and ring state
beside the old ones, and appending the same rows at the same slots twice stores the same codes.
"""
from __future__ import annotations

import math
import random

import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}


# ---- the cases --------------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one decode step of 64 running requests: one token each, a new page for about one in 16
        dict(name="slots_decode_b64", kind="slots", B=64, bs=16, ld=256, pages=12000, prompts=0, longest=1, ended=0, shape=1),
        # a scheduler's mixed step: 900 decodes, 64 prompts of up to 4000 tokens, 60 requests that ended
        dict(name="slots_mixed_b1024", kind="slots", B=1024, bs=16, ld=1024, pages=700000, prompts=64, longest=4000, ended=60, shape=2),
        # the step's new keys and values of 64 requests
        dict(name="append_decode_b64", kind="append", B=64, bs=16, hkv=8, dh=128, fmt="e4m3", pages=2048, longest=1, shape=3),
        # the first chunk of a few prompts, 64-wide heads, pages of 32 tokens that the prompts do not fill
        dict(name="append_prompts", kind="append", B=9, bs=32, hkv=8, dh=64, fmt="int8", pages=1200, longest=4096, shape=4),
        # one user's decode step with the 15 query heads over 5 key/value heads of the vision-language decoder: latency
        dict(name="attn_decode_b1", kind="attn", B=1, H=15, hkv=5, dh=64, bs=16, fmt="int8", held=937, held_lo=937, q=1, q_lo=1,
             window=0, shape=5),
        # a serving batch, contexts from a hundred tokens to 16 thousand
        dict(name="attn_decode_ragged_b48", kind="attn", B=48, H=32, hkv=8, dh=128, bs=16, fmt="e4m3", held=16384, held_lo=100, q=1,
             q_lo=1, window=0, shape=6),
        # two requests with a book in their context: the long axis has to be shared out
        dict(name="attn_decode_long_b2", kind="attn", B=2, H=32, hkv=8, dh=128, bs=64, fmt="int8", held=131000, held_lo=120001, q=1,
             q_lo=1, window=0, shape=7),
        # four drafted tokens checked at once under a sliding window, heads of 80
        dict(name="attn_draft_window_dh80", kind="attn", B=24, H=16, hkv=4, dh=80, bs=16, fmt="int8", held=6000, held_lo=50, q=4, q_lo=4,
             window=1024, shape=8),
        # chunks of prompts beside decodes, over what earlier chunks left in the cache: the compute-bound end
        dict(name="attn_chunks_b8", kind="attn", B=8, H=32, hkv=8, dh=128, bs=32, fmt="e4m3", held=8000, held_lo=1, q=2048, q_lo=1,
             window=0, shape=9),
        # the expert's gated MLP product for a single token: latency, a last group of 16
        dict(name="w4_m1_expert", kind="w4", M=1, N=2048, K=720, group=32, zero=True, bias=False, residual=False),
        # the widest product of a larger decoder for a single token: the bytes of the weight
        dict(name="w4_m1_wide", kind="w4", M=1, N=14336, K=4096, group=128, zero=True, bias=False, residual=False),
        # a batch of 50 rows, with bias and residual, symmetric codes
        dict(name="w4_m50_residual", kind="w4", M=50, N=4096, K=8192, group=128, zero=False, bias=True, residual=True),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case: dict) -> float:
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 4e14)


def _draw(rng) -> dict:
    kind = rng.choice(["slots", "append", "append", "attn", "attn", "attn", "attn", "w4", "w4", "w4"])
    shape = rng.randrange(1 << 30)
    if kind == "slots":
        B, bs = _log(rng, 1, 1024), rng.choice([16, 32, 64])
        longest = rng.choice([1, 1, _log(rng, 2, 4000)])
        ld = -(-_log(rng, 4100, 16384) // bs)
        prompts = 0 if longest == 1 else max(1, min(B, 64) // 2)
        return dict(kind=kind, B=B, bs=bs, ld=ld, pages=B * ld // 2 + 4100 // bs * (prompts + 1), prompts=prompts, longest=longest,
                    ended=rng.choice([0, B // 8]), shape=shape)
    if kind == "append":
        bs, hkv, dh, longest = rng.choice([16, 32, 64]), rng.choice([1, 2, 4, 5, 8]), rng.choice([32, 64, 80, 96, 128, 256]), \
            rng.choice([1, 1, 4, _log(rng, 2, 4096)])
        B = _log(rng, 1, 256) if longest <= 4 else _log(rng, 1, 9)
        return dict(kind=kind, B=B, bs=bs, hkv=hkv, dh=dh, fmt=rng.choice(["int8", "e4m3"]), pages=B * (longest // bs + 3) + 5,
                    longest=longest, shape=shape)
    if kind == "attn":
        hkv, grp = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        if hkv * grp > 64:
            grp = 8
        q = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 9, 2048)])
        held = _log(rng, 1, 131072 if q == 1 else 16384 if q <= 8 else 8192)
        return dict(kind=kind, B=_log(rng, 1, 64 if q <= 8 else 8), H=hkv * grp, hkv=hkv, dh=rng.choice([32, 64, 64, 80, 96, 128, 128, 256]),
                    bs=rng.choice([16, 32, 64]), fmt=rng.choice(["int8", "e4m3"]), held=held, held_lo=max(1, held // rng.choice([1, 4, 100])),
                    q=q, q_lo=rng.choice([1, q]), window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), shape=shape)
    M = rng.choice([1, 1, 1, _log(rng, 2, 64), _log(rng, 2, 64)])
    group = rng.choice([32, 64, 128, 128])
    return dict(kind=kind, M=M, N=_log(rng, 64, 16384), K=8 * _log(rng, 16, 2048), group=group, zero=rng.random() < 0.7,
                bias=rng.random() < 0.5, residual=rng.random() < 0.5)


def draw(rng) -> dict:
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    while True:
        c = _draw(rng)
        if _cost(c) <= most[c["kind"]] and (c["kind"] != "attn" or _cache_bytes(c) <= 3 << 29):
            return c


# ---- lengths: a case has its own, another seed has them in another order -----------------------------------------
def _spread(rng, lo: int, hi: int, n: int) -> list[int]:
    """n lengths over [lo, hi], the longest one among them."""
    v = [_log(rng, lo, hi) for _ in range(n)]
    v[rng.randrange(n)] = hi
    return v


def _slot_lengths(case: dict) -> tuple[list[int], list[int]]:
    """(tokens held, tokens added or -1 for a request that ended) of each request."""
    rng, B = random.Random(case["shape"]), case["B"]
    cap = case["ld"] * case["bs"]
    add = [1] * B
    for b in range(min(B, case["prompts"])):
        add[b] = _log(rng, 1, case["longest"])
    for b in range(B - case["ended"], B):
        add[b] = -1
    held = [0 if b < case["prompts"] and rng.random() < 0.8 else rng.randint(0, cap // 2 - 1) for b in range(B)]
    return [min(h, cap - max(a, 0)) for h, a in zip(held, add)], add


def _append_lengths(case: dict) -> tuple[list[int], list[int]]:
    """(tokens held in the first page written, tokens added) of each request."""
    rng, B = random.Random(case["shape"]), case["B"]
    add = _spread(rng, max(1, case["longest"] // 8), case["longest"], B)
    return [rng.randrange(case["bs"]) if a <= 4 or rng.random() < 0.3 else 0 for a in add], add


def _attn_lengths(case: dict) -> tuple[list[int], list[int]]:
    """(keys with the new ones, new rows) of each request."""
    rng, B = random.Random(case["shape"]), case["B"]
    new = _spread(rng, case["q_lo"], case["q"], B)
    return [h + n - 1 for h, n in zip(_spread(rng, case["held_lo"], case["held"], B), new)], new


def _pairs(L: int, n: int, window: int) -> int:
    """Key and query pairs of n new rows at the end of L keys."""
    first = L - n + 1
    if not window or window >= L:
        return n * first + n * (n - 1) // 2
    return sum(min(first + i, window) for i in range(n))


def _reach(L: int, n: int, window: int) -> int:
    """Keys that any of the n last rows sees."""
    return min(L, window + n - 1) if window else L


def _cache_bytes(case: dict) -> int:
    return sum(2 * L * case["hkv"] * case["dh"] for L in _attn_lengths(case)[0])


def work(case: dict) -> dict:
    k = case["kind"]
    if k == "slots":
        held, add = _slot_lengths(case)
        bs, rows = case["bs"], sum(max(a, 0) for a in add)
        new = sum(-(-(h + a) // bs) - -(-h // bs) for h, a in zip(held, add) if a > 0)
        back = sum(-(-h // bs) for h, a in zip(held, add) if a < 0)
        # per request: held and added read, new length, key count and row offset written, its last page read
        return {"bytes": case["B"] * 24 + rows * 8 + (new + back) * 8, "flops": rows * 4}
    if k == "append":
        held, add = _append_lengths(case)
        bs, n = case["bs"], sum(add)
        runs = sum((h + a - 1) // bs + 1 for h, a in zip(held, add))
        return {"bytes": n * case["hkv"] * case["dh"] * 2 * 3 + runs * case["hkv"] * 8 + n * 4, "flops": n * case["hkv"] * case["dh"] * 2 * 3}
    if k == "attn":
        L, new = _attn_lengths(case)
        keys = sum(_reach(a, n, case["window"]) for a, n in zip(L, new))
        pages = sum(-(-_reach(a, n, case["window"]) // case["bs"]) for a, n in zip(L, new))
        pairs = sum(_pairs(a, n, case["window"]) for a, n in zip(L, new))
        return {"bytes": keys * case["hkv"] * case["dh"] * 2 + pages * (case["hkv"] * 8 + 4) + sum(new) * case["H"] * case["dh"] * 4,
                "flops": 4 * case["dh"] * case["H"] * pairs}
    M, N, K, G = case["M"], case["N"], case["K"], -(-case["K"] // case["group"])
    b = K * N // 2 + G * N * (3 if case["zero"] else 2) + M * K * 2 + M * N * 2
    b += N * 2 * case["bias"] + M * N * 2 * case["residual"]
    return {"bytes": b, "flops": 2 * M * N * K}


# ---- inputs -----------------------------------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed: int):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        self.host = random.Random(seed)

    def normal(self, *shape, std: float = 1.0):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32).mul_(std)

    def order(self, n: int):
        return torch.randperm(n, generator=self.g, device="cuda")

    def codes(self, *shape, high: int = 256):
        return torch.randint(0, high, shape, generator=self.g, device="cuda", dtype=torch.uint8)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _slots_state(case: dict, r: _Rand) -> dict:
    held, add = _slot_lengths(case)
    order = list(range(case["B"]))
    r.host.shuffle(order)
    held, add = [held[i] for i in order], [add[i] for i in order]
    B, bs, ld, pages = case["B"], case["bs"], case["ld"], case["pages"]
    rows = sum(max(a, 0) for a in add)
    perm = r.order(pages).to(torch.int32)
    have = [-(-h // bs) for h in held]
    table = torch.full((B, ld), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(ld, device="cuda")[None, :] < _i32(have)[:, None]
    table[at] = perm[: sum(have)]
    free = pages - sum(have)
    head = r.host.randrange(pages)
    pool = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    pool[(head + torch.arange(free, device="cuda")) % pages] = perm[sum(have):]
    e = lambda n: torch.full((n,), -7, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(table=table, lens=_i32(held), add=_i32(add), pool=pool, state=_i32([head, free, 0]), lens_out=e(B), state_out=e(3),
                row_start=e(B + 1), slots=e(rows), pos=e(rows), kv_len=e(B), rows=rows)


def _channels(r: _Rand, hkv: int, dh: int):
    """A few channels of a key are larger than the others by an order of magnitude."""
    c = torch.ones(hkv, dh, device="cuda")
    c[torch.rand(hkv, dh, generator=r.g, device="cuda") < 0.03] = 8.0
    return c


def _append_state(case: dict, r: _Rand) -> dict:
    held, add = _append_lengths(case)
    order = list(range(case["B"]))
    r.host.shuffle(order)
    bs, hkv, dh, pages = case["bs"], case["hkv"], case["dh"], case["pages"]
    perm = r.order(pages).tolist()
    slots, n = [], 0
    for i in order:
        first = n
        n += (held[i] + add[i] - 1) // bs + 1
        slots += [perm[first + p // bs] * bs + p % bs for p in range(held[i], held[i] + add[i])]
    rows = len(slots)
    fp8 = case["fmt"] == "e4m3"
    k, v = (r.codes(pages, hkv, *s, high=120 if fp8 else 256) for s in ((bs, dh), (dh, bs)))
    ks, vs = (torch.exp2(torch.randint(-9 if fp8 else -7, -5 if fp8 else -3, (pages, hkv), generator=r.g, device="cuda").float()) for _ in "kv")
    x = r.normal(rows, hkv, dh) * _channels(r, hkv, dh)
    y = r.normal(rows, hkv, dh, std=0.5)
    kv = torch.cat([x.reshape(rows, -1), y.reshape(rows, -1)], 1).to(torch.float16)     # the k | v columns of one projection
    return dict(k=k, v=v, ks=ks, vs=vs, kv=kv, slots=_i32(slots), rows=rows, hkv=hkv, dh=dh, bs=bs, pages=pages, fmt=case["fmt"])


def _pow2_scale(amax, fmt: str):
    """The smallest power of two s with amax <= s * the format's largest value, and at least 2^-32."""
    f, e = torch.frexp(amax.clamp_min(2.0 ** -60))
    m, x = (0.9921875, 7) if fmt == "int8" else (0.875, 9)
    e = torch.where(f <= m, e - x, e - x + 1).clamp_min(-32)
    return ((e + 127) << 23).view(torch.float32)


def _to_codes(x, fmt: str):
    """8-bit codes, as bytes, of values already divided by their scale."""
    if fmt == "int8":
        return x.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _from_codes(c, fmt: str):
    return c.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).to(torch.float32)


def _attn_state(case: dict, r: _Rand) -> dict:
    L, new = _attn_lengths(case)
    order = list(range(case["B"]))
    r.host.shuffle(order)
    L, new = [L[i] for i in order], [new[i] for i in order]
    B, H, hkv, dh, bs, fmt = (case[n] for n in ("B", "H", "hkv", "dh", "bs", "fmt"))
    need = [-(-a // bs) for a in L]
    pages, ld = sum(need) + 3, max(need)
    perm = r.order(pages).to(torch.int32)
    table = torch.zeros(B, ld, dtype=torch.int32, device="cuda")
    table[torch.arange(ld, device="cuda")[None, :] < _i32(need)[:, None]] = perm[: sum(need)]
    k = torch.empty(pages, hkv, bs, dh, dtype=torch.uint8, device="cuda")
    v = torch.empty(pages, hkv, dh, bs, dtype=torch.uint8, device="cuda")
    ks, vs = torch.empty(pages, hkv, device="cuda"), torch.empty(pages, hkv, device="cuda")
    ck = _channels(r, hkv, dh)
    step = max(1, (1 << 25) // (hkv * bs * dh))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = (r.normal(n, hkv, bs, dh) * ck[None, :, None, :]).to(torch.float16).float()
        y = (r.normal(n, hkv, dh, bs) * (0.2 + torch.rand(n, hkv, 1, 1, generator=r.g, device="cuda"))).to(torch.float16).float()
        for t, (codes, scale) in ((x, (k, ks)), (y, (v, vs))):
            s = _pow2_scale(t.abs().amax((2, 3)), fmt)
            scale[p:p + n] = s
            codes[p:p + n] = _to_codes(t / s[:, :, None, None], fmt)
    rows = sum(new)
    q = r.normal(rows, H * dh).to(torch.float16)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return dict(k=k, v=v, ks=ks, vs=vs, table=table, kv_len=_i32(L), row_start=_i32(start), q=q, o=torch.empty_like(q), L=L, new=new,
                rows=rows, B=B, H=H, hkv=hkv, dh=dh, bs=bs, fmt=fmt, pages=pages, ld=ld, max_q=max(new), window=case["window"],
                scale=dh ** -0.5)


def _w4_state(case: dict, r: _Rand) -> dict:
    M, N, K, g = case["M"], case["N"], case["K"], case["group"]
    G = -(-K // g)
    # codes about the middle of the range, as a rounded bell of weights gives, eight of consecutive k in a word
    c = (r.normal(K, N, std=2.6) + 8.0).round_().clamp_(0, 15).to(torch.int32).view(K // 8, 8, N)
    w = torch.zeros(K // 8, N, dtype=torch.int32, device="cuda")
    for j in range(8):
        w |= c[:, j] << (4 * j)
    s = ((0.5 + torch.rand(G, N, generator=r.g, device="cuda")) * (0.4 * K ** -0.5)).to(torch.float16)
    z = r.codes(G, N, high=5).add_(6) if case["zero"] else None
    d = dict(w=w, s=s, zp=z, x=r.normal(M, K).to(torch.float16), out=torch.empty(M, N, dtype=torch.float16, device="cuda"),
             M=M, N=N, K=K, group=g, bias=None, residual=None)
    if case["bias"]:
        d["bias"] = r.normal(N, std=0.1).to(torch.float16)
    if case["residual"]:
        d["residual"] = r.normal(M, N).to(torch.float16)
    return d


def _state(case: dict, seed: int) -> dict:
    s = {"slots": _slots_state, "append": _append_state, "attn": _attn_state, "w4": _w4_state}[case["kind"]](case, _Rand(seed))
    s["kind"], s["case"] = case["kind"], case
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _state(case, seed)
    if own:
        _calls(case, s)
    return s


# ---- the library's entry points, their arguments converted once ----------------------------------------------------
def _calls(case: dict, s: dict) -> None:
    import ctypes

    from softhier_mlir_amd import shops
    lib, A, k = shops.load(), shops.addr, s["kind"]
    lib.sh_init()
    fmt = {"int8": shops.SH_INT8, "e4m3": shops.SH_FP8}
    if k in ("append", "attn"):
        s["cache"] = shops.kv_cache(A(s["k"]), A(s["v"]), A(s["ks"]), A(s["vs"]), s["pages"], s["hkv"], s["dh"], s["bs"], fmt[s["fmt"]])
        c = ctypes.byref(s["cache"])
    if k == "slots":
        s["fn"], s["args"] = lib.sh_kv_slots, (
            A(s["table"]), case["ld"], A(s["lens"]), A(s["lens_out"]), A(s["add"]), A(s["pool"]), A(s["state"]), A(s["state_out"]),
            A(s["row_start"]), A(s["slots"]), A(s["pos"]), A(s["kv_len"]), case["B"], case["bs"], case["pages"], s["rows"])
    elif k == "append":
        n = s["hkv"] * s["dh"]
        s["fn"], s["args"] = lib.sh_kv_append, (c, A(s["kv"]), A(s["kv"], n), 2 * n, 2 * n, A(s["slots"]), s["rows"])
    elif k == "attn":
        D = s["H"] * s["dh"]
        need = lib.sh_attention_kv_ws_bytes(c, s["B"], s["rows"], s["max_q"], s["H"], s["ld"])
        s["ws"] = torch.empty(max(1, int(need)), dtype=torch.uint8, device="cuda")
        s["fn"], s["args"] = lib.sh_attention_kv, (
            A(s["q"]), A(s["o"]), c, A(s["table"]), s["ld"], A(s["kv_len"]), A(s["row_start"]), s["B"], s["rows"], s["max_q"], s["H"],
            D, D, s["scale"], s["window"], A(s["ws"]), s["ws"].numel())
    else:
        N = s["N"]
        s["epi"] = shops.epi(bias=A(s["bias"]) if s["bias"] is not None else 0, residual=A(s["residual"]) if s["residual"] is not None else 0,
                             ldr=N if s["residual"] is not None else 0)
        s["fn"], s["args"] = lib.sh_gemm_w4, (
            A(s["x"]), A(s["w"]), A(s["s"]), A(s["zp"]) if s["zp"] is not None else 0, A(s["out"]), s["M"], N, s["K"], s["group"],
            s["K"], N, N, N, ctypes.byref(s["epi"]))


def _outputs(s: dict):
    k = s["kind"]
    if k == "slots":
        return {n: s[n] for n in ("table", "pool", "lens_out", "state_out", "row_start", "slots", "pos", "kv_len")}
    if k == "append":
        t = torch.int8 if s["fmt"] == "int8" else torch.float8_e4m3fn
        return {"k": s["k"].view(t), "v": s["v"].view(t), "ks": s["ks"], "vs": s["vs"]}
    return s["o"] if k == "attn" else s["out"]


def run(s: dict):
    if own:
        rc = s["fn"](*s["args"])
        if rc:
            raise RuntimeError(f"the call returned {rc}")
    else:
        {"slots": _plain_slots, "append": _plain_append, "attn": _plain_attn, "w4": _plain_w4}[s["kind"]](s)
    return _outputs(s)


# ---- plain forms ------------------------------------------------------------------------------------------------
def _plain_slots(s: dict) -> None:
    c = s["case"]
    bs, pages, ld, rows = c["bs"], c["pages"], c["ld"], s["rows"]
    dev, i64 = s["lens"].device, torch.int64
    lens, add, table, pool = s["lens"].to(i64), s["add"].to(i64), s["table"], s["pool"]
    head, count = s["state"][0].to(i64), s["state"][1].to(i64)
    n = add.clamp_min(0)
    end = n.cumsum(0)
    start = torch.cat([torch.zeros(1, dtype=i64, device=dev), end])
    have, want = (lens + bs - 1) // bs, (lens + n + bs - 1) // bs
    ok = (add >= 0) & (lens + n <= ld * bs) & (end <= rows)
    need = torch.where(ok, want - have, 0)
    upto = need.cumsum(0)
    ok &= (need == 0) | (upto <= count)
    back = torch.where(add < 0, have, 0)
    back_upto = back.cumsum(0)
    j = torch.arange(ld, device=dev)[None, :]
    # ended requests' pages behind the ring's last one, then the new pages from its head: the two ranges do not meet
    at = (head + count + (back_upto - back)[:, None] + j) % pages
    gone = j < back[:, None]
    pool[at[gone]] = table[gone]
    at = (head + (upto - need)[:, None] + j - have[:, None]) % pages
    fresh = ok[:, None] & (j >= have[:, None]) & (j < want[:, None])
    table.copy_(torch.where(fresh, pool[at], table))
    used = torch.where(ok & (need > 0), upto, 0).max()
    r = torch.arange(rows, device=dev)
    b = torch.searchsorted(end, r, right=True).clamp_max(len(lens) - 1)
    p = lens[b] + r - start[b]
    inside = ok[b] & (r < end[-1])
    page = table[b, (p // bs).clamp_max(ld - 1)].to(i64)
    s["slots"].copy_(torch.where(inside, page * bs + p % bs, -1))
    s["pos"].copy_(torch.where(inside, p, -1))
    s["row_start"].copy_(start)
    s["kv_len"].copy_(torch.where(ok, lens + n, 0))
    s["lens_out"].copy_(torch.where(ok, lens + n, torch.where(add < 0, 0, lens)))
    s["state_out"].copy_(torch.stack([(head + used) % pages, count - used + back_upto[-1], ((add >= 0) & ~ok).sum()]))


def _plain_append(s: dict) -> None:
    bs, hkv, dh, fmt = s["bs"], s["hkv"], s["dh"], s["fmt"]
    n = hkv * dh
    slot = s["slots"].to(torch.int64)
    page, off = slot // bs, slot % bs
    lead = torch.ones_like(page, dtype=torch.bool)
    lead[1:] = page[1:] != page[:-1]
    run_of = lead.cumsum(0) - 1
    rp, old = page[lead], off[lead]
    t = torch.arange(bs, device=slot.device)
    for codes, scales, x, key in ((s["k"], s["ks"], s["kv"][:, :n], True), (s["v"], s["vs"], s["kv"][:, n:], False)):
        x = torch.nan_to_num(x.float(), nan=0.0, posinf=65504.0, neginf=-65504.0).view(-1, hkv, dh)
        top = torch.zeros(len(rp), hkv, device=x.device).scatter_reduce(0, run_of[:, None].expand(-1, hkv), x.abs().amax(2), "amax")
        was = torch.where(old[:, None] > 0, scales[rp], 0.0)
        sc = torch.maximum(was, _pow2_scale(top, fmt))
        scales[rp] = sc
        held = codes[rp]
        again = _to_codes(_from_codes(held, fmt) * (was / sc)[:, :, None, None], fmt)
        before = t[None, :] < old[:, None]
        before = before[:, None, :, None] if key else before[:, None, None, :]
        codes[rp] = torch.where(before & ((was != sc)[:, :, None, None]), again, held)
        new = _to_codes(x / sc[run_of][:, :, None], fmt)
        if key:
            codes[page, :, off] = new
        else:
            codes[page, :, :, off] = new


def _plain_attn(s: dict) -> None:
    H, hkv, dh, bs, fmt, window = s["H"], s["hkv"], s["dh"], s["bs"], s["fmt"], s["window"]
    grp, r0 = H // hkv, 0
    for b, (L, n) in enumerate(zip(s["L"], s["new"])):
        lo = max(0, L - n + 1 - window) // bs if window else 0
        tb = s["table"][b, lo:-(-L // bs)].to(torch.int64)
        k = _from_codes(s["k"][tb], fmt) * s["ks"][tb][:, :, None, None]
        v = _from_codes(s["v"][tb], fmt) * s["vs"][tb][:, :, None, None]
        k = k.permute(1, 0, 2, 3).reshape(hkv, -1, dh)[:, : L - lo * bs]
        v = v.permute(1, 0, 3, 2).reshape(hkv, -1, dh)[:, : L - lo * bs]
        q = s["q"][r0:r0 + n].float().view(n, hkv, grp, dh).permute(1, 2, 0, 3).reshape(hkv, grp * n, dh)
        z = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
        j = torch.arange(lo * bs, L, device=z.device)
        if n > 1 or window:
            at = torch.arange(L - n, L, device=z.device)[:, None]
            no = j[None, :] > at
            if window:
                no |= j[None, :] <= at - window
            z.view(hkv, grp, n, -1).masked_fill_(no, -math.inf)
        p = torch.exp(z - z.amax(2, keepdim=True))
        o = torch.matmul(p, v) / p.sum(2, keepdim=True)
        s["o"][r0:r0 + n] = o.view(hkv, grp, n, dh).permute(2, 0, 1, 3).reshape(n, H * dh).to(torch.float16)
        r0 += n


def _plain_w4(s: dict) -> None:
    K, N, g = s["K"], s["N"], s["group"]
    sh = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)[None, :, None]
    c = ((s["w"].view(K // 8, 1, N) >> sh) & 15).view(K, N).float()
    of = torch.arange(K, device="cuda") // g
    w = (c - (8.0 if s["zp"] is None else s["zp"].float()[of])) * s["s"].float()[of]
    z = s["x"].float() @ w
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if s["residual"] is not None:       # the epilogue's residual is added to the rounded sum
        z = z.to(torch.float16).float() + s["residual"].float()
    s["out"].copy_(z)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _value64(codes, fmt: str):
    """The number each 8-bit code stands for: two's complement, or sign, 4 bits of exponent (bias 7), 3 of fraction."""
    c = codes.to(torch.int64)
    if fmt == "int8":
        return torch.where(c > 127, c - 256, c).double()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (8 + m) * _two_to(e - 10), m * 2.0 ** -9)
    return torch.where(c > 127, -v, v)


def _round64(x, fmt: str):
    """The nearest value of the format, ties to the even code."""
    if fmt == "int8":
        return x.round().clamp(-127, 127)
    step = _two_to(torch.frexp(x.abs().clamp_min(2.0 ** -6)).exponent - 4)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_append(s: dict):
    bs, hkv, dh, fmt = s["bs"], s["hkv"], s["dh"], s["fmt"]
    most, n, at = QMAX[fmt], hkv * dh, s["slots"].tolist()
    out = {"k": _value64(s["k"], fmt), "v": _value64(s["v"], fmt).transpose(2, 3), "ks": s["ks"].double(), "vs": s["vs"].double()}
    x = s["kv"].double().view(-1, 2, hkv, dh)
    i = 0
    while i < len(at):
        e = i + 1
        while e < len(at) and at[e] // bs == at[i] // bs:
            e += 1
        page, off = at[i] // bs, at[i] % bs
        for c, (codes, scales) in enumerate((("k", "ks"), ("v", "vs"))):
            rows = x[i:e, c].transpose(0, 1)                                       # [hkv, tokens, dh]
            f, p = torch.frexp((rows.abs().amax((1, 2)) / most).clamp_min(2.0 ** -32))
            sc = _two_to(torch.where(f == 0.5, p - 1, p))
            if off:
                was = out[scales][page].clone()
                sc = torch.maximum(sc, was)
                out[codes][page, :, :off] = _round64(out[codes][page, :, :off] * (was / sc)[:, None, None], fmt)
            out[scales][page] = sc
            out[codes][page, :, off:off + e - i] = _round64(rows / sc[:, None, None], fmt)
        i = e
    out["v"] = out["v"].transpose(2, 3).contiguous()
    return out


def _exact_attn(s: dict):
    grp, dh, bs = s["H"] // s["hkv"], s["dh"], s["bs"]
    out, r0 = torch.empty(s["rows"], s["H"], dh, dtype=torch.float64, device="cuda"), 0
    for b, (L, n) in enumerate(zip(s["L"], s["new"])):
        t = torch.arange(L, device="cuda")
        page, off = s["table"][b, t // bs].long(), t % bs
        see = t[None, :] <= (L - n + torch.arange(n, device="cuda"))[:, None]
        if s["window"]:
            see &= t[None, :] > (L - n + torch.arange(n, device="cuda") - s["window"])[:, None]
        for h in range(s["hkv"]):
            k = _value64(s["k"][page, h, off], s["fmt"]) * s["ks"][page, h].double()[:, None]
            v = _value64(s["v"][page, h, :, off], s["fmt"]) * s["vs"][page, h].double()[:, None]
            for g in range(h * grp, h * grp + grp):
                w = s["q"][r0:r0 + n, g * dh:g * dh + dh].double() @ k.T * s["scale"]
                out[r0:r0 + n, g] = torch.softmax(torch.where(see, w, -math.inf), 1) @ v
        r0 += n
    return out.view(s["rows"], -1)


def _exact_w4(s: dict):
    out = torch.zeros(s["M"], s["N"], dtype=torch.float64, device="cuda")
    for k0 in range(0, s["K"], s["group"]):
        k1, gi = min(s["K"], k0 + s["group"]), k0 // s["group"]
        c = torch.stack([(s["w"][k // 8].long() >> (4 * (k % 8))) & 15 for k in range(k0, k1)]).double()
        c -= 8.0 if s["zp"] is None else s["zp"][gi].double()
        out += (s["x"][:, k0:k1].double() @ c) * s["s"][gi].double()
    if s["bias"] is not None:
        out += s["bias"].double()
    return out if s["residual"] is None else out + s["residual"].double()


def exact(case: dict, seed: int):
    k = case["kind"]
    if k == "slots" or (k == "attn" and work(case)["flops"] > 1e12):
        return None                                     # whole numbers throughout; too long in 64 bits
    s = _state(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "w4": _exact_w4}[k](s)
