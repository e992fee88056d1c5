"""More operators of a decoder's step, as they are measured: rotary positions, by themselves and on the way into the 8-bit
cache, and products whose operands are both microscaled 4-bit floating point.

A case is a dict of plain values. `prepare` makes what a serving program holds before the call; `run` is one pass, through
the library's entry points where `own` is true and in elementary torch operations (fp32, angles in 64 bits, rounded once at the
end) where it is false; `exact` computes the same outputs in 64 bits, written apart from both; `work` is what a pass cannot do without.

  rope    sh_rope_pos: the query and key heads of a projection's rows turned by the rows' positions, whole heads or their first
          columns, two column layouts, frequencies as they are or stretched for long contexts; rows at position -1 are left
  append  sh_kv_append_rope: the same for a step's queries, while its keys are turned on their way into the 8-bit paged cache
          beside the values (rounded to fp16, then to codes with one power-of-two scale for each page and head)
  quant   sh_mx4_quant: rows in e2m1 codes with a power-of-two scale for every 32 columns
  mx4     sh_gemm_mx4: z = x . W + bias [GELU] [+ residual] of two operands in that format, and sh_gemm_mx4_f16, which
          takes few fp16 rows and brings them into it on the way

Every pass leaves its state so that the next one computes the same outputs: the turned rows go to a buffer of their own, and
appending the same rows at the same slots twice stores the same codes. The cache is e4m3 here: a code of it is compared as the value it
stands for. (Of int8 codes, whole numbers, one in some thousand millions lies so near a border that the last bit of an angle decides.)
"""
from __future__ import annotations

import math
import random

import torch

own = False

HALF, PAIRS = 0, 1                      # column i with i + rot / 2; column 2 i with 2 i + 1


# ---- the cases --------------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one decode step of 64 slots, four of them idle, anywhere in a stretched context of 128 thousand
        dict(name="rope_decode_b64", kind="rope", rows=64, idle=4, requests=60, H=32, hkv=8, dh=128, rot=128, layout=HALF, base=5e5,
             scaling="bands", factor=8.0, ctx=8192, far=131072),
        # a chunk of prompts, half of each head turned, neighbouring columns: the bytes of the rows
        dict(name="rope_prompts_partial", kind="rope", rows=16001, idle=1, requests=9, H=32, hkv=8, dh=128, rot=64, layout=PAIRS, base=1e4,
             scaling="none", factor=1.0, ctx=8192, far=8192),
        # one user's decode step with the heads of the vision-language decoder: latency
        dict(name="append_b1", kind="append", B=1, idle=0, bs=16, H=15, hkv=5, dh=64, rot=64, layout=HALF, base=1e5, scaling="none",
             factor=1.0, ctx=8192, far=8192, pages=64, longest=1, shape=1),
        # the step's rows of 64 requests in a batch of 80 slots, long stretched contexts
        dict(name="append_decode_b64", kind="append", B=64, idle=16, bs=16, H=32, hkv=8, dh=128, rot=128, layout=HALF, base=5e5,
             scaling="bands", factor=8.0, ctx=8192, far=131072, pages=2048, longest=1, shape=2),
        # the first chunk of a few prompts, pages of 32 tokens that the prompts do not fill, half of each head turned
        dict(name="append_prompts", kind="append", B=9, idle=0, bs=32, H=32, hkv=8, dh=128, rot=64, layout=PAIRS, base=1e4, scaling="ramp",
             factor=4.0, ctx=4096, far=16384, pages=1200, longest=4096, shape=3),
        # the rows of a small batch on their way into a product
        dict(name="quant_rows50", kind="quant", rows=50, cols=4096, ldx=4096),
        # a prompt chunk's widest activations: HBM
        dict(name="quant_prompts", kind="quant", rows=8192, cols=14336, ldx=14336),
        # the expert's gated MLP product for a single token: latency, a last block of 16
        dict(name="mx4_m1_expert", kind="mx4", f16=True, M=1, N=2048, K=720, bias=False, gelu=False, residual=False),
        # the widest product of a larger decoder for a single token: the bytes of the weight
        dict(name="mx4_m1_wide", kind="mx4", f16=True, M=1, N=14336, K=4096, bias=False, gelu=False, residual=False),
        # a batch of 50 rows, with bias and residual
        dict(name="mx4_m50_residual", kind="mx4", f16=False, M=50, N=4096, K=8192, bias=True, gelu=False, residual=True),
        # a ragged chunk of prompts through an MLP's first product
        dict(name="mx4_m700_gelu", kind="mx4", f16=False, M=700, N=5000, K=2880, bias=True, gelu=True, residual=False),
        # a full batch of prompt rows: the compute-bound end
        dict(name="mx4_m8192", kind="mx4", f16=False, M=8192, N=8192, K=8192, bias=False, gelu=False, residual=False),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case: dict) -> float:
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 2e15)


def _positions(rng) -> dict:
    scaling = rng.choice(["none", "linear", "bands", "ramp"])
    ctx = rng.choice([2048, 4096, 8192])
    factor = 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0])
    return dict(layout=rng.choice([HALF, PAIRS]), base=rng.choice([1e4, 1e5, 5e5, 1e6]), scaling=scaling, factor=factor, ctx=ctx, far=int(ctx * factor))


def _draw(rng) -> dict:
    kind = rng.choice(["rope", "rope", "append", "append", "append", "quant", "quant", "mx4", "mx4", "mx4", "mx4"])
    if kind == "rope":
        dh = rng.choice([32, 64, 72, 80, 96, 128, 128, 256])
        rows = _log(rng, 1, 16384)
        return dict(kind=kind, rows=rows, idle=rng.choice([0, 0, rows // 5]), requests=rng.choice([rows, min(rows, 9)]),
                    H=rng.choice([1, 4, 8, 15, 16, 32, 64]), hkv=rng.choice([1, 2, 5, 8]), dh=dh,
                    rot=rng.choice([dh, dh, dh // 2, dh // 4, 2 * rng.randint(1, dh // 2)]) & ~1, **_positions(rng))
    if kind == "append":
        bs, hkv, dh, longest = rng.choice([16, 32, 64]), rng.choice([1, 2, 4, 5, 8]), rng.choice([32, 64, 80, 96, 128, 256]), \
            rng.choice([1, 1, 4, _log(rng, 2, 4096)])
        B = _log(rng, 1, 256) if longest <= 4 else _log(rng, 1, 9)
        return dict(kind=kind, B=B, idle=rng.choice([0, 0, B // 4]), bs=bs, H=hkv * rng.choice([1, 2, 3, 4, 8]), hkv=hkv, dh=dh,
                    rot=rng.choice([dh, dh, dh // 2 // 8 * 8, 8 * rng.randint(1, dh // 8)]), pages=B * (longest // bs + 3) + 5, longest=longest,
                    shape=rng.randrange(1 << 30), **_positions(rng))
    if kind == "quant":
        cols = rng.choice([_log(rng, 1, 16384), 32 * _log(rng, 1, 512)])
        return dict(kind=kind, rows=_log(rng, 1, 8192), cols=cols, ldx=cols + rng.choice([0, 0, 1, 8, cols]))
    M = rng.choice([1, _log(rng, 1, 16), _log(rng, 2, 64), _log(rng, 64, 8192), _log(rng, 64, 8192)])
    return dict(kind=kind, f16=M <= 16 and rng.random() < 0.5, M=M, N=_log(rng, 16, 16384), K=rng.choice([_log(rng, 16, 16384), 32 * _log(rng, 1, 512)]),
                bias=rng.random() < 0.5, gelu=rng.random() < 0.3, residual=rng.random() < 0.5)


def draw(rng) -> dict:
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    while True:
        c = _draw(rng)
        if c.get("rot", 2) >= 2 and _cost(c) <= most[c["kind"]]:
            return c


# ---- lengths: a case has its own, another seed has them in another order -----------------------------------------
def _append_lengths(case: dict) -> tuple[list[int], list[int]]:
    """(tokens held in the first page written, tokens added) of each request."""
    rng, B = random.Random(case["shape"]), case["B"]
    lo = max(1, case["longest"] // 8)
    add = [_log(rng, lo, case["longest"]) for _ in range(B)]
    add[rng.randrange(B)] = case["longest"]
    return [rng.randrange(case["bs"]) if a <= 4 or rng.random() < 0.3 else 0 for a in add], add


def work(case: dict) -> dict:
    k = case["kind"]
    if k == "rope":
        n = case["rows"] - case["idle"]
        heads = case["H"] + case["hkv"]
        return {"bytes": n * (heads * case["dh"] * 4 + 4) + case["rot"] * 4, "flops": n * heads * case["rot"] * 3}
    if k == "append":
        held, add = _append_lengths(case)
        n, wide = sum(add), case["hkv"] * case["dh"]
        runs = sum((h + a - 1) // case["bs"] + 1 for h, a in zip(held, add))
        b = n * (wide * 2 * 3 + case["H"] * case["dh"] * 4) + runs * case["hkv"] * 8 + n * 8 + case["rot"] * 4
        return {"bytes": b, "flops": n * (wide * 2 * 3 + (case["H"] + case["hkv"]) * case["rot"] * 3)}
    if k == "quant":
        n = case["rows"] * case["cols"]
        blocks = case["rows"] * -(-case["cols"] // 32)
        return {"bytes": n * 2 + blocks * 17, "flops": n * 3}
    M, N, K = case["M"], case["N"], case["K"]
    nb = -(-K // 32)
    b = N * nb * 17 + (M * K * 2 if case["f16"] else M * nb * 17) + M * N * 2 + N * 2 * case["bias"] + M * N * 2 * case["residual"]
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


def _frequencies(case: dict) -> tuple[list[float], float]:
    """Radians a position turns each pair by, and what cosine and sine are multiplied by.
    linear: all slower by the factor. bands: by how often a pair turns within the first context: often (4 times and more) as it
    is, seldom (once and less) slower by the factor, linear between. ramp: the same by the pair's index, from that of 32 turns to that of one,
    with cosine and sine a little larger."""
    rot, base, f, ctx = case["rot"], case["base"], case["factor"], case["ctx"]
    w = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    kind = case["scaling"]
    if kind == "linear":
        w = [x / f for x in w]
    elif kind == "bands":
        keep = [min(1.0, max(0.0, (x * ctx / (2 * math.pi) - 1.0) / 3.0)) for x in w]
        w = [x * (k + (1 - k) / f) for x, k in zip(w, keep)]
    elif kind == "ramp":
        at = lambda turns: rot * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(0, math.floor(at(32.0))), min(rot - 1, math.ceil(at(1.0)))
        keep = [1.0 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(rot // 2)]
        w = [x * (k + (1 - k) / f) for x, k in zip(w, keep)]
    return w, 0.1 * math.log(f) + 1.0 if kind == "ramp" else 1.0


def _angles(case: dict, d: dict) -> None:
    """The frequencies, and the plan that a program keeps of them: turns per position as 64-bit fractions."""
    w, d["mscale"] = _frequencies(case)
    d["freq"] = torch.tensor(w, dtype=torch.float64, device="cuda")
    d["step"] = torch.tensor([int(x / (2 * math.pi) * 2.0 ** 64) for x in w], dtype=torch.int64, device="cuda")
    d["rot"], d["layout"] = case["rot"], case["layout"]


def _channels(r: _Rand, heads: int, dh: int):
    """A few channels of a query or key are larger than the others by an order of magnitude."""
    c = torch.ones(heads, dh, device="cuda")
    c[torch.rand(heads, dh, generator=r.g, device="cuda") < 0.03] = 8.0
    return c


def _rope_state(case: dict, r: _Rand) -> dict:
    H, hkv, dh, rows = case["H"], case["hkv"], case["dh"], case["rows"]
    heads, wide = H + hkv, (H + 2 * hkv) * dh
    x = r.normal(rows, wide)
    x[:, : heads * dh] *= _channels(r, heads, dh).view(1, -1)
    live = rows - case["idle"]
    n = max(1, min(live, case["requests"]))
    cut = sorted(r.host.sample(range(1, live), n - 1)) if 1 < n < live else list(range(1, n))
    pos = []
    for a, b in zip([0] + cut, cut + [live]):
        first = r.host.randrange(max(1, case["far"] - (b - a)))
        pos += range(first, first + b - a)
    d = dict(x=x.to(torch.float16), y=torch.zeros(rows, heads * dh, dtype=torch.float16, device="cuda"), pos=_i32(pos + [-1] * case["idle"]),
             rows=rows, heads=heads, dh=dh, wide=wide)
    _angles(case, d)
    return d


def _append_state(case: dict, r: _Rand) -> dict:
    held, add = _append_lengths(case)
    order = list(range(case["B"]))
    r.host.shuffle(order)
    bs, H, hkv, dh, pages = (case[n] for n in ("bs", "H", "hkv", "dh", "pages"))
    perm = r.order(pages).tolist()
    slots, pos, n = [], [], 0
    for i in order:
        first = n
        n += (held[i] + add[i] - 1) // bs + 1
        slots += [perm[first + p // bs] * bs + p % bs for p in range(held[i], held[i] + add[i])]
        p0 = held[i] + bs * r.host.randrange(max(1, (case["far"] - held[i] - add[i]) // bs))
        pos += range(p0, p0 + add[i])
    slots, pos = slots + [-1] * case["idle"], pos + [-1] * case["idle"]
    rows = len(slots)
    k, v = (r.codes(pages, hkv, *s, high=120) for s in ((bs, dh), (dh, bs)))
    ks, vs = (torch.exp2(torch.randint(-9, -5, (pages, hkv), generator=r.g, device="cuda").float()) for _ in "kv")
    x = r.normal(rows, H + hkv, dh) * _channels(r, H + hkv, dh)
    y = r.normal(rows, hkv * dh, std=0.5)
    qkv = torch.cat([x.reshape(rows, -1), y], 1).to(torch.float16)                 # the q | k | v columns of one projection
    d = dict(k=k, v=v, ks=ks, vs=vs, qkv=qkv, q=torch.zeros(rows, H * dh, dtype=torch.float16, device="cuda"), slots=_i32(slots), pos=_i32(pos),
             rows=rows, H=H, hkv=hkv, dh=dh, bs=bs, pages=pages)
    _angles(case, d)
    return d


def _quant_state(case: dict, r: _Rand) -> dict:
    rows, cols, ldx = case["rows"], case["cols"], case["ldx"]
    nb = -(-cols // 32)
    x = torch.empty(rows, ldx, dtype=torch.float16, device="cuda")
    step = max(1, (1 << 26) // ldx)
    for i in range(0, rows, step):                   # activations: rows of different size, a few large columns
        t = r.normal(min(step, rows - i), ldx)
        x[i:i + step] = t * torch.exp2(r.normal(t.shape[0], 1)) * (1 + 7 * (torch.rand(1, ldx, generator=r.g, device="cuda") < 0.02))
    return dict(x=x, codes=torch.zeros(rows, 16 * nb, dtype=torch.uint8, device="cuda"),
                scales=torch.zeros(rows, -(-nb // 4) * 4, dtype=torch.uint8, device="cuda"), rows=rows, cols=cols, ldx=ldx)


def _mx4_operand(r: _Rand, rows: int, K: int, spread: int) -> tuple:
    """Codes of a rounded bell (zeros behind K) and scales about the size that makes products of unit size."""
    nb = -(-K // 32)
    codes = torch.empty(rows, 16 * nb, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (16 * nb))
    for i in range(0, rows, step):
        n = min(step, rows - i)
        a = r.normal(n, 32 * nb, std=2.0)
        c = (_e2m1(a.abs()) | ((a < 0).to(torch.uint8) << 3))
        c[:, K:] = 0
        codes[i:i + n] = c[:, 0::2] | (c[:, 1::2] << 4)
    scales = torch.full((rows, -(-nb // 4) * 4), 127, dtype=torch.uint8, device="cuda")
    scales[:, :nb] = 127 - 1 - spread + r.codes(rows, nb, high=spread + 1)
    return codes, scales


def _mx4_state(case: dict, r: _Rand) -> dict:
    M, N, K = case["M"], case["N"], case["K"]
    d = dict(M=M, N=N, K=K, nb=-(-K // 32), z=torch.empty(M, N, dtype=torch.float16, device="cuda"), gelu=case["gelu"], bias=None, residual=None)
    if case["f16"]:
        d["x"] = r.normal(M, K).mul_(torch.exp2(r.normal(M, 1) * 0.5)).to(torch.float16)
    else:
        d["xc"], d["xs"] = _mx4_operand(r, M, K, 3)
    d["wc"], d["ws"] = _mx4_operand(r, N, K, 1)
    shift = round(math.log2(K) / 2)
    d["ws"][:, : d["nb"]] -= shift                   # weights of about 1 / sqrt(K)
    if case["bias"]:
        d["bias"] = r.normal(N, std=0.1).to(torch.float16)
    if case["residual"]:
        d["residual"] = r.normal(M, N).to(torch.float16)
    return d


def _state(case: dict, seed: int) -> dict:
    s = {"rope": _rope_state, "append": _append_state, "quant": _quant_state, "mx4": _mx4_state}[case["kind"]](case, _Rand(seed))
    s["kind"] = case["kind"]
    return s


def prepare(case: dict, seed: int) -> dict:
    return _state(case, seed)


# ---- the library's entry points ------------------------------------------------------------------------------------
def _bind(s: dict) -> tuple:
    """The entry point and its arguments, converted once as a program does for buffers that it keeps."""
    import ctypes

    from softhier_mlir_amd import shops
    lib, A, k = shops.load(), shops.addr, s["kind"]
    lib.sh_init()
    if k in ("rope", "append"):
        s["plan"] = shops.rope_plan(A(s["step"]), s["rot"], s["layout"], s["mscale"])
        p = ctypes.byref(s["plan"])
    if k == "rope":
        return lib.sh_rope_pos, (A(s["y"]), A(s["x"]), A(s["pos"]), p, s["rows"], s["heads"], s["dh"], s["heads"] * s["dh"], s["wide"])
    if k == "append":
        nq, nk = s["H"] * s["dh"], s["hkv"] * s["dh"]
        s["cache"] = shops.kv_cache(A(s["k"]), A(s["v"]), A(s["ks"]), A(s["vs"]), s["pages"], s["hkv"], s["dh"], s["bs"], shops.SH_FP8)
        x, wide = s["qkv"], nq + 2 * nk
        return lib.sh_kv_append_rope, (ctypes.byref(s["cache"]), p, A(s["q"]), A(x), A(x, nq), A(x, nq + nk), A(s["pos"]), A(s["slots"]), s["rows"],
                                       s["H"], nq, wide, wide, wide)
    if k == "quant":
        return lib.sh_mx4_quant, (A(s["codes"]), A(s["scales"]), A(s["x"]), s["rows"], s["cols"], s["codes"].shape[1], s["scales"].shape[1], s["ldx"])
    M, N, K = s["M"], s["N"], s["K"]
    b, r = s["bias"], s["residual"]
    s["epi"] = shops.epi(bias=A(b) if b is not None else 0, act=shops.SH_ACT_GELU if s["gelu"] else shops.SH_ACT_NONE,
                         residual=A(r) if r is not None else 0, ldr=N if r is not None else 0)
    w = (A(s["wc"]), A(s["ws"]), A(s["z"]), M, N, K)
    ldw = (s["wc"].shape[1], s["ws"].shape[1], N, ctypes.byref(s["epi"]))
    if "x" in s:
        return lib.sh_gemm_mx4_f16, (A(s["x"]), *w, K, *ldw)
    return lib.sh_gemm_mx4, (A(s["xc"]), A(s["xs"]), *w, s["xc"].shape[1], s["xs"].shape[1], *ldw)


def _outputs(s: dict):
    k = s["kind"]
    if k == "rope":
        return s["y"]
    if k == "append":
        return {"q": s["q"], "k": s["k"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn), "ks": s["ks"], "vs": s["vs"]}
    if k == "quant":
        return {"codes": s["codes"], "scales": s["scales"][:, : -(-s["cols"] // 32)]}
    return s["z"]


def run(s: dict):
    if own:
        fn, args = s.get("call") or s.setdefault("call", _bind(s))
        rc = fn(*args)
        if rc:
            raise RuntimeError(f"the call returned {rc}")
    else:
        {"rope": _plain_rope, "append": _plain_append, "quant": _plain_quant, "mx4": _plain_mx4}[s["kind"]](s)
    return _outputs(s)


# ---- plain forms ------------------------------------------------------------------------------------------------
def _turned(x, s: dict):
    """x [rows, heads, dh] in fp32 with the first `rot` columns turned by the rows' positions, rounded to fp16."""
    rot, h = s["rot"], s["rot"] // 2
    a = s["pos"].double()[:, None] * s["freq"][None, :]
    c, n = ((t * s["mscale"]).float()[:, None, :] for t in (torch.cos(a), torch.sin(a)))
    x1, x2 = (x[..., :h], x[..., h:rot]) if s["layout"] == HALF else (x[..., 0:rot:2], x[..., 1:rot:2])
    y1, y2 = x1 * c - x2 * n, x2 * c + x1 * n
    y = torch.cat([y1, y2], -1) if s["layout"] == HALF else torch.stack([y1, y2], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1).to(torch.float16)


def _plain_rope(s: dict) -> None:
    n = s["heads"] * s["dh"]
    y = _turned(s["x"][:, :n].float().view(-1, s["heads"], s["dh"]), s).view(-1, n)
    s["y"].copy_(torch.where(s["pos"][:, None] >= 0, y, s["y"]))


def _pow2_scale(amax):
    """The smallest power of two s >= 2^-32 with amax <= 448 s."""
    f, e = torch.frexp(amax.clamp_min(2.0 ** -60))
    return ((torch.where(f <= 0.875, e - 9, e - 8).clamp_min(-32) + 127) << 23).view(torch.float32)


def _to_codes(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_append(s: dict) -> None:
    bs, H, hkv, dh = s["bs"], s["H"], s["hkv"], s["dh"]
    nq, nk = H * dh, hkv * dh
    x = _turned(s["qkv"][:, : nq + nk].float().view(-1, H + hkv, dh), s)
    s["q"].copy_(torch.where(s["pos"][:, None] >= 0, x[:, :H].reshape(-1, nq), s["q"]))
    slot = s["slots"].to(torch.int64)
    live = slot >= 0
    key, val = x[:, H:].float()[live], s["qkv"][:, nq + nk:].float().view(-1, hkv, dh)[live]
    slot = slot[live]
    page, off = slot // bs, slot % bs
    lead = torch.ones_like(page, dtype=torch.bool)
    lead[1:] = page[1:] != page[:-1]
    run_of = lead.cumsum(0) - 1
    rp, old = page[lead], off[lead]
    t = torch.arange(bs, device=slot.device)
    for codes, scales, x, is_key in ((s["k"], s["ks"], key, True), (s["v"], s["vs"], val, False)):
        top = torch.zeros(len(rp), hkv, device=x.device).scatter_reduce(0, run_of[:, None].expand(-1, hkv), x.abs().amax(2), "amax")
        was = torch.where(old[:, None] > 0, scales[rp], 0.0)
        sc = torch.maximum(was, _pow2_scale(top))
        scales[rp] = sc
        held = codes[rp]
        again = _to_codes(held.view(torch.float8_e4m3fn).float() * (was / sc)[:, :, None, None])
        before = t[None, :] < old[:, None]
        before = before[:, None, :, None] if is_key else before[:, None, None, :]
        codes[rp] = torch.where(before & ((was != sc)[:, :, None, None]), again, held)
        new = _to_codes(x / sc[run_of][:, :, None])
        if is_key:
            codes[page, :, off] = new
        else:
            codes[page, :, :, off] = new


def _e2m1(a):
    """Codes of values >= 0 (0, 0.5, 1, 1.5, 2, 3, 4, 6), nearest, ties to the even code."""
    c = (a > 0.25).to(torch.uint8)
    for border, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= border) if up else (a > border)
    return c


def _mx4_codes(x, cols: int) -> tuple:
    """(packed codes, scale bytes) of fp32 rows: the smallest power of two s >= 2^-32 with |x| <= 6 s for 32 columns; 255 and
    codes of 0 where one of them is not finite."""
    rows, nb = x.shape[0], -(-cols // 32)
    x = torch.nn.functional.pad(x[:, :cols], (0, 32 * nb - cols)).view(rows, nb, 32)
    top = x.abs().amax(2)
    fine = torch.isfinite(top)
    f, e = torch.frexp(torch.where(fine, top, 0.0).clamp_min(2.0 ** -60))
    e = torch.where(f <= 0.75, e - 3, e - 2).clamp_min(-32)
    x = x / ((e + 127) << 23).view(torch.float32)[:, :, None]
    c = _e2m1(x.abs()) | (torch.signbit(x).to(torch.uint8) << 3)
    c = torch.where(fine[:, :, None], c, 0).view(rows, -1)
    return c[:, 0::2] | (c[:, 1::2] << 4), torch.where(fine, e + 127, 255).to(torch.uint8)


def _plain_quant(s: dict) -> None:
    c, b = _mx4_codes(s["x"].float(), s["cols"])
    s["codes"].copy_(c)
    s["scales"][:, : b.shape[1]] = b


def _mx4_values(codes, scales, nb: int):
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    v = torch.cat([v, -v])
    x = torch.stack([v[(codes & 15).int()], v[(codes >> 4).int()]], -1).view(-1, nb, 32)
    b = scales[:, :nb].int()
    return (x * torch.where(b < 255, torch.exp2((b - 127).float()), math.nan)[:, :, None]).view(-1, nb * 32)


def _plain_mx4(s: dict) -> None:
    nb = s["nb"]
    xc, xs = _mx4_codes(s["x"].float(), s["K"]) if "x" in s else (s["xc"], s["xs"])
    z = _mx4_values(xc, xs, nb) @ _mx4_values(s["wc"], s["ws"], nb).T
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if s["gelu"]:
        z = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if s["residual"] is not None:       # the epilogue's residual is added to the rounded sum
        z = z.to(torch.float16).float() + s["residual"].float()
    s["z"].copy_(z)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_turn(x, s: dict):
    """Each pair as a complex number times m e^{i pos w}."""
    rot, x = s["rot"], x.double()
    w = torch.polar(torch.full_like(s["freq"], s["mscale"]).expand(len(s["pos"]), -1).contiguous(), s["pos"].double()[:, None] * s["freq"])
    out = x.clone()
    at = torch.arange(rot // 2, device=x.device)
    i, j = (at, at + rot // 2) if s["layout"] == HALF else (2 * at, 2 * at + 1)
    z = torch.complex(x[:, :, i], x[:, :, j]) * w[:, None, :]
    out[:, :, i], out[:, :, j] = z.real, z.imag
    return out


def _exact_rope(s: dict):
    n, live = s["heads"] * s["dh"], s["pos"] >= 0
    out = torch.zeros(s["rows"], n, dtype=torch.float64, device="cuda")
    out[live] = _exact_turn(s["x"][:, :n].reshape(-1, s["heads"], s["dh"]), s).view(-1, n)[live]
    return out


def _value64(codes):
    """The number an e4m3 code stands for: sign, 4 bits of exponent (bias 7), 3 of fraction."""
    c = codes.to(torch.int64)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (8 + m) * _two_to(e - 10), m * 2.0 ** -9)
    return torch.where(c > 127, -v, v)


def _round64(x):
    """The nearest e4m3 value, ties to the even code."""
    step = _two_to(torch.frexp(x.abs().clamp_min(2.0 ** -6)).exponent - 4)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_append(s: dict):
    bs, H, hkv, dh, at = s["bs"], s["H"], s["hkv"], s["dh"], s["slots"].tolist()
    x = s["qkv"].double().view(-1, H + 2 * hkv, dh)
    turned = _exact_turn(x[:, : H + hkv], s)
    q = torch.zeros(s["rows"], H * dh, dtype=torch.float64, device="cuda")
    live = s["pos"] >= 0
    q[live] = turned[:, :H].reshape(-1, H * dh)[live]
    out = {"q": q, "k": _value64(s["k"]), "v": _value64(s["v"]).transpose(2, 3), "ks": s["ks"].double(), "vs": s["vs"].double()}
    new = {"k": turned[:, H:].to(torch.float16).double(), "v": x[:, H + hkv:]}      # the turned key is an fp16 row before it is codes
    i = 0
    while i < len(at) and at[i] >= 0:                    # a run of rows in one page after the other
        e = i + 1
        while e < len(at) and at[e] >= 0 and at[e] // bs == at[i] // bs:
            e += 1
        page, off = at[i] // bs, at[i] % bs
        for c in "kv":
            rows = new[c][i:e].transpose(0, 1)                                     # [hkv, tokens, dh]
            f, p = torch.frexp((rows.abs().amax((1, 2)) / 448.0).clamp_min(2.0 ** -32))
            sc = _two_to(torch.where(f == 0.5, p - 1, p))
            if off:
                was = out[c + "s"][page].clone()
                sc = torch.maximum(sc, was)
                out[c][page, :, :off] = _round64(out[c][page, :, :off] * (was / sc)[:, None, None])
            out[c + "s"][page] = sc
            out[c][page, :, off:off + e - i] = _round64(rows / sc[:, None, None])
        i = e
    out["v"] = out["v"].transpose(2, 3).contiguous()
    return out


def _fp4_value64(codes):
    """The number an e2m1 code stands for: sign, 2 bits of exponent (bias 1), 1 of fraction."""
    c = codes.to(torch.int64)
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e > 0, (2 + m) * _two_to(e - 2), m * 0.5)
    return torch.where(c > 7, -v, v)


def _exact_operand(codes, scales):
    x = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device="cuda")
    x[:, 0::2], x[:, 1::2] = _fp4_value64(codes & 15), _fp4_value64(codes >> 4)
    return x * _two_to(scales[:, : codes.shape[1] // 16].long() - 127).repeat_interleave(32, 1)


def _exact_rows(x):
    """fp16 rows as the values that their codes stand for: in each block a power of two t with max |x| <= 6 t, and the nearest of
    the format's values, found by its step (0.5 below 2, 1 below 4, 2 above) with ties to even."""
    out = torch.zeros(x.shape[0], -(-x.shape[1] // 32) * 32, dtype=torch.float64, device="cuda")
    out[:, : x.shape[1]] = x.double()
    v = out.view(x.shape[0], -1, 32)
    t = 2.0 ** torch.ceil(torch.log2((v.abs().amax(2) / 6).clamp_min(2.0 ** -32)))
    t = t.unsqueeze(2)
    u = v / t
    step = torch.where(u.abs() < 2, 0.5, torch.where(u.abs() < 4, 1.0, 2.0))
    return ((u / step).round() * step * t).view_as(out)


def _exact_mx4(s: dict):
    x = _exact_rows(s["x"]) if "x" in s else _exact_operand(s["xc"], s["xs"])
    z = x @ _exact_operand(s["wc"], s["ws"]).T.contiguous()
    if s["bias"] is not None:
        z += s["bias"].double()
    if s["gelu"]:
        z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z if s["residual"] is None else z + s["residual"].double()


def exact(case: dict, seed: int):
    k = case["kind"]
    if k == "quant":
        return None                                     # whole numbers throughout
    s = _state(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "mx4": _exact_mx4}[k](s)
