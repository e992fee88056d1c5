// Rotary positions of rows (sh_rope_pos) and the plan of their frequencies (sh_rope_steps). On the way into the 8-bit cache:
// sh_kv.hip.
#include "sh_rope.h"
#include <algorithm>
#include <cmath>

int sh_rope_check(const char *name, const sh_rope_plan *p, uint32_t dh, RopePlan *out) {
    if (!p || !p->step) { sh_set_error(-1, "[%s] NULL plan or step address", name); return -1; }
    if (p->step % 8) { sh_set_error(-1, "[%s] steps must be 8-byte aligned", name); return -1; }
    if (p->layout > SH_ROPE_PAIRS) { sh_set_error(-1, "[%s] unknown layout %u", name, p->layout); return -1; }
    if (p->rot < 2 || p->rot % 2 || p->rot > dh) { sh_set_error(-1, "[%s] %u turned columns of %u (even, 2 .. the head's width)", name, p->rot, dh); return -1; }
    if (!std::isfinite(p->mscale)) { sh_set_error(-1, "[%s] mscale is not finite", name); return -1; }
    *out = RopePlan{(const uint64_t *)p->step, p->rot, p->layout == SH_ROPE_PAIRS, (double)p->mscale};
    return 0;
}

namespace {

struct StepArgs { uint64_t *step; uint32_t pairs, scaling, ctx; double base, factor, lo, hi; };

// One thread a pair, in fp64; once for a model (3.4 us). w is off by (|ln w| + 8) 2^-53 of itself at most: its exponent's rounding, two steps of the power, three
// more operations; turns by 1.5e-16 at most, where w is 1.
__global__ void k_rope_steps(StepArgs a) {
    const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.pairs) return;
    const double two_pi = 6.283185307179586476925, rot = 2.0 * a.pairs;
    double w = pow(a.base, -2.0 * i / rot), keep = 1.0;                                 // keep: how much of the frequency stays
    if (a.scaling == SH_ROPE_LINEAR) keep = 0.0;
    else if (a.scaling == SH_ROPE_BANDS) keep = fmin(1.0, fmax(0.0, (w * a.ctx / two_pi - a.lo) / (a.hi - a.lo)));
    else if (a.scaling == SH_ROPE_RAMP) {
        const double per = rot / (2.0 * log(a.base));                                   // index of the pair with n turns: per log(ctx / (2 pi n))
        const double first = fmax(0.0, floor(per * log(a.ctx / (two_pi * a.hi)))), last = fmin(rot - 1.0, ceil(per * log(a.ctx / (two_pi * a.lo))));
        keep = 1.0 - fmin(1.0, fmax(0.0, (i - first) / fmax(last - first, 1e-3)));
    }
    if (a.scaling != SH_ROPE_NONE) w *= keep + (1.0 - keep) / a.factor;
    const double turns = w / two_pi;
    a.step[i] = (uint64_t)rint((turns - floor(turns)) * 0x1p64);
}

// Bound by HBM where rows are many (16 thousand rows, 328 MB: 66 us, 5.0 TB/s; all columns turned 63), else by the launch (64 rows 3.3 to 3.9 us). Turned columns that are no
// multiple of 8 go pair by pair, two bytes a lane (16 thousand rows of 40 heads of 80, 205 MB: 20 turned 76 us, 16 turned 56).
template <int P>
__global__ __launch_bounds__(256) void k_rope_pos(RopeArgs a) { rope_rows<P>(a, blockIdx.x * 256u + threadIdx.x); }

template <int P>
void launch_rope(RopeArgs a, bool in_place, hipStream_t st) {
    const uint32_t chunks = (in_place ? a.p.rot : a.dh) / (2 * P);
    a.dch = sh_make_div(chunks);
    const uint64_t all = (uint64_t)a.rows * a.heads * chunks;
    // Heads that share a thread's angles: as few as keep some million threads (16 thousand rows of 40 heads of 128, half of them turned: 9 heads 70.0 us,
    // 4 66.2, 2 67.6, 1 81.5; with 2000 rows 1 to 9 are level).
    a.hs = (uint32_t)std::min<uint64_t>(a.heads, std::max<uint64_t>(1, all >> 20));
    const uint32_t groups = sh_cdiv(a.heads, a.hs);
    a.dhg = sh_make_div(groups);
    const uint64_t per = (uint64_t)chunks * groups;
    const uint32_t most = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(a.rows, (1ull << 31) / per));     // items of a launch stay below 2^32
    const uint32_t rows = a.rows;
    for (uint64_t r = 0; r < rows; r += most) {
        a.row0 = (uint32_t)r;
        a.rows = (uint32_t)std::min<uint64_t>(rows, r + most);
        hipLaunchKernelGGL(k_rope_pos<P>, dim3((uint32_t)(((a.rows - a.row0) * per + 255) / 256)), dim3(256), 0, st, a);
    }
}

}  // namespace

extern "C" {

int sh_rope_steps(uint64_t step, uint32_t rot, double base, uint32_t scaling, double factor, double lo, double hi, uint32_t ctx) {
    if (!step || step % 8) { sh_set_error(-1, "[sh_rope_steps] NULL address, or not 8-byte aligned"); return -1; }
    if (rot < 2 || rot % 2 || rot > 65536) { sh_set_error(-1, "[sh_rope_steps] %u turned columns (even, 2 .. 65536)", rot); return -1; }
    if (!std::isfinite(base) || base <= 1.0) { sh_set_error(-1, "[sh_rope_steps] base %g (greater than 1)", base); return -1; }
    if (scaling > SH_ROPE_RAMP) { sh_set_error(-1, "[sh_rope_steps] unknown scaling %u", scaling); return -1; }
    if (scaling != SH_ROPE_NONE && !(std::isfinite(factor) && factor > 0.0 && std::isfinite(1.0 / factor))) { sh_set_error(-1, "[sh_rope_steps] factor %g", factor); return -1; }
    if (scaling >= SH_ROPE_BANDS && !(lo > 0.0 && hi > lo && std::isfinite(hi) && ctx)) {
        sh_set_error(-1, "[sh_rope_steps] turns %g .. %g of a context of %u", lo, hi, ctx);
        return -1;
    }
    hipLaunchKernelGGL(k_rope_steps, dim3(sh_cdiv(rot / 2, 64)), dim3(64), 0, sh_stream(),
                       StepArgs{(uint64_t *)step, rot / 2, scaling, ctx, base, factor, lo, hi});
    return sh_launch_ok("sh_rope_steps") ? 0 : SH_EHIP;
}

int sh_rope_pos(uint64_t y, uint64_t x, uint64_t pos, const sh_rope_plan *p, uint32_t rows, uint32_t heads, uint32_t dh, uint32_t ldy, uint32_t ldx) {
    RopeArgs a{};
    if (!dh || dh % 2) { sh_set_error(-1, "[sh_rope_pos] head width %u (even)", dh); return -1; }
    if (int rc = sh_rope_check("sh_rope_pos", p, dh, &a.p)) return rc;
    if (!rows || !heads) return 0;
    if (!y || !x || !pos) { sh_set_error(-1, "[sh_rope_pos] NULL address"); return -1; }
    if ((x | y) % 2 || pos % 4) { sh_set_error(-1, "[sh_rope_pos] rows must be 2-byte aligned, positions 4-byte aligned"); return -1; }
    const uint64_t wide = (uint64_t)heads * dh;
    if (ldy < wide || ldx < wide) { sh_set_error(-1, "[sh_rope_pos] leading dim %u or %u < %llu", ldy, ldx, (unsigned long long)wide); return -1; }
    if (rows >= (1u << 31)) { sh_set_error(-1, "[sh_rope_pos] %u rows", rows); return -1; }
    if (x == y && ldx != ldy) { sh_set_error(-1, "[sh_rope_pos] in place with leading dims %u and %u", ldy, ldx); return -1; }
    a.y = (uint16_t *)y; a.x = (const uint16_t *)x;
    a.pos = (const int32_t *)pos;
    a.ldy = ldy; a.ldx = ldx;
    a.rows = rows; a.heads = heads; a.dh = dh;
    const hipStream_t st = sh_stream();
    const bool in_place = x == y;
    if (dh % 16 == 0 && a.p.rot % 16 == 0 && (uint64_t)rows * wide >= (1u << 22)) launch_rope<8>(a, in_place, st);
    else if (dh % 8 == 0 && a.p.rot % 8 == 0) launch_rope<4>(a, in_place, st);
    else launch_rope<1>(a, in_place, st);
    return sh_launch_ok("sh_rope_pos") ? 0 : SH_EHIP;
}

}  // extern "C"
