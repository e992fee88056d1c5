// Rotary positions: what sh_rope_pos and sh_kv_append_rope share (not part of the C ABI).
#pragma once
#include "sh_common.h"
#include <type_traits>

// A checked sh_rope_plan.
struct RopePlan {
    const uint64_t *step;
    uint32_t rot, pairs;     // pairs: neighbouring columns (SH_ROPE_PAIRS)
    double m;
};
// 0 and *out, or -1 with the message set. dh: the head's width.
int sh_rope_check(const char *name, const sh_rope_plan *p, uint32_t dh, RopePlan *out);

// (c, s) = m (cos, sin) of 2 pi phase / 2^64, phase = pos step mod 2^64: the whole turns fall off the product, so by a given step far positions
// lose nothing (the step's own error counts pos times). The phase is taken to the nearest quarter turn, the rest |a| <= pi / 4 goes through Taylor's series (sine to a^11,
// cosine to a^12: 7e-12 off at most), in fp64, whose rate is that of fp32 here. Rounded to fp32 once: other programs' 64-bit angles
// give the same cosine and sine, but for one in thousands of far positions.
__device__ __forceinline__ void rope_angle(uint32_t pos, uint64_t step, double m, float &c, float &s) {
    const uint64_t phase = step * pos;
    const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
    const uint64_t rest = phase - ((uint64_t)quarter << 62);                            // |rest| <= 2^61 as a signed number
    const double k = 6.283185307179586476925 * 0x1p-64;
    const double a = __builtin_fma((double)(int32_t)(rest >> 32), k * 0x1p32, (double)(uint32_t)rest * k), z = a * a;
    double p = __builtin_fma(z, -1.0 / 39916800, 1.0 / 362880), q = __builtin_fma(z, 1.0 / 479001600, -1.0 / 3628800);
    p = __builtin_fma(z, p, -1.0 / 5040);
    q = __builtin_fma(z, q, 1.0 / 40320);
    p = __builtin_fma(z, p, 1.0 / 120);
    q = __builtin_fma(z, q, -1.0 / 720);
    p = __builtin_fma(z, p, -1.0 / 6);
    q = __builtin_fma(z, q, 1.0 / 24);
    p = __builtin_fma(z * a, p, a);
    q = __builtin_fma(z, q, -0.5);
    q = __builtin_fma(z, q, 1.0);
    const float sn = (float)(p * m), cs = (float)(q * m);
    const bool odd = quarter & 1;
    c = odd ? sn : cs;
    s = odd ? cs : sn;
    if ((quarter + 1) & 2) c = -c;
    if (quarter & 2) s = -s;
}

// One pair, each product and each sum rounded to fp32, then fp16: what a table of fp32 cosines and sines gives.
__device__ __forceinline__ void rope_pair(uint16_t &h1, uint16_t &h2, float c, float s) {
#pragma clang fp contract(off)
    const float x1 = sh_dev_h2f(h1), x2 = sh_dev_h2f(h2);
    const float a = x1 * c, b = x2 * s, d = x2 * c, e = x1 * s;
    h1 = sh_dev_f2h(a - b);
    h2 = sh_dev_f2h(d + e);
}

// 2 P columns of a head: its chunk ch turns the pairs P ch .. P ch + P - 1, which lie in two groups of P columns from `a` and `b`; the chunks
// behind rot / 2 P are columns that stay.
template <int P>
__device__ __forceinline__ void rope_columns(const RopePlan &p, uint32_t ch, uint32_t &a, uint32_t &b) {
    const bool halves = !p.pairs && ch < p.rot / (2 * P);
    a = halves ? P * ch : 2 * P * ch;
    b = halves ? p.rot / 2 + P * ch : a + P;
}
template <int P>
__device__ __forceinline__ void rope_angles(const RopePlan &p, uint32_t ch, uint32_t pos, float (&c)[P], float (&s)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) rope_angle(pos, p.step[P * ch + i], p.m, c[i], s[i]);
}
// The turn of two groups of P columns (halves in w, first group first).
template <int P>
__device__ __forceinline__ void rope_turn(uint32_t (&w)[P], bool pairs, const float (&c)[P], const float (&s)[P]) {
    static_assert(P == 4 || P == 8, "columns of a group");
    if (pairs) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            uint16_t u = (uint16_t)w[i], v = (uint16_t)(w[i] >> 16);
            rope_pair(u, v, c[i], s[i]);
            w[i] = u | (uint32_t)v << 16;
        }
    } else {
#pragma unroll
        for (int i = 0; i < P / 2; ++i) {
            uint16_t u = (uint16_t)w[i], v = (uint16_t)w[i + P / 2], u2 = (uint16_t)(w[i] >> 16), v2 = (uint16_t)(w[i + P / 2] >> 16);
            rope_pair(u, v, c[2 * i], s[2 * i]);
            rope_pair(u2, v2, c[2 * i + 1], s[2 * i + 1]);
            w[i] = u | (uint32_t)u2 << 16;
            w[i + P / 2] = v | (uint32_t)v2 << 16;
        }
    }
}
// P halves at 2-byte alignment.
template <int P>
__device__ __forceinline__ void rope_load(const uint16_t *p, uint32_t *w) {
    if constexpr (P == 8) { const uint4 v = sh_ld16_any(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else { const sh_u2v_a2 v = *(const sh_u2v_a2 *)p; w[0] = v.x; w[1] = v.y; }
}
template <int P>
__device__ __forceinline__ void rope_store(uint16_t *p, const uint32_t *w) {
    if constexpr (P == 8) *(sh_u4v_a2 *)p = (sh_u4v){w[0], w[1], w[2], w[3]};
    else *(sh_u2v_a2 *)p = (sh_u2v_a2){w[0], w[1]};
}

// Heads of rows turned by their positions. A thread has one chunk of columns, its row's angles for them, and up to `hs` heads that they serve.
struct RopeArgs {
    RopePlan p;
    uint16_t *y;
    const uint16_t *x;
    const int32_t *pos;
    uint64_t ldy, ldx;
    uint32_t row0, rows, heads, dh, hs;
    ShDiv dch, dhg;           // by chunks of a head, by groups of hs heads
};
template <int P>
__device__ __forceinline__ void rope_rows(const RopeArgs &a, uint32_t item) {
    const uint32_t t = sh_div(item, a.dch), ch = item - t * a.dch.d, r = sh_div(t, a.dhg), row = a.row0 + r, h0 = (t - r * a.dhg.d) * a.hs;
    if (row >= a.rows) return;
    const int32_t pos = a.pos[row];
    if (pos < 0) return;
    const uint32_t h1 = min(h0 + a.hs, a.heads);
    const uint16_t *x = a.x + row * a.ldx + (uint64_t)h0 * a.dh;
    uint16_t *y = a.y + row * a.ldy + (uint64_t)h0 * a.dh;
    uint32_t ca, cb;
    rope_columns<P>(a.p, ch, ca, cb);
    const bool turned = ch < a.p.rot / (2 * P);
    float c[P], s[P];
    if (turned) rope_angles<P>(a.p, ch, (uint32_t)pos, c, s);
    if constexpr (P == 1) {
        for (uint32_t h = h0; h < h1; ++h, x += a.dh, y += a.dh) {
            uint16_t u = x[ca], v = x[cb];
            if (turned) rope_pair(u, v, c[0], s[0]);
            y[ca] = u;
            y[cb] = v;
        }
    } else {
        const auto heads = [&](auto count) {                         // some heads at once: their loads are on their way together
            constexpr int N = decltype(count)::value;
            uint32_t w[N][P];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                rope_load<P>(x + i * a.dh + ca, w[i]);
                rope_load<P>(x + i * a.dh + cb, w[i] + P / 2);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (turned) rope_turn<P>(w[i], a.p.pairs, c, s);
                rope_store<P>(y + i * a.dh + ca, w[i]);
                rope_store<P>(y + i * a.dh + cb, w[i] + P / 2);
            }
            x += N * a.dh;
            y += N * a.dh;
        };
        uint32_t h = h0;
        for (; h + 4 <= h1; h += 4) heads(std::integral_constant<int, 4>{});
        for (; h < h1; ++h) heads(std::integral_constant<int, 1>{});
    }
}
