// Attention over the 8-bit paged key / value cache (sh_attention_kv).
//
// Rows of one key / value head are taken together: row r of a request is new token r / grp and query head h grp + r % grp,
// so that grouped heads share every key read. Sixteen rows are a tile of the matrix instruction's columns:
//   S^T[key, row] = K . Q^T,  O^T[d, row] = V^T . P^T   (v_mfma_f32_16x16x32_f16, codes converted to fp16 exactly)
// over tiles of 64 keys, with the running maximum and sum of a softmax. The k order of a product is free as long as both
// operands use the same one, so no operand is moved between lanes:
//   - lane (m, g) (m = lane % 16, g = lane / 16) reads 16 consecutive codes of its key's row at 64 p + 16 g: K in whole
//     16-byte loads, Q at the same columns;
//   - row m of S^T's tile T is key 16 (m / 4) + 4 T + m % 4, so that lane (m, g) ends up with the scores of keys 16 g .. 16 g + 15
//     of row m: in order, as the second product's operand wants them, and all of one page;
//   - V^T's row d is stored with its tokens consecutive, so the lane reads the same 16 keys in one load.
// The scales of a page: the key's multiplies the scores of a lane (one page), the value's the probabilities. In fp16 p x vs
// could leave the range, so they are held as p x vs x cn, cn a power of two that brings the largest value scale
// met so far to 2^14 (smaller ones keep their precision until 2^-28 of it); the accumulators are brought along where cn changes.
#include "sh_kv.h"
#include <math.h>

namespace {

constexpr uint32_t KT = 64;                // keys of a tile
constexpr uint32_t QT = 16;                // rows of a tile
constexpr uint32_t GROUPS = 512;           // workgroups: two for each CU

struct AttnArgs {
    KvCache c;
    const uint16_t *q;
    uint16_t *o;
    const int32_t *table, *kv_len, *row_start;
    uint64_t ldq, ldo;
    uint32_t ld, B, rows, max_q, grp, prow, window, groups;
    float sc;                              // scale x log2 e
    float *part, *ml;                      // partials [groups][2][prow][dh], their (max, sum) [groups][2][prow][2]
    int4 *meta;                            // [groups]: request, item, last workgroup of the item begun here (-1: none)
};

struct Seq {
    uint32_t r0, n, nf, nqt, ft, nt;       // first row, rows served, rows of the request, row tiles, first key tile, key tiles
    int32_t L;
};

__device__ __forceinline__ Seq seq_of(const AttnArgs &a, uint32_t b) {
    Seq s;
    int32_t r0 = (int32_t)b, r1 = (int32_t)b + 1;
    if (a.row_start) { r0 = a.row_start[b]; r1 = a.row_start[b + 1]; }
    r0 = max(r0, 0);
    s.r0 = (uint32_t)r0;
    s.nf = r1 > r0 ? (uint32_t)(r1 - r0) : 0u;
    s.n = min(min(s.nf, a.max_q), s.r0 < a.rows ? a.rows - s.r0 : 0u);
    s.L = min(max(a.kv_len[b], 0), (int32_t)(a.ld << a.c.lbs));
    s.nqt = (s.n * a.grp + QT - 1) / QT;
    const int64_t lo = a.window ? max((int64_t)s.L - s.nf + 1 - a.window, (int64_t)0) : 0;
    s.ft = (uint32_t)lo / KT;
    s.nt = s.n ? max((uint32_t)(s.L + KT - 1) / KT, s.ft + 1) - s.ft : 0u;
    return s;
}

__device__ __forceinline__ float max_xor16_32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float sum_xor16_32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor((long long)v, d);
    return v;
}

// Bytes lo .. hi - 1 of a 16-byte value kept, the others cleared.
__device__ __forceinline__ uint4 keep_bytes(uint4 v, int lo, int hi) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int l = min(max(lo - 4 * i, 0), 4), h = min(max(hi - 4 * i, 0), 4);
        const uint32_t up = h == 4 ? ~0u : (1u << (8 * h)) - 1, dn = l == 4 ? ~0u : (1u << (8 * l)) - 1;
        w[i] &= up & ~dn;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Four consecutive outputs of a row.
__device__ __forceinline__ void store4(uint16_t *p, float a, float b, float c, float d) {
    const sh_h2 x = {(_Float16)a, (_Float16)b}, y = {(_Float16)c, (_Float16)d};
    *(sh_u2v_a2 *)p = (sh_u2v_a2){__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y)};
}

// All tiles of all (request, head, row tile) items, one behind the other, are dealt out evenly: workgroup i of N takes
// tiles i T / N .. (i + 1) T / N, its four waves a quarter each. A wave that has an item from its first tile to its last stores the
// result; parts of items are joined through LDS, and what crosses workgroups through `part` by k_kv_join. The lengths are
// on the GPU only, so the host cannot choose a split; this one keeps every CU busy whether one request is long or many are short.
template <int DP, bool FP8>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void k_kv_attn(AttnArgs a) {
    constexpr int NP = DP / 64, MT = DP / 16;
    extern __shared__ float s_o[];                                  // [8][prow][DP]
    __shared__ float s_ml[8][QT][2];
    __shared__ uint32_t s_seg[8][5];                                // request, item, first tile, end tile, tiles; request -1: none
    __shared__ uint64_t s_sum[4], s_base[4];
    __shared__ uint32_t s_b[4];
    const KvCache &c = a.c;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4;
    const uint32_t dh = c.dh;

    // ---- this wave's tiles
    uint64_t mine = 0;
    for (uint32_t b = tid; b < a.B; b += 256) { const Seq s = seq_of(a, b); mine += (uint64_t)s.nt * s.nqt * c.hkv; }
    const uint64_t wsum = wave_sum64(mine);
    if (lane == 0) s_sum[wave] = wsum;
    if (tid < 8) s_seg[tid][0] = ~0u;
    __syncthreads();
    const uint64_t T = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    const uint32_t N = (uint32_t)min((uint64_t)a.groups, max(T / 4, (uint64_t)1)), wg = blockIdx.x;
    if (wg >= N || T == 0) {
        if (tid == 0) a.meta[wg] = make_int4(-1, 0, 0, 0);
        return;
    }
    const uint64_t g0 = wg * T / N, g1 = (wg + 1) * T / N;
    uint64_t t = g0 + wave * (g1 - g0) / 4;
    const uint64_t t1 = g0 + (wave + 1) * (g1 - g0) / 4;
    {
        uint64_t carry = 0;
        for (uint32_t b0 = 0; b0 < a.B; b0 += 256) {
            const uint32_t b = b0 + tid;
            uint64_t w = 0;
            if (b < a.B) { const Seq s = seq_of(a, b); w = (uint64_t)s.nt * s.nqt * c.hkv; }
            uint64_t v = w;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint64_t x = (uint64_t)__shfl_up((long long)v, d);
                if ((int)lane >= d) v += x;
            }
            __syncthreads();
            if (lane == 63) s_sum[wave] = v;
            __syncthreads();
            uint64_t base = carry;
            for (uint32_t i = 0; i < 4; ++i) { if (i < wave) base += s_sum[i]; carry += s_sum[i]; }
            v += base;
            for (uint32_t i = 0; i < 4; ++i) {
                const uint64_t x = g0 + i * (g1 - g0) / 4;
                if (w && v - w <= x && x < v) { s_b[i] = b; s_base[i] = v - w; }
            }
        }
        __syncthreads();
    }
    uint32_t b = 0, item = 0, j0 = 0;
    Seq s{};
    if (t < t1) {
        b = __builtin_amdgcn_readfirstlane(s_b[wave]);
        s = seq_of(a, b);
        const uint64_t in = t - s_base[wave];
        item = __builtin_amdgcn_readfirstlane((uint32_t)(in / s.nt));
        j0 = __builtin_amdgcn_readfirstlane((uint32_t)(in - (uint64_t)item * s.nt));
    }
    const uint32_t kg = m >> 2, kr0 = m & 3;
    while (t < t1) {
        const uint32_t h = item / s.nqt, qt = item - h * s.nqt;
        const uint32_t j1 = (uint32_t)min((uint64_t)s.nt, j0 + (t1 - t));
        // ---- rows
        const uint32_t r = qt * QT + m, nrow = s.n * a.grp;
        const uint32_t qi = r / a.grp, qh = h * a.grp + (r - qi * a.grp);
        const int32_t first = s.L - (int32_t)s.nf;                                      // position of the request's first row
        const int32_t pos = r < nrow ? first + (int32_t)qi : -1;
        const int32_t pmin = first + (int32_t)(qt * QT / a.grp), pmax = first + (int32_t)((min(qt * QT + QT, nrow) - 1) / a.grp);
        const int32_t slo = a.window ? max(max(pmin, 0) - (int32_t)a.window + 1, 0) : 0;        // keys that any row sees: slo .. pmax
        const uint16_t *qp = a.q + (uint64_t)(s.r0 + qi) * a.ldq + (uint64_t)qh * dh;
        uint16_t *op = a.o + (uint64_t)(s.r0 + qi) * a.ldo + (uint64_t)qh * dh;
        sh_h8 qf[2 * NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            uint4 x = make_uint4(0, 0, 0, 0), y = x;
            if (r < nrow && 64 * p + 16 * g < dh) { x = sh_ld16_any(qp + 64 * p + 16 * g); y = sh_ld16_any(qp + 64 * p + 16 * g + 8); }
            qf[2 * p] = __builtin_bit_cast(sh_h8, x);
            qf[2 * p + 1] = __builtin_bit_cast(sh_h8, y);
        }
        sh_f4v oa[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) oa[i] = sh_f4v{0.f, 0.f, 0.f, 0.f};
        float mx = -1e30f, l = 0.f, cn = 0.f;

        const int32_t *tb = a.table + (uint64_t)b * a.ld;
        const uint32_t npg = max((uint32_t)(s.L + c.bs - 1) >> c.lbs, 1u), hoff = h * c.bs * dh;
        auto page_at = [&](uint32_t tok) { return (uint32_t)tb[min(tok >> c.lbs, npg - 1)]; };
        for (uint32_t j = j0; j < j1; ++j) {
            const uint32_t k0 = (s.ft + j) * KT;
            if ((int32_t)k0 > pmax || (int32_t)(k0 + KT) <= slo) continue;                  // no row of the item sees these keys
            const uint32_t kt = k0 + 16 * kg, vt = k0 + 16 * g;
            uint32_t kp = page_at(kt), vp = page_at(vt);
            const bool bad = vp >= c.pages;
            kp = kp < c.pages ? kp : 0;
            vp = bad ? 0 : vp;
            const uint8_t *kb = c.k + kp * c.pgk + hoff + ((kt & (c.bs - 1)) + kr0) * dh + 16 * g;
            const uint8_t *vb = c.v + vp * c.pgv + hoff + m * c.bs + (vt & (c.bs - 1));
            uint4 kr[4][NP], vr[MT];
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    kr[q][p] = 64 * p + 16 * g < dh ? *(const uint4 *)(kb + (uint64_t)(4 * q) * dh + 64 * p) : make_uint4(0, 0, 0, 0);
            const float ksc = c.ks[(uint64_t)vp * c.pgs + h] * a.sc;
            float vsc = c.vs[(uint64_t)vp * c.pgs + h];
#pragma unroll
            for (int i = 0; i < MT; ++i) vr[i] = 16u * i < dh ? *(const uint4 *)(vb + (uint64_t)(16 * i) * c.bs) : make_uint4(0, 0, 0, 0);

            sh_f4v sa[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                sa[q] = sh_f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    sa[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv_half8<FP8>(kr[q][p].x, kr[q][p].y), qf[2 * p], sa[q], 0, 0, 0);
                    sa[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv_half8<FP8>(kr[q][p].z, kr[q][p].w), qf[2 * p + 1], sa[q], 0, 0, 0);
                }
            }
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = sa[i >> 2][i & 3] * ksc;
            const bool edge = (int32_t)(k0 + KT - 1) > pmin || (a.window && (int32_t)k0 < pmax - (int32_t)a.window + 1) || __any(bad);
            if (edge) {
                const int32_t at = (int32_t)vt, from = a.window ? max(pos, 0) - (int32_t)a.window + 1 : 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = !bad && at + i <= pos && at + i >= from ? x[i] : -INFINITY;
                // what no row sees may hold anything: its codes and scale must not meet a probability of 0
                const int lo = bad ? 16 : max(slo - at, 0), hi = max(pmax + 1 - at, 0);
                if (lo >= min(hi, 16)) vsc = 0.f;
#pragma unroll
                for (int i = 0; i < MT; ++i) vr[i] = keep_bytes(vr[i], lo, hi);
            }
            float tm = x[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) tm = fmaxf(tm, x[i]);
            tm = max_xor16_32(tm);
            const float mn = fmaxf(mx, tm), vm = max_xor16_32(vsc);
            float cs = cn;
            if (!(vm * cn <= 16384.f) || cn == 0.f) cs = __builtin_amdgcn_ldexpf(1.f, 14 - (vm > 1e-30f ? __builtin_amdgcn_frexp_expf(vm) : -99));
            if (__any(mn > mx) || cs != cn) {
                const float al = sh_fast_exp2(mx - mn), be = al * (cn == 0.f ? 0.f : cs / cn);
                l *= al;
#pragma unroll
                for (int i = 0; i < MT; ++i) oa[i] *= be;
                mx = mn;
                cn = cs;
            }
            const float w = vsc * cn;
            sh_h8 pf[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = sh_fast_exp2(x[i] - mx);
                l += e;
                pf[i >> 3][i & 7] = (_Float16)(e * w);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
                if (16u * i < dh) {
                    oa[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv_half8<FP8>(vr[i].x, vr[i].y), pf[0], oa[i], 0, 0, 0);
                    oa[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv_half8<FP8>(vr[i].z, vr[i].w), pf[1], oa[i], 0, 0, 0);
                }
        }
        l = sum_xor16_32(l);
        const float ic = cn > 0.f ? 1.f / cn : 0.f;
        if (j0 == 0 && j1 == s.nt) {
            const float f = l > 0.f || l != l ? ic / l : 0.f;
            if (r < nrow)
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    if (16u * i < dh) store4(op + 16 * i + 4 * g, oa[i][0] * f, oa[i][1] * f, oa[i][2] * f, oa[i][3] * f);
        } else {
            const uint32_t sg = 2 * wave + (j0 ? 0 : 1);
            if (m < a.prow) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    if (16u * i < dh) *(sh_f4v *)&s_o[(sg * a.prow + m) * DP + 16 * i + 4 * g] = oa[i] * ic;
                if (g == 0) { s_ml[sg][m][0] = mx; s_ml[sg][m][1] = l; }
            }
            if (lane == 0) { s_seg[sg][0] = b; s_seg[sg][1] = item; s_seg[sg][2] = j0; s_seg[sg][3] = j1; s_seg[sg][4] = s.nt; }
        }
        t += j1 - j0;
        j0 = 0;
        if (j1 == s.nt && t < t1) {
            if (++item == s.nqt * c.hkv) {
                item = 0;
                do { s = seq_of(a, ++b); } while (s.nt == 0 && b + 1 < a.B);
            }
        }
    }
    __syncthreads();

    // ---- parts that belong together: consecutive, the first and the last may reach beyond this workgroup
    if (tid == 0) a.meta[wg] = make_int4(-1, 0, 0, 0);
    uint32_t i0 = 0;
    while (i0 < 8) {
        if (s_seg[i0][0] == ~0u) { ++i0; continue; }
        const uint32_t bb = s_seg[i0][0], it = s_seg[i0][1], ja = s_seg[i0][2], nt = s_seg[i0][4];
        uint32_t i1 = i0, je = s_seg[i0][3];
        for (uint32_t i = i0 + 1; i < 8; ++i)
            if (s_seg[i][0] == bb && s_seg[i][1] == it) { i1 = i; je = s_seg[i][3]; }
        const Seq q = seq_of(a, bb);
        const uint32_t h = it / q.nqt, qt = it - h * q.nqt, nrow = q.n * a.grp, qn = dh / 4;
        const bool whole = ja == 0 && je == nt;
        const uint32_t slot = ja ? 0 : 1;
        for (uint32_t e = tid; e < a.prow * qn; e += 256) {
            const uint32_t row = e / qn, d = 4 * (e - row * qn), r = qt * QT + row;
            if (r >= nrow) continue;
            float M = -1e30f, l = 0.f;
            sh_f4v o = {0.f, 0.f, 0.f, 0.f};
            for (uint32_t i = i0; i <= i1; ++i) if (s_seg[i][0] == bb && s_seg[i][1] == it) M = fmaxf(M, s_ml[i][row][0]);
            for (uint32_t i = i0; i <= i1; ++i)
                if (s_seg[i][0] == bb && s_seg[i][1] == it) {
                    const float f = sh_fast_exp2(s_ml[i][row][0] - M);
                    l += f * s_ml[i][row][1];
                    o += f * *(const sh_f4v *)&s_o[(i * a.prow + row) * DP + d];
                }
            if (whole) {
                const float f = l > 0.f || l != l ? 1.f / l : 0.f;
                const uint32_t qi = r / a.grp, qh = h * a.grp + (r - qi * a.grp);
                store4(a.o + (uint64_t)(q.r0 + qi) * a.ldo + (uint64_t)qh * dh + d, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
            } else {
                const uint64_t at = ((uint64_t)wg * 2 + slot) * a.prow + row;
                *(sh_f4v *)&a.part[at * dh + d] = o;
                if (d == 0) { a.ml[at * 2] = M; a.ml[at * 2 + 1] = l; }
            }
        }
        if (!whole && slot && tid == 0) {
            const uint64_t te = g1 + (nt - je);                                          // the item's end: it leaves here at je
            a.meta[wg] = make_int4((int)bb, (int)it, (int)((te * N - 1) / T), 0);
        }
        i0 = i1 + 1;
    }
}

// The items that cross workgroups: the one that began in workgroup x, its parts in order.
template <int DP>
__global__ __launch_bounds__(256) void k_kv_join(AttnArgs a) {
    constexpr uint32_t L = DP / 4, P = 256 / L;                     // lanes of a row, parts in flight
    __shared__ sh_f4v s_o[256];
    __shared__ float s_m[P], s_l[P];
    const int4 me = a.meta[blockIdx.x];
    if (me.x < 0) return;
    const uint32_t wg = blockIdx.x, dh = a.c.dh, row = blockIdx.y, y = threadIdx.x / L, d = 4 * (threadIdx.x % L);
    const Seq q = seq_of(a, (uint32_t)me.x);
    const uint32_t h = (uint32_t)me.y / q.nqt, qt = (uint32_t)me.y - h * q.nqt, r = qt * QT + row;
    if (r >= q.n * a.grp) return;
    float M = -1e30f, l = 0.f;
    sh_f4v o = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t i = wg + y; i <= (uint32_t)me.z; i += P) {
        const uint64_t at = ((uint64_t)i * 2 + (i == wg ? 1 : 0)) * a.prow + row;
        const float m = a.ml[at * 2], s = a.ml[at * 2 + 1];
        const sh_f4v v = d < dh ? *(const sh_f4v *)&a.part[at * dh + d] : sh_f4v{0.f, 0.f, 0.f, 0.f};
        const float mn = fmaxf(M, m), f = sh_fast_exp2(M - mn), e = sh_fast_exp2(m - mn);
        o = o * f + v * e;
        l = l * f + s * e;
        M = mn;
    }
    s_o[threadIdx.x] = o;
    if (d == 0) { s_m[y] = M; s_l[y] = l; }
    __syncthreads();
    if (y) return;
    float X = -1e30f, t = 0.f;
    for (uint32_t i = 0; i < P; ++i) X = fmaxf(X, s_m[i]);
    o = sh_f4v{0.f, 0.f, 0.f, 0.f};
    for (uint32_t i = 0; i < P; ++i) {
        const float e = sh_fast_exp2(s_m[i] - X);
        t += e * s_l[i];
        o += e * s_o[i * L + threadIdx.x];
    }
    if (d >= dh) return;
    const float f = t > 0.f || t != t ? 1.f / t : 0.f;
    const uint32_t qi = r / a.grp, qh = h * a.grp + (r - qi * a.grp);
    store4(a.o + (uint64_t)(q.r0 + qi) * a.ldo + (uint64_t)qh * dh + d, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
}

uint32_t part_rows(uint32_t max_q, uint32_t grp) { return (uint32_t)min((uint64_t)QT, (uint64_t)max_q * grp); }

template <int DP, bool FP8>
bool launch_attn(const AttnArgs &a, hipStream_t st) {
    static bool set = false;
    const uint32_t lds = 8 * a.prow * DP * 4;
    if (!set) {
        if (!sh_hip_ok(hipFuncSetAttribute((const void *)k_kv_attn<DP, FP8>, hipFuncAttributeMaxDynamicSharedMemorySize, 8 * QT * DP * 4),
                       "sh_attention_kv hipFuncSetAttribute")) return false;
        set = true;
    }
    hipLaunchKernelGGL((k_kv_attn<DP, FP8>), dim3(a.groups), dim3(256), lds, st, a);
    hipLaunchKernelGGL(k_kv_join<DP>, dim3(a.groups, a.prow), dim3(256), 0, st, a);
    return sh_launch_ok("sh_attention_kv");
}

}  // namespace

extern "C" {

uint64_t sh_attention_kv_ws_bytes(const sh_kv_cache *c, uint32_t B, uint32_t rows, uint32_t max_q, uint32_t H, uint32_t ld_table) {
    if (!c || !B || !rows || !max_q || !c->hkv || !H || !ld_table || !c->dh) return 0;
    const uint64_t prow = part_rows(max_q, H / c->hkv);
    return (uint64_t)GROUPS * (2 * prow * (c->dh + 2) * 4 + 16);
}

int sh_attention_kv(uint64_t q, uint64_t o, const sh_kv_cache *c, uint64_t table, uint32_t ld_table, uint64_t kv_len, uint64_t row_start,
                    uint32_t B, uint32_t rows, uint32_t max_q, uint32_t H, uint32_t ldq, uint32_t ldo, float scale, uint32_t window,
                    uint64_t ws, uint64_t ws_bytes) {
    AttnArgs a{};
    if (int rc = sh_kv_check("sh_attention_kv", c, &a.c)) return rc;
    if (!H || H % c->hkv) { sh_set_error(-1, "[sh_attention_kv] %u heads over %u key / value heads", H, c->hkv); return -1; }
    if (!B || !rows || !max_q) return 0;
    if (!q || !o || !table || !kv_len) { sh_set_error(-1, "[sh_attention_kv] NULL address"); return -1; }
    if ((q | o) % 2 || (table | kv_len | row_start) % 4) {
        sh_set_error(-1, "[sh_attention_kv] rows must be 2-byte aligned, table and lengths 4-byte aligned");
        return -1;
    }
    if (!ld_table || (uint64_t)ld_table * c->bs > (1ull << 31) - 128 || B > 65536 || rows > (1u << 30)) {
        sh_set_error(-1, "[sh_attention_kv] bad B=%u rows=%u ld_table=%u", B, rows, ld_table);
        return -1;
    }
    if ((uint64_t)H * c->dh > ldq || (uint64_t)H * c->dh > ldo) {
        sh_set_error(-1, "[sh_attention_kv] leading dim %u or %u < %u", ldq, ldo, H * c->dh);
        return -1;
    }
    const uint32_t grp = H / c->hkv;
    if ((uint64_t)min(max_q, rows) * grp >= (1ull << 31)) { sh_set_error(-1, "[sh_attention_kv] %u rows of %u heads", max_q, H); return -1; }
    if (!(fabsf(scale) <= 3.4e38f)) { sh_set_error(-1, "[sh_attention_kv] scale is not finite"); return -1; }
    const uint64_t need = sh_attention_kv_ws_bytes(c, B, rows, max_q, H, ld_table);
    if (!ws || ws % 16) { sh_set_error(-1, "[sh_attention_kv] ws must be a 16-byte aligned address"); return -1; }
    if (ws_bytes < need) {
        sh_set_error(-2, "[sh_attention_kv] workspace of %llu B < %llu B", (unsigned long long)ws_bytes, (unsigned long long)need);
        return -2;
    }
    a.q = (const uint16_t *)q; a.o = (uint16_t *)o;
    a.table = (const int32_t *)table; a.kv_len = (const int32_t *)kv_len; a.row_start = (const int32_t *)row_start;
    a.ldq = ldq; a.ldo = ldo; a.ld = ld_table;
    a.B = B; a.rows = rows; a.max_q = min(max_q, rows); a.grp = grp; a.prow = part_rows(max_q, grp);
    a.window = window < ld_table * c->bs ? window : 0;               // (one that no key falls out of is none)
    a.groups = GROUPS;
    a.sc = scale * 1.4426950408889634f;
    a.meta = (int4 *)ws;
    a.part = (float *)(ws + GROUPS * 16);
    a.ml = a.part + (uint64_t)GROUPS * 2 * a.prow * c->dh;
    const hipStream_t st = sh_stream();
    const bool f8 = c->fmt == SH_FP8;
    bool ok;
    if (c->dh <= 64) ok = f8 ? launch_attn<64, true>(a, st) : launch_attn<64, false>(a, st);
    else if (c->dh <= 128) ok = f8 ? launch_attn<128, true>(a, st) : launch_attn<128, false>(a, st);
    else ok = f8 ? launch_attn<256, true>(a, st) : launch_attn<256, false>(a, st);
    return ok ? 0 : SH_EHIP;
}

}  // extern "C"
