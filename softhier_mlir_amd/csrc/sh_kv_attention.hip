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
//
// Single tokens are bound by HBM once the keys are many (two requests of 131 thousand keys, 516 MB: 90 us, 5.7 TB/s) and by latency
// below: the lengths, a page, its codes, the join, one after the other (one request of 937 keys 9.4 us; in a table of 128 pages and more, where
// items are cut and joined by a second launch, 11.2).
#include "sh_kv.h"
#include <algorithm>
#include <type_traits>

namespace {

constexpr uint32_t KT = 64;                // keys of a tile
constexpr uint32_t QT = 16;                // rows of a tile
constexpr uint32_t GROUPS = 256;           // workgroups at most: one for each CU, which is what their registers allow (512 are two rounds: 60 requests of
                                           // 600 keys, 64 wide, 19.1 us against 13.1)
constexpr uint32_t WHOLE_TILES = 4;        // key tiles of an item for each wave up to which it is not cut between workgroups (8 heads, 128 wide: 1000 keys
                                           // 11.6 us whole, 13.1 cut; 4000 keys 26.0 and 13.1)

struct ChunkUnit { uint32_t parts, r0, nrow, qt, h, step, pad[2]; };      // a cut unit: of an item's first part; parts 0: another part

struct AttnArgs {
    KvCache c;
    const uint16_t *q;
    uint16_t *o;
    const int32_t *table, *kv_len, *row_start;
    uint64_t ldq, ldo;
    uint32_t ld, B, rows, max_q, grp, prow, lq, window, groups, wide, whole, once;
    float sc;                              // scale x log2 e
    float *part, *ml;                      // partials [groups][2][prow][dh], their (max, sum) [groups][2][prow][2]
    ChunkUnit *unit;                       // [places]
    uint32_t places;                       // cut units of a call of chunks, at most
    int4 *meta;                            // [groups][2]: of the item begun here and not ended: its last tile (-1: none), first row, rows, head;
                                           // the request's first row, tiles of a workgroup, workgroups with one more
};

struct Seq {
    uint32_t r0, n, nf, nqt, ft, nt;       // first row, rows served, rows of the request, row tiles, first key tile, key tiles
    int32_t L;
};

// lq: log2 of a tile's rows.
__device__ __forceinline__ Seq seq_of(const AttnArgs &a, uint32_t b, uint32_t lq) {
    Seq s;
    int32_t r0 = (int32_t)b, r1 = (int32_t)b + 1;
    if (a.row_start) { r0 = a.row_start[b]; r1 = a.row_start[b + 1]; }
    r0 = max(r0, 0);
    s.r0 = (uint32_t)r0;
    s.nf = r1 > r0 ? (uint32_t)(r1 - r0) : 0u;
    s.n = min(min(s.nf, a.max_q), s.r0 < a.rows ? a.rows - s.r0 : 0u);
    s.L = min(max(a.kv_len[b], 0), (int32_t)(a.ld << a.c.lbs));
    s.nqt = (s.n * a.grp + (1u << lq) - 1) >> lq;
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

template <bool ONCE>                        // ONCE: not kept in the caches
__device__ __forceinline__ uint4 ld_codes(const uint8_t *p) {
    if constexpr (ONCE) {
        const sh_u4v q = __builtin_nontemporal_load((const sh_u4v *)p);
        return make_uint4(q.x, q.y, q.z, q.w);
    } else {
        return *(const uint4 *)p;
    }
}

// Eight halves of a row of q, infinities as NaN (x + 0 x): a score is then NaN for every key that the row sees and -inf for the others, so that
// a row whose scores are all -inf is not taken for one that sees no key.
__device__ __forceinline__ sh_h8 row8(uint4 v) {
    const sh_h8 x = __builtin_bit_cast(sh_h8, v);
    return __builtin_elementwise_fma(x, (sh_h8)(_Float16)0.f, x);
}
// The running maximum of a row that has seen no key, and the magnitude from which a maximum is `far` (below): 2^(x ks - mx) in one
// multiply-add is off by the rounding of mx = x ks, half a step: 2^-5 at 2^20, a factor of 2^32 at 2^30. There x ks is rounded before mx is
// taken off, and log2 w, which -mx would swallow, is added last.
constexpr float LOWEST = -3.4028234663852886e38f, FAR = 1048576.f;
__device__ __forceinline__ bool is_far(float mx) { return fabsf(mx) > FAR && mx != LOWEST; }
__device__ __forceinline__ float less_max(float x, float ks, float mx) {
#pragma clang fp contract(off)
    const float y = x * ks;
    return y - mx;
}

// Four consecutive outputs of a row.
__device__ __forceinline__ void store4(uint16_t *p, float a, float b, float c, float d) {
    const sh_h2 x = {(_Float16)a, (_Float16)b}, y = {(_Float16)c, (_Float16)d};
    *(sh_u2v_a2 *)p = (sh_u2v_a2){__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y)};
}

__device__ __forceinline__ Seq lane_seq(const Seq &s, uint32_t b) {
    const auto rl = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)b); };
    return Seq{rl(s.r0), rl(s.n), rl(s.nf), rl(s.nqt), rl(s.ft), rl(s.nt), (int32_t)rl((uint32_t)s.L)};
}

// All tiles of all (request, head, row tile) items, one behind the other, are dealt out evenly: T tiles to N workgroups, T / N
// or one more each, and those to its NW waves. A wave that has an item from its first tile to its last stores the
// result; parts of items are joined through LDS, and what crosses workgroups through `part` by k_kv_join. The lengths are
// on the GPU only, so the host cannot choose a split; this one keeps every CU busy whether one request is long or many are short.
// `whole`: where the table bounds an item to a few tiles for each wave, items are not cut between workgroups (each belongs to the
// one its first tile falls to) and the joining launch is not made.
// Up to 64 requests a lane holds a request and every wave finds its tiles by itself, up to a workgroup's threads they are in LDS
// (`wide`); MANY: more, the lengths are read in rounds. What runs once is kept short: its instructions come from memory, not the
// instruction cache, and cost more than the work (with 64-bit divisions and unrolled joins, 27 KB against 12: 64 requests of 300 to 500 keys 20.3 us
// against 16.6).
// DH: the head's width, or 0: any up to DP.
template <int DP, int DH, bool FP8, int NW, bool MANY>
__global__ __launch_bounds__(64 * NW) void k_kv_attn(AttnArgs a) {
    constexpr int NP = DP / 64, MT = (DH ? DH : DP) / 16;
    extern __shared__ float s_o[];                                  // [2 NW][prow][DP]
    __shared__ float s_ml[2 * NW][QT][2];
    __shared__ uint32_t s_seg[2 * NW][9];                           // request (-1: none), item, first tile, end tile, tiles; first row tile row, rows, head, first row
    __shared__ uint32_t s_sum[NW], s_b[NW], s_base[NW], s_up[MANY ? 1 : 64 * NW];
    __shared__ Seq s_seq[MANY ? 1 : 64 * NW];
    const KvCache &c = a.c;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4;
    const uint32_t dh = DH ? DH : c.dh, wg = blockIdx.x;
    const auto uni = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    const auto at_lane = [](uint32_t v, uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)i); };

    // ---- this wave's tiles
    Seq mine{};
    uint32_t T = 0, up = 0;
    if (lane < 2) s_seg[2 * wave + lane][0] = ~0u;                  // (only this wave writes these two until the barrier)
    if constexpr (MANY) {
        uint32_t sum = 0;
        for (uint32_t i = tid; i < a.B; i += 64 * NW) { const Seq q = seq_of(a, i, a.lq); sum += q.nt * q.nqt * c.hkv; }
        sum = kv_wave_scan(sum);
        if (lane == 63) s_sum[wave] = sum;
        __syncthreads();
        for (uint32_t i = 0; i < NW; ++i) T += s_sum[i];
        __syncthreads();
    } else {
        const uint32_t ix = a.wide ? tid : lane;
        if (ix < a.B) mine = seq_of(a, ix, a.lq);
        up = kv_wave_scan(mine.nt * mine.nqt * c.hkv);
        T = at_lane(up, 63);
        if (a.wide) {
            if (lane == 63) s_sum[wave] = up;
            s_seq[tid] = mine;
            __syncthreads();
            uint32_t z = 0;
            T = 0;
            for (uint32_t i = 0; i < NW; ++i) { const uint32_t v = s_sum[i]; z += i < wave ? v : 0u; T += v; }
            s_up[tid] = up + z;
            __syncthreads();
        }
    }
    T = uni(T);
    const uint32_t N = min(a.groups, max(T / NW, 1u));
    if (wg >= N || T == 0) {
        if (tid == 0 && !a.whole) a.meta[2 * wg] = make_int4(-1, 0, 0, 0);
        return;
    }
    const uint32_t share = T / N, more = T - share * N;
    uint32_t g0 = wg * share + min(wg, more), g1 = g0 + share + (wg < more ? 1 : 0), b = 0, base = 0;
    // the request that tile x < T belongs to
    const auto owner = [&](uint32_t x) {
        if (!a.wide) return (uint32_t)__builtin_ctzll(__ballot(up > x));
        uint32_t lo = 0, hi = a.B - 1;
        while (lo < hi) {
            const uint32_t i = (lo + hi) / 2;
            if (uni(s_up[i]) > x) hi = i; else lo = i + 1;
        }
        return lo;
    };
    const auto before = [&](uint32_t i) { return !i ? 0u : a.wide ? uni(s_up[i - 1]) : at_lane(up, i - 1); };
    if (!MANY && a.whole) {
        for (int k = 0; k < 2; ++k) {                               // to the first item that begins there or behind
            uint32_t &x = k ? g1 : g0;
            if (x >= T) continue;
            const uint32_t i = owner(x), z = before(i), nt = a.wide ? uni(s_seq[i].nt) : at_lane(mine.nt, i);
            x = z + (x - z + nt - 1) / nt * nt;
        }
    }
    const uint32_t t0 = g0 + wave * (g1 - g0) / NW, t1 = g0 + (wave + 1) * (g1 - g0) / NW;
    uint32_t t = t0;
    if constexpr (MANY) {
        uint32_t carry = 0;
        for (uint32_t b0 = 0; b0 < a.B; b0 += 64 * NW) {
            const uint32_t i = b0 + tid;
            uint32_t w = 0;
            if (i < a.B) { const Seq q = seq_of(a, i, a.lq); w = q.nt * q.nqt * c.hkv; }
            uint32_t v = kv_wave_scan(w);
            __syncthreads();
            if (lane == 63) s_sum[wave] = v;
            __syncthreads();
            uint32_t z = carry;
            for (uint32_t k = 0; k < NW; ++k) { const uint32_t x = s_sum[k]; z += k < wave ? x : 0u; carry += x; }
            v += z;
            for (uint32_t k = 0; k < NW; ++k) {
                const uint32_t x = g0 + k * (g1 - g0) / NW;
                if (w && v - w <= x && x < v) { s_b[k] = i; s_base[k] = v - w; }
            }
        }
        __syncthreads();
        if (t < t1) { b = uni(s_b[wave]); base = uni(s_base[wave]); }
    } else if (t < t1) {
        b = owner(t);
        base = before(b);
    }
    uint32_t from = 0;                                              // MANY: lane i holds request from + i
    const auto take = [&](uint32_t i) {
        from = i;
        mine = Seq{};
        if (i + lane < a.B) mine = seq_of(a, i + lane, a.lq);
    };
    const auto get = [&](uint32_t i) {
        if constexpr (!MANY)
            if (!a.wide) return lane_seq(mine, i);
        if constexpr (MANY) {
            take(i);
            return lane_seq(mine, 0);
        }
        const Seq q = s_seq[i];
        return Seq{uni(q.r0), uni(q.n), uni(q.nf), uni(q.nqt), uni(q.ft), uni(q.nt), (int32_t)uni((uint32_t)q.L)};
    };
    Seq s{};
    uint32_t item = 0, j0 = 0;
    if (t < t1) {
        s = get(b);
        item = uni((t - base) / s.nt);
        j0 = uni(t - base - item * s.nt);
    }
    // Codes that the Infinity Cache (256 MB) will not hold until the next call are read without allocating (120 MB and up here, one row tile): 48 requests
    // of up to 16384 keys, 311 MB, 72.6 -> 68.0 us; what it holds would be lost by that: 8 requests of 1000 keys 13.0 -> 14.5 us.
    const bool stream = a.once && T * (uint64_t)(2 * KT * dh) >= (120u << 20);
    // A probability's fp16 operand is off by up to 2^-11 of it, which shows where values cancel (a quarter more error in all). In items of
    // eight rows columns 8 .. 15 are the same rows again, and their operand of the second product is what the rounding of the first
    // eight's took off: the two columns' sum keeps 22 bits (48 requests of up to 16384 keys 60.1 -> 61.6 us, 937 keys 8.9 -> 9.4).
    // Items of sixteen keep the one: a second product of their own took 48 requests to 70.0.
    const bool two = a.lq == 3;
    const float rest = two && m >= QT / 2 ? 1.f : 0.f;
    const uint32_t kg = m >> 2, kr0 = m & 3;
    uint32_t kcol[NP];                                              // columns past the head's width: read as its first ones, against zeros of Q
#pragma unroll
    for (int p = 0; p < NP; ++p) kcol[p] = 64 * p + 16 * g < dh ? 64 * p + 16 * g : 0;
    while (t < t1) {
        const uint32_t h = item / s.nqt, qt = item - h * s.nqt;
        const uint32_t j1 = min(s.nt, j0 + (t1 - t));
        // ---- rows
        const uint32_t q0 = qt << a.lq, r = q0 + (two ? m & 7 : m), nrow = s.n * a.grp;
        const uint32_t qi = r / a.grp, qh = h * a.grp + (r - qi * a.grp);
        const int32_t first = s.L - (int32_t)s.nf;                                      // position of the request's first row
        const int32_t pos = r < nrow ? first + (int32_t)qi : -1;
        const int32_t pmin = first + (int32_t)(q0 / a.grp), pmax = first + (int32_t)((min(q0 + (1u << a.lq), nrow) - 1) / a.grp);
        const int32_t slo = a.window ? max(max(pmin, 0) - (int32_t)a.window + 1, 0) : 0;        // keys that any row sees: slo .. pmax
        // ---- key tiles that any row sees
        const uint32_t ja = max(j0, (uint32_t)slo / KT - s.ft), jb = pmax < 0 ? 0u : min(j1, (uint32_t)pmax / KT + 1 - s.ft);
        const int32_t *tb = a.table + (uint64_t)b * a.ld;
        const uint32_t npg = max((uint32_t)(s.L + c.bs - 1) >> c.lbs, 1u), hoff = h * c.bs * dh;
        const auto page_at = [&](uint32_t j, uint32_t sub) { return (uint32_t)tb[min(((s.ft + j) * KT + sub) >> c.lbs, npg - 1)]; };
        uint4 kr[4][NP], vr[MT];
        float ksc = 0.f, vsc = 0.f;
        uint32_t kp = 0, vp = 0;
        bool bad = false;
        const auto load_k = [&](auto once, uint32_t j) {
            const uint32_t kt = (s.ft + j) * KT + 16 * kg, pk = kp < c.pages ? kp : 0, pv = vp < c.pages ? vp : 0;
            const uint8_t *kb = c.k + pk * c.pgk + hoff + ((kt & (c.bs - 1)) + kr0) * dh;
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int p = 0; p < NP; ++p) kr[q][p] = ld_codes<decltype(once)::value>(kb + 4 * q * dh + kcol[p]);
            ksc = c.ks[(uint64_t)pv * c.pgs + h];
            vsc = c.vs[(uint64_t)pv * c.pgs + h];
        };
        const auto load_v = [&](auto once, uint32_t j, uint32_t page) {
            const uint32_t vt = (s.ft + j) * KT + 16 * g, pv = page < c.pages ? page : 0;
            const uint8_t *vb = c.v + pv * c.pgv + hoff + m * c.bs + (vt & (c.bs - 1));
#pragma unroll
            for (int i = 0; i < MT; ++i)
                if (DH || 16u * i < dh) vr[i] = ld_codes<decltype(once)::value>(vb + 16 * i * c.bs);
        };
        uint32_t vpc = 0;
        if (ja < jb) { kp = page_at(ja, 16 * kg); vp = page_at(ja, 16 * g); }
        const uint16_t *qp = a.q + (uint64_t)(s.r0 + qi) * a.ldq + (uint64_t)qh * dh;
        uint16_t *op = a.o + (uint64_t)(s.r0 + qi) * a.ldo + (uint64_t)qh * dh;
        sh_h8 qf[2 * NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            uint4 x = make_uint4(0, 0, 0, 0), y = x;
            if (r < nrow && 64 * p + 16 * g < dh) { x = sh_ld16_any(qp + 64 * p + 16 * g); y = sh_ld16_any(qp + 64 * p + 16 * g + 8); }
            qf[2 * p] = row8(x);
            qf[2 * p + 1] = row8(y);
        }
        sh_f4v oa[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) oa[i] = sh_f4v{0.f, 0.f, 0.f, 0.f};
        float mx = LOWEST, l = 0.f, cn = 0.f;
        bool far = false;
        const auto walk = [&](auto once) {
            if (ja < jb) {
                const uint32_t kn = page_at(ja + 1, 16 * kg), vn = page_at(ja + 1, 16 * g);
                vpc = vp;
                load_k(once, ja);
                load_v(once, ja, vpc);
                kp = kn;
                vp = vn;
            }
            for (uint32_t j = ja; j < jb; ++j) {
                const uint32_t k0 = (s.ft + j) * KT, vt = k0 + 16 * g;
                bad = vpc >= c.pages;
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
                float x[16], vs = vsc;
                const float ks = fmaxf(ksc * a.sc, 1e-37f);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = sa[i >> 2][i & 3];
                // the pages after the next tile's first (loads end in order), then its keys
                const uint32_t vcur = vp;
                if (j + 1 < jb) {
                    const uint32_t kn = page_at(j + 2, 16 * kg), vn = page_at(j + 2, 16 * g);
                    load_k(once, j + 1);
                    kp = kn;
                    vp = vn;
                }
                const bool edge = (int32_t)(k0 + KT - 1) > pmin || (a.window && (int32_t)k0 < pmax - (int32_t)a.window + 1) || __any(bad);
                if (edge) {
                    const int32_t at = (int32_t)vt, from = a.window ? max(pos, 0) - (int32_t)a.window + 1 : 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = !bad && at + i <= pos && at + i >= from ? x[i] : -INFINITY;
                    // what no row sees may hold anything: its codes and scale must not meet a probability of 0
                    const int lo = bad ? 16 : max(slo - at, 0), hi = max(pmax + 1 - at, 0);
                    if (lo >= min(hi, 16)) vs = 0.f;
#pragma unroll
                    for (int i = 0; i < MT; ++i) vr[i] = keep_bytes(vr[i], lo, hi);
                }
                float tm = x[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) tm = fmaxf(tm, x[i]);
                tm = max_xor16_32(tm * ks);                             // (a lane's scores have one scale)
                const float mn = fmaxf(mx, tm), vm = max_xor16_32(vs);
                float cs = cn;
                if (!(vm * cn <= 16384.f) || cn == 0.f) cs = __builtin_amdgcn_ldexpf(1.f, 14 - (vm > 1e-30f ? __builtin_amdgcn_frexp_expf(vm) : -99));
                if (__any(mn > mx) || cs != cn || far) {
                    const float al = sh_fast_exp2(mx - mn), be = al * (cn == 0.f ? 0.f : cs / cn);
                    l *= al;
#pragma unroll
                    for (int i = 0; i < MT; ++i) oa[i] *= be;
                    mx = mn;
                    cn = cs;
                    far = __any(is_far(mx));
                    if (far)
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = less_max(x[i], ks, mx);
                }
                // probability and weight in one exponential: 2^(score - maximum + log2 w), the sum taken back from it
                const float w = fmaxf(vs * cn, 1e-30f), z = __builtin_amdgcn_logf(w) - (far ? 0.f : mx), kx = far ? 1.f : ks;
                float sum = 0.f;
                sh_h8 pf[2];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float e = sh_fast_exp2(fmaf(x[i], kx, z));
                    sum += e;
                    pf[i >> 3][i & 7] = (_Float16)fmaf(-(float)(_Float16)e, rest, e);
                }
                l = fmaf(sum, sh_fast_rcp(w), l);
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    if (DH || 16u * i < dh) {
                        oa[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv_half8<FP8>(vr[i].x, vr[i].y), pf[0], oa[i], 0, 0, 0);
                        oa[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv_half8<FP8>(vr[i].z, vr[i].w), pf[1], oa[i], 0, 0, 0);
                    }
                vpc = vcur;
                if (j + 1 < jb) load_v(once, j + 1, vpc);
            }
        };
        if constexpr (DH != 0) { if (stream) walk(std::true_type{}); else walk(std::false_type{}); }
        else walk(std::false_type{});
        l = sum_xor16_32(l);
        if (two)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k)                         // (row_ror:8)
                    oa[i][k] += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(oa[i][k]), 0x128, 0xf, 0xf, true));
        const float ic = cn > 0.f ? 1.f / cn : 0.f;
        if (j0 == 0 && j1 == s.nt) {
            const float f = l > 0.f || l != l ? ic / l : 0.f;
            if (r < nrow && (m < 8 || !two))
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    if (DH || 16u * i < dh) store4(op + 16 * i + 4 * g, oa[i][0] * f, oa[i][1] * f, oa[i][2] * f, oa[i][3] * f);
        } else {
            const uint32_t sg = 2 * wave + (j0 ? 0 : 1);
            if (m < a.prow) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    if (DH || 16u * i < dh) *(sh_f4v *)&s_o[(sg * a.prow + m) * DP + 16 * i + 4 * g] = oa[i] * ic;
                if (g == 0) { s_ml[sg][m][0] = mx; s_ml[sg][m][1] = l; }
            }
            if (lane == 0) {
                s_seg[sg][0] = b; s_seg[sg][1] = item; s_seg[sg][2] = j0; s_seg[sg][3] = j1; s_seg[sg][4] = s.nt;
                s_seg[sg][5] = q0; s_seg[sg][6] = nrow; s_seg[sg][7] = h; s_seg[sg][8] = s.r0;
            }
        }
        t += j1 - j0;
        j0 = 0;
        if (j1 == s.nt && t < t1) {
            if (++item == s.nqt * c.hkv) {
                item = 0;
                if constexpr (MANY) {                               // the next request with tiles, 64 at a time: idle ones may be thousands
                    uint64_t has = 0;
                    for (++b; b < a.B && !has;) {
                        if (b - from >= 64) take(b);
                        has = __ballot(mine.nt != 0) >> (b - from);
                        b = has ? b + __builtin_ctzll(has) : from + 64;
                    }
                    if (!has) break;                                // (lengths that changed while the kernel ran)
                    s = lane_seq(mine, b - from);
                } else {
                    do { s = get(++b); } while (s.nt == 0 && b + 1 < a.B);
                }
            }
        }
    }
    __syncthreads();

    // ---- parts that belong together: consecutive, the first and the last may reach beyond this workgroup. A wave takes every NW-th
    // 64 elements (four columns of a row each) of all of them.
    if (tid == 0 && !a.whole) a.meta[2 * wg] = make_int4(-1, 0, 0, 0);
    const uint32_t gs = min(lane, 2u * NW - 1);                     // lane i holds part i
    const uint32_t gb = lane < 2 * NW ? s_seg[gs][0] : ~0u, gi = s_seg[gs][1];
    const uint32_t qn = dh / 4, blocks = (a.prow * qn + 63) / 64;
    uint32_t turn = wave;
    for (uint64_t left = __ballot(gb != ~0u); left;) {
        const uint32_t i0 = __builtin_ctzll(left);
        const uint64_t in = __ballot(gb == at_lane(gb, i0) && gi == at_lane(gi, i0));
        left &= ~in;
        const uint32_t iz = 63 - __builtin_clzll(in);
        const uint32_t ja = uni(s_seg[i0][2]), je = uni(s_seg[iz][3]), nt = uni(s_seg[i0][4]), q0 = uni(s_seg[i0][5]), nrow = uni(s_seg[i0][6]),
                       h = uni(s_seg[i0][7]), r0 = uni(s_seg[i0][8]);
        const bool all = ja == 0 && je == nt;
        for (; turn < blocks; turn += NW) {
            const uint32_t e = turn * 64 + lane, row = e / qn, d = 4 * (e - row * qn), r = q0 + row;
            if (row >= a.prow || r >= nrow) continue;
            float M = LOWEST, l = 0.f;
            sh_f4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (uint64_t k = in; k; k &= k - 1) {
                const uint32_t i = __builtin_ctzll(k);
                const float pm = s_ml[i][row][0], mn = fmaxf(M, pm), f = sh_fast_exp2(M - mn), x = sh_fast_exp2(pm - mn);
                l = l * f + s_ml[i][row][1] * x;
                o = o * f + *(const sh_f4v *)&s_o[(i * a.prow + row) * DP + d] * x;
                M = mn;
            }
            if (all) {
                const float f = l > 0.f || l != l ? 1.f / l : 0.f;
                const uint32_t qi = r / a.grp, qh = h * a.grp + (r - qi * a.grp);
                store4(a.o + (uint64_t)(r0 + qi) * a.ldo + (uint64_t)qh * dh + d, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
            } else {
                const uint64_t at = ((uint64_t)wg * 2 + (ja ? 0 : 1)) * a.prow + row;
                *(sh_f4v *)&a.part[at * dh + d] = o;
                if (d == 0) { a.ml[at * 2] = M; a.ml[at * 2 + 1] = l; }
            }
        }
        turn -= blocks;
        if (!all && !ja && tid == 0) {                              // it begins here and leaves at je: where it ends, and how tiles are shared
            a.meta[2 * wg] = make_int4((int)(g1 + (nt - je) - 1), (int)q0, (int)nrow, (int)h);
            a.meta[2 * wg + 1] = make_int4((int)r0, (int)share, (int)more, 0);
        }
    }
}

// The items that cross workgroups: the one that began in workgroup x, its parts in order.
template <int DP>
__global__ __launch_bounds__(256) void k_kv_join(AttnArgs a) {
    constexpr uint32_t L = DP / 4, P = 256 / L;                     // lanes of a row, parts in flight
    __shared__ sh_f4v s_o[256];
    __shared__ float s_m[P], s_l[P];
    const int4 me = a.meta[2 * blockIdx.x], at_ = a.meta[2 * blockIdx.x + 1];
    if (me.x == -1) return;
    const uint32_t wg = blockIdx.x, dh = a.c.dh, row = blockIdx.y, y = threadIdx.x / L, d = 4 * (threadIdx.x % L), r = (uint32_t)me.y + row;
    if (r >= (uint32_t)me.z) return;
    // the workgroup of the item's last tile
    const uint32_t x = (uint32_t)me.x, share = (uint32_t)at_.y, more = (uint32_t)at_.z, big = more * (share + 1);
    const uint32_t end = x < big ? x / (share + 1) : more + (x - big) / share;
    float M = LOWEST, l = 0.f;
    sh_f4v o = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t i = wg + y; i <= end; i += P) {
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
    float X = LOWEST, t = 0.f;
    for (uint32_t i = 0; i < P; ++i) X = fmaxf(X, s_m[i]);
    o = sh_f4v{0.f, 0.f, 0.f, 0.f};
    for (uint32_t i = 0; i < P; ++i) {
        const float e = sh_fast_exp2(s_m[i] - X);
        t += e * s_l[i];
        o += e * s_o[i * L + threadIdx.x];
    }
    if (d >= dh) return;
    const float f = t > 0.f || t != t ? 1.f / t : 0.f;
    const uint32_t qi = r / a.grp, qh = (uint32_t)me.w * a.grp + (r - qi * a.grp);
    store4(a.o + (uint64_t)((uint32_t)at_.x + qi) * a.ldo + (uint64_t)qh * dh + d, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
}

// ---- many rows: chunks of prompts ------------------------------------------------------------------------------------
// A workgroup of four waves takes 128 rows of an item, 32 a wave, through the keys the rows see, 64 at a time: the codes are converted
// once for all four waves into LDS (K rows and V^T rows of fp16, padded by 16 bytes: the operand reads then meet every bank once), two
// buffers, the codes after the next in flight. S^T and O^T on v_mfma_f32_32x32x16_f16. As above no operand moves between
// lanes: row m of a score tile's A operand is key 16 (m / 16) + 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4, so that the lane (n, hi) gets
// the scores of keys 16 q + 8 hi + 0 .. 7 of row n, which is the second product's operand.
// Bound by no one pipe: 512 rows each of four requests of 8000 keys, 32 heads over 8, take 370 us (700 TFLOP/s), of which the vector pipe
// is busy half (a multiply-add, an exponential and an addition a score, half a maximum, half a conversion, the codes of its share), the
// matrix pipe 31 % (32 instructions for 64 keys by 32 rows), LDS 30 % (32 KB read a wave and tile). One comes after the other: two waves a SIMD,
// 1.7 on average, and a barrier a tile overlap them little, and of its time a wave waits 25 % for data and barriers and 27 % to
// issue. 4096 rows of one prompt 220 us, 620 TFLOP/s.
// The keys of an item are cut into parts of C tiles, C a 768th of all tiles (and at least 8): one long request among short ones, or a
// few rows over a long context, then keep every CU busy. Units are dealt out by the hardware, the request's last row tiles first
// (they see most). A request that is cut has more than C tiles, so cut units number at most 2 T / C <= 1536, and no more than all units cut
// at the table's width: their parts go to as many places of `part`, which k_kv_chunk_join adds up. The launch has enough blocks, and
// `part` enough places, while row_start does not decrease; where it does (an error of the caller's), the units behind the last block
// or place do not exist, and an item that lacks parts for that is not joined.
constexpr uint32_t LCT = 7, CT = 1u << LCT;  // rows of a unit
constexpr uint32_t CUT = 768;              // units that share the whole evenly: three workgroups a CU, two of them at a time
constexpr uint32_t CUT_MIN = 8;            // tiles of a part at least
template <int DP, bool FP8>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void k_kv_chunk(AttnArgs a) {
    constexpr int KS = DP / 16, DT = DP / 32, NC = DP / 64;          // k-steps, column tiles, 16-byte chunks of K (of V) a thread stages
    constexpr uint32_t KLD = DP + 8, VLD = KT + 8;
    __shared__ __align__(16) uint16_t s_k[2][KT * KLD];
    __shared__ __align__(16) uint16_t s_v[2][DP * VLD];
    __shared__ float s_sc[2][4][2];
    __shared__ uint32_t s_bad[2][4];
    const KvCache &c = a.c;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, hi = lane >> 5, dh = c.dh;

    // ---- the unit: heads first, then parts, then row tiles from the last one on, then requests
    uint64_t all = 0;
    Seq q{};
    for (uint32_t b0 = 0; b0 < a.B; b0 += 64) {
        q = Seq{};
        if (b0 + lane < a.B) q = seq_of(a, b0 + lane, LCT);
        all += (uint64_t)q.nt * q.nqt * c.hkv;
    }
    all = wave_sum64(all);
    const uint32_t C = (uint32_t)max((all + CUT - 1) / CUT, (uint64_t)CUT_MIN);
    uint32_t idx = blockIdx.x, b = 0, parts = 1, cut0 = 0;           // cut0: cut units before this request
    uint32_t base = 0, cuts = 0;                                     // block 0: units of the earlier rounds, cut units that this launch has
    Seq s{};
    bool found = false;
    for (uint32_t b0 = 0; b0 < a.B; b0 += 64) {
        if (a.B > 64) {
            q = Seq{};
            if (b0 + lane < a.B) q = seq_of(a, b0 + lane, LCT);
        }
        const uint32_t p = (q.nt + C - 1) / C, w = q.nqt * c.hkv * p, up = kv_wave_scan(w), cu = kv_wave_scan(p > 1 ? w : 0u);
        const auto last = [](uint32_t v, uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)i); };
        const uint64_t hit = found ? 0 : __ballot(up > idx);
        if (hit) {
            const uint32_t i = __builtin_ctzll(hit);
            b = b0 + i;
            s = lane_seq(q, i);
            parts = last(p, i);
            idx -= i ? last(up, i - 1) : 0u;
            cut0 += i ? last(cu, i - 1) : 0u;
            found = true;
            if (blockIdx.x) break;
        } else if (!found) {
            idx -= last(up, 63);
            cut0 += last(cu, 63);
        }
        if (!blockIdx.x) {
            const uint32_t z = base + up - w;
            cuts += last(kv_wave_scan(p > 1 && z < gridDim.x ? min(w, gridDim.x - z) : 0u), 63);
            base = min(base + last(up, 63), gridDim.x);
        }
    }
    if (!blockIdx.x && tid == 0) a.meta[0].x = (int)min(cuts, a.places);
    if (!found) return;
    // (all of it is uniform: kept in scalar registers)
    const auto uni = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    s = Seq{uni(s.r0), uni(s.n), uni(s.nf), uni(s.nqt), uni(s.ft), uni(s.nt), (int32_t)uni((uint32_t)s.L)};
    b = uni(b); parts = uni(parts); idx = uni(idx); cut0 = uni(cut0);
    const uint32_t h = idx % c.hkv, sp = idx / c.hkv % parts, qt = s.nqt - 1 - idx / c.hkv / parts, cut = cut0 + idx;
    if (parts > 1 && cut >= a.places) return;                       // (only where row_start decreases)

    // ---- rows
    const uint32_t nrow = s.n * a.grp, w0 = qt * CT + 32 * wave, r = w0 + n;
    const uint32_t qi = r / a.grp, qh = h * a.grp + (r - qi * a.grp);
    const int32_t first = s.L - (int32_t)s.nf;
    const int32_t pos = r < nrow ? first + (int32_t)qi : -1;
    const auto row_pos = [&](uint32_t x) { return first + (int32_t)(min(x, nrow - 1) / a.grp); };
    const int32_t pmin = row_pos(qt * CT), pmax = row_pos(qt * CT + CT - 1);                // of the workgroup, and of this wave
    const int32_t wmin = row_pos(w0), wmax = w0 < nrow ? row_pos(w0 + 31) : -1;
    const int32_t win = (int32_t)a.window;
    const int32_t slo = win ? max(max(pmin, 0) - win + 1, 0) : 0;
    uint32_t ja = (uint32_t)slo / KT, jb = pmax < 0 ? ja : (uint32_t)pmax / KT + 1;
    if (parts > 1) {
        const uint32_t t = jb - ja, z = ja;
        ja = z + (uint32_t)((uint64_t)sp * t / parts);
        jb = z + (uint32_t)((uint64_t)(sp + 1) * t / parts);
    }
    const uint16_t *qp = a.q + (uint64_t)(s.r0 + qi) * a.ldq + (uint64_t)qh * dh;
    sh_h8 qf[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < nrow && 16u * k < dh) x = sh_ld16_any(qp + 16 * k + 8 * hi);
        qf[k] = row8(x);
    }

    // ---- staging: K chunk i of the wave is keys (64 wave + 256 i) / (DP / 16) on (16 at most, of one page), a lane 16 columns of one;
    // V chunk i is keys 16 wave .. 16 wave + 15 of column 64 i + lane. So a wave's pages are scalars, a lane's offsets constants.
    typedef const __attribute__((address_space(4))) int32_t *Table;
    const Table tb = (Table)(uintptr_t)(a.table + (uint64_t)b * a.ld);
    const uint32_t npg = max((uint32_t)(s.L + c.bs - 1) >> c.lbs, 1u), hoff = h * c.bs * dh;
    const uint32_t kcol = 16 * (lane % (DP / 16)), kofs = lane / (DP / 16) * dh + (kcol < dh ? kcol : 0);
    uint32_t vofs[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) vofs[i] = min(64u * i + lane, dh - 1) * c.bs;
    uint32_t kpg[NC], vpg = 0, vpc = 0;
    uint4 kr[NC], vr[NC];
    float ksc = 0.f, vsc = 0.f;
    const auto key_of = [&](int i) { return (64u * wave + 256u * i) / (DP / 16); };
    const auto pages = [&](uint32_t j) {
#pragma unroll
        for (int i = 0; i < NC; ++i) kpg[i] = (uint32_t)tb[min((j * KT + key_of(i)) >> c.lbs, npg - 1)];
        vpg = (uint32_t)tb[min((j * KT + 16 * wave) >> c.lbs, npg - 1)];
    };
    const auto load = [&](uint32_t j) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const uint32_t p = kpg[i] < c.pages ? kpg[i] : 0, key = (j * KT + key_of(i)) & (c.bs - 1);
            kr[i] = *(const uint4 *)(c.k + (uint64_t)p * c.pgk + (hoff + key * dh) + kofs);
        }
        vpc = vpg;
        const uint32_t p = vpg < c.pages ? vpg : 0, key = (j * KT + 16 * wave) & (c.bs - 1);
#pragma unroll
        for (int i = 0; i < NC; ++i) vr[i] = *(const uint4 *)(c.v + (uint64_t)p * c.pgv + (hoff + key) + vofs[i]);
        ksc = c.ks[(uint64_t)p * c.pgs + h];
        vsc = c.vs[(uint64_t)p * c.pgs + h];
    };
    const auto store16 = [](uint16_t *p, uint4 v) {
        *(sh_h8 *)p = kv_half8<FP8>(v.x, v.y);
        *(sh_h8 *)(p + 8) = kv_half8<FP8>(v.z, v.w);
    };
    const auto stage = [&](uint32_t j) {
        const uint32_t u = j & 1;
        const int32_t at = (int32_t)(j * KT + 16 * wave);
        const bool bad = vpc >= c.pages;
        const int lo = bad ? 16 : max(slo - at, 0), hic = max(pmax + 1 - at, 0);            // what no row sees may hold anything
        if (lo > 0 || hic < 16)
#pragma unroll
            for (int i = 0; i < NC; ++i) vr[i] = keep_bytes(vr[i], lo, hic);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            // (columns past the head's width: zeros, for whatever bytes were read)
            store16(&s_k[u][(key_of(i) + lane / (DP / 16)) * KLD + kcol], kcol < dh ? kr[i] : make_uint4(0, 0, 0, 0));
            store16(&s_v[u][(64 * i + lane) * VLD + 16 * wave], vr[i]);
        }
        if (lane == 0) {
            s_sc[u][wave][0] = fmaxf(ksc * a.sc, 1e-37f);
            s_sc[u][wave][1] = lo >= min(hic, 16) ? 0.f : vsc;
            s_bad[u][wave] = bad;
        }
    };

    sh_f16v oa[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) oa[i] = sh_f16v{};
    float mx = LOWEST, l = 0.f, cn = 0.f;
    bool far = false;
    if (ja < jb) {
        pages(ja);
        load(ja);
        pages(ja + 1);
        stage(ja);
        if (ja + 1 < jb) { load(ja + 1); pages(ja + 2); }
    }
    const uint32_t krow = 16 * (n >> 4) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);
    for (uint32_t j = ja; j < jb; ++j) {
        __syncthreads();                                            // tile j is staged, tile j - 1 is read
        if (j + 1 < jb) {
            stage(j + 1);
            if (j + 2 < jb) { load(j + 2); pages(j + 3); }
        }
        const uint32_t u = j & 1;
        const int32_t k0 = (int32_t)(j * KT);
        if (k0 > wmax || (win && k0 + (int32_t)KT <= max(wmin, 0) - win + 1)) continue;     // this wave's rows see none of these keys
        sh_f16v sa[2] = {};
        const uint16_t *kp = &s_k[u][krow * KLD + 8 * hi];
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int t = 0; t < 2; ++t)
                sa[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const sh_h8 *)(kp + 32 * t * KLD + 16 * k), qf[k], sa[t], 0, 0, 0);
        float ks[4], vs[4];
        uint32_t bad = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) { ks[q] = s_sc[u][q][0]; vs[q] = s_sc[u][q][1]; bad |= s_bad[u][q] << q; }
        bad = __builtin_amdgcn_readfirstlane(bad);
        if (k0 + (int32_t)KT - 1 > wmin || (win && k0 < wmax - win + 1) || bad) {
            const int32_t at = k0 + 8 * (int32_t)hi, from = win ? max(pos, 0) - win + 1 : 0;
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int32_t key = at + 16 * q + e;
                    float &x = ((float *)&sa[q >> 1])[8 * (q & 1) + e];
                    x = key <= pos && key >= from && !(bad >> q & 1) ? x : -INFINITY;
                }
        }
        // a page's scores have one scale: its largest is the largest product's
        float tm = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float m8 = sa[q >> 1][8 * (q & 1)];
#pragma unroll
            for (int e = 1; e < 8; ++e) m8 = fmaxf(m8, sa[q >> 1][8 * (q & 1) + e]);
            tm = fmaxf(tm, m8 * ks[q]);
        }
        const float mn = fmaxf(mx, sh_max_xor32(tm)), vm = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
        float cs = cn;
        if (!(vm * cn <= 16384.f) || cn == 0.f) cs = __builtin_amdgcn_ldexpf(1.f, 14 - (vm > 1e-30f ? __builtin_amdgcn_frexp_expf(vm) : -99));
        if (__any(mn > mx) || cs != cn || far) {
            const float al = sh_fast_exp2(mx - mn), be = al * (cn == 0.f ? 0.f : cs / cn);
            l *= al;
#pragma unroll
            for (int i = 0; i < DT; ++i) oa[i] *= be;
            mx = mn;
            cn = cs;
            far = __any(is_far(mx));
            if (far)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float &x = ((float *)&sa[q >> 1])[8 * (q & 1) + e];
                        x = less_max(x, ks[q], mx);
                    }
        }
        // probability and weight in one exponential: 2^(score - maximum + log2 w), the sum taken back from it
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float w = fmaxf(vs[q] * cn, 1e-30f), z = __builtin_amdgcn_logf(w) - (far ? 0.f : mx), kx = far ? 1.f : ks[q];
            float sum = 0.f;
            sh_h8 pf;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = sh_fast_exp2(fmaf(sa[q >> 1][8 * (q & 1) + e], kx, z));
                sum += p;
                pf[e] = (_Float16)p;
            }
            l = fmaf(sum, sh_fast_rcp(w), l);
            const uint16_t *vp = &s_v[u][n * VLD + 16 * q + 8 * hi];
#pragma unroll
            for (int i = 0; i < DT; ++i) oa[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const sh_h8 *)(vp + 32 * i * VLD), pf, oa[i], 0, 0, 0);
        }
    }
    const auto lr = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(lr[0]) + __uint_as_float(lr[1]);
    const float ic = cn > 0.f ? 1.f / cn : 0.f;
    if (parts == 1) {
        if (r >= nrow) return;
        uint16_t *op = a.o + (uint64_t)(s.r0 + qi) * a.ldo + (uint64_t)qh * dh;
        const float f = l > 0.f || l != l ? ic / l : 0.f;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t d = 32 * i + 8 * k + 4 * hi;
                if (d < dh) store4(op + d, oa[i][4 * k] * f, oa[i][4 * k + 1] * f, oa[i][4 * k + 2] * f, oa[i][4 * k + 3] * f);
            }
    } else {
        if (tid == 0) a.unit[cut] = ChunkUnit{sp ? 0u : parts, s.r0, nrow, qt, h, c.hkv, {0, 0}};
        if (r >= nrow) return;
        const uint64_t at = (uint64_t)cut * CT + 32 * wave + n;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t d = 32 * i + 8 * k + 4 * hi;
                if (d < dh) *(sh_f4v *)&a.part[at * dh + d] = sh_f4v{oa[i][4 * k], oa[i][4 * k + 1], oa[i][4 * k + 2], oa[i][4 * k + 3]} * ic;
            }
        if (hi == 0) { a.ml[at * 2] = mx; a.ml[at * 2 + 1] = l; }
    }
}

// The parts of a cut item, in order: its first unit, the others follow `step` places apart, all among the launch's `cuts`. A block takes every gridDim.x-th unit, and
// of its rows the blockIdx.y-th share.
__global__ __launch_bounds__(256) void k_kv_chunk_join(AttnArgs a) {
    const uint32_t cuts = (uint32_t)a.meta[0].x, dh = a.c.dh, qn = dh / 4, share = CT / gridDim.y;
    for (uint32_t cut = blockIdx.x; cut < cuts; cut += gridDim.x) {
        const ChunkUnit u = a.unit[cut];
        if (!u.parts || cut + (u.parts - 1) * u.step >= cuts) continue;
        for (uint32_t e = threadIdx.x; e < share * qn; e += 256) {
            const uint32_t row = blockIdx.y * share + e / qn, d = 4 * (e % qn), r = u.qt * CT + row;
            if (r >= u.nrow) break;
            float M = LOWEST, l = 0.f;
            sh_f4v o = {0.f, 0.f, 0.f, 0.f};
            for (uint32_t i = 0; i < u.parts; ++i) {
                const uint64_t at = (uint64_t)(cut + i * u.step) * CT + row;
                const float m = a.ml[at * 2], s = a.ml[at * 2 + 1];
                const sh_f4v v = *(const sh_f4v *)&a.part[at * dh + d];
                const float mn = fmaxf(M, m), f = sh_fast_exp2(M - mn), g = sh_fast_exp2(m - mn);
                o = o * f + v * g;
                l = l * f + s * g;
                M = mn;
            }
            const float f = l > 0.f || l != l ? 1.f / l : 0.f;
            const uint32_t qi = r / a.grp, qh = u.h * a.grp + (r - qi * a.grp);
            store4(a.o + (uint64_t)(u.r0 + qi) * a.ldo + (uint64_t)qh * dh + d, o[0] * f, o[1] * f, o[2] * f, o[3] * f);
        }
    }
}

uint32_t part_rows(uint32_t max_q, uint32_t grp) { return (uint32_t)std::min<uint64_t>(QT, (uint64_t)max_q * grp); }

template <int DP, int DH, bool FP8, int NW, bool MANY>
bool launch_attn_many(const AttnArgs &a, hipStream_t st) {
    static bool set = false;
    const uint32_t lds = 2 * NW * a.prow * DP * 4;
    if (!set) {
        if (!sh_hip_ok(hipFuncSetAttribute((const void *)k_kv_attn<DP, DH, FP8, NW, MANY>, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * NW * QT * DP * 4),
                       "sh_attention_kv hipFuncSetAttribute")) return false;
        set = true;
    }
    hipLaunchKernelGGL((k_kv_attn<DP, DH, FP8, NW, MANY>), dim3(a.groups), dim3(64 * NW), lds, st, a);
    if (!a.whole) hipLaunchKernelGGL(k_kv_join<DP>, dim3(a.groups, a.prow), dim3(256), 0, st, a);
    return sh_launch_ok("sh_attention_kv");
}
template <int DP, int DH, bool FP8, int NW>
bool launch_attn(AttnArgs a, uint32_t tiles, hipStream_t st) {
    const uint64_t rows = (uint64_t)a.max_q * a.grp;
    a.groups = GROUPS;
    a.lq = rows <= QT / 2 ? 3 : 4;
    if (a.B > 64 * NW) return launch_attn_many<DP, 0, FP8, NW, true>(a, st);
    a.wide = a.B > 64;
    a.whole = tiles <= WHOLE_TILES * NW;
    a.once = rows <= QT;
    // Nine rows and more in items of eight, for the precision of those, where that does not make more of them than workgroups (24 requests of
    // four drafts, 16 heads over 4: 13.2 us against 13.5): more would read keys twice that one item of sixteen reads once.
    if (a.whole && (uint64_t)a.B * a.c.hkv * ((rows + 7) / 8) <= GROUPS) {
        a.lq = 3;
        a.prow = std::min(a.prow, QT / 2);
    }
    return launch_attn_many<DP, DH, FP8, NW, false>(a, st);
}
template <bool FP8>
bool launch_attn_width(const AttnArgs &a, uint32_t tiles, hipStream_t st) {
    switch (a.c.dh) {
    case 32: return launch_attn<64, 32, FP8, 8>(a, tiles, st);
    case 64: return launch_attn<64, 64, FP8, 8>(a, tiles, st);
    case 80: return launch_attn<128, 80, FP8, 8>(a, tiles, st);
    case 96: return launch_attn<128, 96, FP8, 8>(a, tiles, st);
    case 128: return launch_attn<128, 128, FP8, 8>(a, tiles, st);
    case 256: return launch_attn<256, 256, FP8, 4>(a, tiles, st);
    }
    if (a.c.dh < 64) return launch_attn<64, 0, FP8, 8>(a, tiles, st);
    if (a.c.dh < 128) return launch_attn<128, 0, FP8, 8>(a, tiles, st);
    return launch_attn<256, 0, FP8, 4>(a, tiles, st);
}

template <bool FP8>
bool launch_chunk(const AttnArgs &a, uint32_t units, hipStream_t st) {
    if (a.c.dh <= 64) hipLaunchKernelGGL((k_kv_chunk<64, FP8>), dim3(units), dim3(256), 0, st, a);
    else if (a.c.dh <= 128) hipLaunchKernelGGL((k_kv_chunk<128, FP8>), dim3(units), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_kv_chunk<256, FP8>), dim3(units), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_kv_chunk_join, dim3(768, 8), dim3(256), 0, st, a);
    return sh_launch_ok("sh_attention_kv");
}

// More rows a request than CHUNK_ROWS: the kernel that shares converted keys between the rows of a workgroup. 16 requests of up to 8000
// keys, 32 heads over 8, rows by 16 (the other kernel) against by 128: 20 rows 45 against 70 us, 32 rows 47 against 74, 64 rows 77 against 79.
constexpr uint32_t CHUNK_ROWS = 64;
bool chunked(uint32_t max_q, uint32_t grp) { return (uint64_t)max_q * grp > CHUNK_ROWS; }

// Row tiles of a call of chunks, each request's last one short; and its cut units, at most.
uint64_t chunk_tiles(uint32_t B, uint32_t rows, uint32_t max_q, uint32_t grp) {
    return std::min<uint64_t>((uint64_t)B * (((uint64_t)max_q * grp + CT - 1) / CT), ((uint64_t)rows * grp + CT - 1) / CT + B);
}
uint64_t chunk_places(const sh_kv_cache &c, uint32_t B, uint32_t rows, uint32_t max_q, uint32_t grp, uint32_t ld) {
    const uint64_t nt = ((uint64_t)ld * c.bs + KT - 1) / KT, units = chunk_tiles(B, rows, max_q, grp) * c.hkv;
    return nt <= CUT_MIN ? 0 : std::min<uint64_t>(2 * CUT, units * ((nt + CUT_MIN - 1) / CUT_MIN));
}

}  // namespace

extern "C" {

uint64_t sh_attention_kv_ws_bytes(const sh_kv_cache *c, uint32_t B, uint32_t rows, uint32_t max_q, uint32_t H, uint32_t ld_table) {
    if (!c || !B || !rows || !max_q || !c->hkv || !H || !ld_table || !c->dh) return 0;
    max_q = std::min(max_q, rows);
    const uint32_t grp = H / c->hkv;
    const uint64_t prow = part_rows(max_q, grp), few = (uint64_t)GROUPS * (2 * prow * (c->dh + 2) * 4 + 32);
    if (!chunked(max_q, grp)) return few;
    // (never less than a call of fewer rows needs)
    return std::max(few, chunk_places(*c, B, rows, max_q, grp, ld_table) * ((uint64_t)CT * (c->dh + 2) * 4 + sizeof(ChunkUnit)) + 16);
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
    if ((uint64_t)std::min(max_q, rows) * grp >= (1ull << 31)) { sh_set_error(-1, "[sh_attention_kv] %u rows of %u heads", max_q, H); return -1; }
    a.sc = scale * 1.4426950408889634f;
    if (!(scale > 0.f && a.sc <= 3.4e38f)) { sh_set_error(-1, "[sh_attention_kv] scale %g must be positive and finite", (double)scale); return -1; }
    const uint64_t need = sh_attention_kv_ws_bytes(c, B, rows, max_q, H, ld_table);
    if (!ws || ws % 16) { sh_set_error(-1, "[sh_attention_kv] ws must be a 16-byte aligned address"); return -1; }
    if (ws_bytes < need) {
        sh_set_error(-2, "[sh_attention_kv] workspace of %llu B < %llu B", (unsigned long long)ws_bytes, (unsigned long long)need);
        return -2;
    }
    a.q = (const uint16_t *)q; a.o = (uint16_t *)o;
    a.table = (const int32_t *)table; a.kv_len = (const int32_t *)kv_len; a.row_start = (const int32_t *)row_start;
    a.ldq = ldq; a.ldo = ldo; a.ld = ld_table;
    a.B = B; a.rows = rows; a.max_q = std::min(max_q, rows); a.grp = grp; a.prow = part_rows(a.max_q, grp);
    a.window = window < ld_table * c->bs ? window : 0;               // (one that no key falls out of is none)
    a.groups = GROUPS;
    a.meta = (int4 *)ws;
    const hipStream_t st = sh_stream();
    if (chunked(a.max_q, grp)) {
        // units: the row tiles, and at most CUT parts more (a launch has fewer than 2^32 threads)
        const uint64_t tiles = chunk_tiles(B, rows, a.max_q, grp);
        if (tiles * c->hkv + CUT >= (1ull << 24)) { sh_set_error(-1, "[sh_attention_kv] %u rows of %u heads", rows, H); return -1; }
        const uint32_t units = (uint32_t)(tiles * c->hkv) + CUT;
        a.places = (uint32_t)chunk_places(*c, B, rows, a.max_q, grp, ld_table);
        a.unit = (ChunkUnit *)(ws + 16);
        a.part = (float *)(ws + 16 + a.places * sizeof(ChunkUnit));
        a.ml = a.part + (uint64_t)a.places * CT * c->dh;
        return (c->fmt == SH_FP8 ? launch_chunk<true>(a, units, st) : launch_chunk<false>(a, units, st)) ? 0 : SH_EHIP;
    }
    a.part = (float *)(ws + GROUPS * 32);
    a.ml = a.part + (uint64_t)GROUPS * 2 * a.prow * c->dh;
    uint64_t tiles = ((uint64_t)ld_table * c->bs + KT - 1) / KT + 1;                     // an item's, at most
    const uint64_t items = (uint64_t)c->hkv * (((uint64_t)a.max_q * grp + QT - 1) / QT);
    if (tiles * items >= (1ull << 32) / B) {                        // (tile counts of 32 bits)
        sh_set_error(-1, "[sh_attention_kv] %u requests of up to %llu tokens and %u heads", B, (unsigned long long)ld_table * c->bs, H);
        return -1;
    }
    if (a.window) tiles = std::min<uint64_t>(tiles, ((uint64_t)a.window + a.max_q) / KT + 2);
    const bool ok = c->fmt == SH_FP8 ? launch_attn_width<true>(a, (uint32_t)tiles, st) : launch_attn_width<false>(a, (uint32_t)tiles, st);
    return ok ? 0 : SH_EHIP;
}

}  // extern "C"
