// Few rows times a weight of 4-bit codes (sh_gemm_w4).
//
// z[m][n] = sum_g s[g][n] (sum_{k in g} x[m][k] c[k][n] - z[g][n] sum_{k in g} x[m][k]): both inner sums on MFMA
// (v_mfma_f32_16x16x32_f16, 16 rows by 16 columns, the second against ones), the scale and the zero applied to the fp32 sums.
// A word holds eight k of one column, which is one lane's operand of a step: lane (n, g) reads the word of column n and octet
// 4 step + g, so no operand is moved. A code in the low four bits of a half is the subnormal c 2^-24, which the matrix pipe multiplies
// exactly, and 16 times that four bits higher: two codes, eight k apart in the word's halves, are masked out at once, and
// only every second pair needs a shift: 5 vector instructions for 8 codes, 11 where they are made numbers 1024 + c and the zero is taken off
// each (one row of 4096 x 14336: 8.2 us, 3.7 TB/s, against 10.7 before that). The pairs are the k (0, 4) and (2, 6), and (1, 5) and (3, 7) 16 times as large: of
// two steps' words the former make one operand, the latter another with a sum of its own, and x's are put into the same order.
#include "sh_common.h"
#include <algorithm>

namespace {

struct W4Args {
    const uint16_t *x, *scale;
    const uint32_t *w;
    const uint8_t *zero;
    uint16_t *z;
    uint32_t M, N, K, groups, per;     // per: (GS steps) of a group
    uint64_t ldx, ldw, lds, ldz, ldr;
    const void *bias;
    const uint16_t *res;
    uint32_t bias_fp32, act;
};

// CW consecutive words (halves, bytes) at the alignment of one.
template <int CW> struct Run { uint32_t w[CW]; };
template <int CW>
__device__ __forceinline__ Run<CW> ld_words(const uint32_t *p) {
    Run<CW> r;
    if constexpr (CW == 4) {
        typedef sh_u4v u4 __attribute__((aligned(4)));
        const sh_u4v v = *(const u4 *)p;
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else if constexpr (CW == 2) {
        typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(4)));
        const u2 v = *(const u2 *)p;
        r.w[0] = v.x; r.w[1] = v.y;
    } else r.w[0] = *p;
    return r;
}
template <int CW>
__device__ __forceinline__ void ld_scales(const uint16_t *p, float (&s)[CW]) {
    if constexpr (CW == 4) {
        const sh_u2v_a2 v = *(const sh_u2v_a2 *)p;
        s[0] = sh_dev_h2f((uint16_t)v.x); s[1] = sh_dev_h2f((uint16_t)(v.x >> 16));
        s[2] = sh_dev_h2f((uint16_t)v.y); s[3] = sh_dev_h2f((uint16_t)(v.y >> 16));
    } else if constexpr (CW == 2) {
        const uint32_t v = *(const sh_u1_a2 *)p;
        s[0] = sh_dev_h2f((uint16_t)v); s[1] = sh_dev_h2f((uint16_t)(v >> 16));
    } else s[0] = sh_dev_h2f(*p);
}
template <int CW>
__device__ __forceinline__ uint32_t ld_zeros(const uint8_t *p) {
    if constexpr (CW == 4) { typedef uint32_t u __attribute__((aligned(1))); return *(const u *)p; }
    else if constexpr (CW == 2) { typedef uint16_t u __attribute__((aligned(1))); return *(const u *)p; }
    else return *p;
}

// Two words' codes of k 0, 4, 2, 6 as c 2^-24, and of k 1, 5, 3, 7 as c 2^-20.
__device__ __forceinline__ sh_h8 codes_lo(uint32_t a, uint32_t b) {
    constexpr uint32_t m = 0x000F000Fu;
    return __builtin_bit_cast(sh_h8, make_uint4(a & m, (a >> 8) & m, b & m, (b >> 8) & m));
}
__device__ __forceinline__ sh_h8 codes_hi(uint32_t a, uint32_t b) {
    constexpr uint32_t m = 0x00F000F0u;
    return __builtin_bit_cast(sh_h8, make_uint4(a & m, (a >> 8) & m, b & m, (b >> 8) & m));
}
// One word's codes of k 0, 4, 1, 5, 2, 6, 3, 7 as c 2^-20.
__device__ __forceinline__ sh_h8 codes_one(uint32_t a) {
    constexpr uint32_t m = 0x00F000F0u;
    return __builtin_bit_cast(sh_h8, make_uint4((a << 4) & m, a & m, (a >> 4) & m, (a >> 8) & m));
}
// Eight consecutive halves: k 0, 4 / 1, 5 / 2, 6 / 3, 7.
struct XPairs { uint32_t p04, p15, p26, p37; };
__device__ __forceinline__ XPairs x_pairs(uint4 v) {
    return XPairs{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                  __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
}

// A workgroup of NW waves: 16 CW columns (lane n has CW consecutive ones), 16 MT rows; wave i takes the units (SU
// steps of 32 k) i, i + NW, ..., the next one's words in flight while it multiplies; the waves' sums are added in LDS in wave order. Every
// GS steps of a unit the sums are scaled: GS = 4, 2, 1 for groups that are multiples of 128, 64, 32. Columns and octets past the end
// are read from the last ones: their products are dropped or meet zeros of x.
template <int MT, int CW, int NW, int GS, int SU>
__global__ __launch_bounds__(64 * NW) void k_w4(W4Args a) {
    constexpr uint32_t LC = 16 * CW + 1;
    constexpr int NG = SU / GS;
    constexpr bool PX = MT * CW <= 4;                               // x's next operands too
    extern __shared__ float s_z[];                                  // [NW][rows][LC]
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const uint32_t col0 = blockIdx.x * 16 * CW, m0 = blockIdx.y * 16 * MT, nrow = min(a.M - m0, 16u * MT);
    const uint32_t col = min(col0 + CW * n, a.N - CW);
    const uint32_t oct = a.K / 8, units = (oct + 4 * SU - 1) / (4 * SU);
    const uint64_t ldw = a.ldw;
    const uint32_t *wp = a.w + g * ldw + col;
    const uint16_t *xr[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xr[i] = a.x + min(m0 + 16 * i + n, a.M - 1) * a.ldx + 8 * g;
    sh_f4v acc[MT][CW];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < CW; ++j) acc[i][j] = sh_f4v{0.f, 0.f, 0.f, 0.f};
    struct Ops { Run<CW> w[SU]; uint4 x[PX ? SU : 1][MT]; float sc[NG][CW]; uint32_t zr[NG]; };
    // octets past K: the last one again
    const auto back = [&](uint32_t u, int s) { const uint32_t o = (u * SU + s) * 4 + g; return o < oct ? 0u : o - (oct - 1); };
    const auto load_x = [&](uint32_t u, int s, uint4 (&x)[MT]) {
#pragma unroll
        for (int i = 0; i < MT; ++i) x[i] = sh_ld16_any(xr[i] + (uint64_t)(u * SU + s) * 32 - 8 * back(u, s));
    };
    const auto load = [&](uint32_t u, Ops &o) {
        const uint32_t *p = wp + (uint64_t)u * (4 * SU) * ldw;
        if ((u + 1) * 4 * SU <= oct) {
#pragma unroll
            for (int s = 0; s < SU; ++s) o.w[s] = ld_words<CW>(p + s * 4 * ldw);
        } else {
#pragma unroll
            for (int s = 0; s < SU; ++s) o.w[s] = ld_words<CW>(p + s * 4 * ldw - back(u, s) * ldw);
        }
        if constexpr (PX)
#pragma unroll
            for (int s = 0; s < SU; ++s) load_x(u, s, o.x[s]);
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            const uint64_t gi = (uint64_t)min((u * NG + k) / a.per, a.groups - 1) * a.lds + col;
            ld_scales<CW>(a.scale + gi, o.sc[k]);
            o.zr[k] = ld_zeros<CW>(a.zero ? a.zero + gi : (const uint8_t *)(a.scale + gi));       // (read either way: see below)
        }
    };
    const auto multiply = [&](uint32_t u, Ops &o) {
        uint4 x[SU][MT];
#pragma unroll
        for (int s = 0; s < SU; ++s)
            if constexpr (PX) {
#pragma unroll
                for (int i = 0; i < MT; ++i) x[s][i] = o.x[s][i];
            } else load_x(u, s, x[s]);
        const bool tail = (u + 1) * 4 * SU > oct;
        if (tail)
#pragma unroll
            for (int s = 0; s < SU; ++s)
                if (back(u, s))
#pragma unroll
                    for (int i = 0; i < MT; ++i) x[s][i] = make_uint4(0, 0, 0, 0);
        const sh_f4v zero = {0.f, 0.f, 0.f, 0.f};
        const sh_h8 ones = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            sh_f4v lo[MT][CW], hi[MT][CW], xs[MT];                  // sums of x c 2^-24, of x c 2^-20, of x
#pragma unroll
            for (int i = 0; i < MT; ++i) xs[i] = zero;
            if constexpr (GS == 1) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const XPairs q = x_pairs(x[k][i]);
                    const sh_h8 xf = __builtin_bit_cast(sh_h8, make_uint4(q.p04, q.p15, q.p26, q.p37));
                    xs[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf, ones, zero, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < CW; ++j) hi[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf, codes_one(o.w[k].w[j]), zero, 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int s = k * GS; s < (k + 1) * GS; s += 2) {
                    sh_h8 cl[CW], ch[CW];
#pragma unroll
                    for (int j = 0; j < CW; ++j) { cl[j] = codes_lo(o.w[s].w[j], o.w[s + 1].w[j]); ch[j] = codes_hi(o.w[s].w[j], o.w[s + 1].w[j]); }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const XPairs p = x_pairs(x[s][i]), q = x_pairs(x[s + 1][i]);
                        const sh_h8 xl = __builtin_bit_cast(sh_h8, make_uint4(p.p04, p.p26, q.p04, q.p26)),
                                    xh = __builtin_bit_cast(sh_h8, make_uint4(p.p15, p.p37, q.p15, q.p37));
                        xs[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, ones, xs[i], 0, 0, 0);
                        xs[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, ones, xs[i], 0, 0, 0);
#pragma unroll
                        for (int j = 0; j < CW; ++j) {
                            lo[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, cl[j], s > k * GS ? lo[i][j] : zero, 0, 0, 0);
                            hi[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, ch[j], s > k * GS ? hi[i][j] : zero, 0, 0, 0);
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                const float sc = o.sc[k][j], sz = -sc * (a.zero ? (float)((o.zr[k] >> (8 * j)) & 15u) : 8.f), s24 = sc * 0x1p24f, s20 = sc * 0x1p20f;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float t = fmaf(xs[i][e], sz, acc[i][j][e]);
                        if constexpr (GS > 1) t = fmaf(lo[i][j][e], s24, t);
                        acc[i][j][e] = fmaf(hi[i][j][e], s20, t);
                    }
            }
        }
    };
    // (The next loads are made without a condition, behind the last unit of it again: under one the compiler would wait for all of
    // them before each product.)
    Ops o0, o1;
    uint32_t u = wave;
    if (u < units) {
        load(u, o0);
        for (;;) {
            uint32_t v = u + NW;
            load(v < units ? v : u, o1);
            multiply(u, o0);
            u = v;
            if (u >= units) break;
            v = u + NW;
            load(v < units ? v : u, o0);
            multiply(u, o1);
            u = v;
            if (u >= units) break;
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t r = 16 * i + 4 * g + e;
            if (r < nrow)
#pragma unroll
                for (int j = 0; j < CW; ++j)
                    if (col + j >= col0) s_z[(wave * nrow + r) * LC + (col + j - col0)] = acc[i][j][e];
        }
    __syncthreads();
    const uint32_t ncol = min(a.N - col0, 16u * CW);
    for (uint32_t i = threadIdx.x; i < nrow * 16 * CW; i += 64 * NW) {
        const uint32_t r = i / (16 * CW), c = i % (16 * CW), m = m0 + r, nn = col0 + c;
        if (c >= ncol) continue;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < NW; ++k) v += s_z[(k * nrow + r) * LC + c];
        if (a.bias) v += a.bias_fp32 ? ((const float *)a.bias)[nn] : sh_dev_h2f(((const uint16_t *)a.bias)[nn]);
        if (a.act == SH_ACT_GELU) v = sh_gelu_f32(v);
        uint16_t hz = sh_dev_f2h_rr(v);
        if (a.res) hz = sh_dev_f2h_rr(sh_dev_h2f(hz) + sh_dev_h2f(a.res[m * a.ldr + nn]));
        a.z[m * a.ldz + nn] = hz;
    }
}

template <int MT, int CW, int GS, int SU, uint32_t NW = 8>
bool launch_w4(const W4Args &a, hipStream_t st) {
    constexpr uint32_t most = NW * 16 * MT * (16 * CW + 1) * 4;
    static bool set = false;
    if (!set && most > 65536) {
        if (!sh_hip_ok(hipFuncSetAttribute((const void *)k_w4<MT, CW, NW, GS, SU>, hipFuncAttributeMaxDynamicSharedMemorySize, most),
                       "sh_gemm_w4 hipFuncSetAttribute")) return false;
        set = true;
    }
    const uint32_t lds = NW * (a.M < 16 * MT ? a.M : 16 * MT) * (16 * CW + 1) * 4;
    hipLaunchKernelGGL((k_w4<MT, CW, NW, GS, SU>), dim3(sh_cdiv(a.N, 16 * CW), sh_cdiv(a.M, 16 * MT)), dim3(64 * NW), lds, st, a);
    return sh_launch_ok("sh_gemm_w4");
}
// The tile with the least rounds of workgroups over the 256 CUs times the time of one, counted as one workgroup a CU (which is what the
// registers of the 64-column tiles allow; of the 16- and 32-column ones two fit): wider columns convert a word once for every 16 rows
// and read x once for every 16 CW columns, narrower ones make more workgroups. The times are those of a round at K = 4096 in groups
// of 128 (1 x 64 columns 7.0 us, x 32 5.2, x 16 4.5; 32 rows x 64 columns 11.5). Measured: 50 rows, K = 8192,
// 4096 columns (256 workgroups of 16 x 64) 15.3 us against 20.5 for 32 x 32; 64 rows, K = 4096, 4160 columns in 32 x 64 13.3 against 18.0
// in tiles of 16 rows, in groups of 32 15.2 against 23.3.
template <int GS, int SU>
bool launch_w4_tile(const W4Args &a, hipStream_t st) {
    const uint64_t mt = sh_cdiv(a.M, 16);
    const auto cost = [&](uint64_t m, uint32_t c, uint64_t t) { return a.N < c ? ~0ull : ((sh_cdiv(a.N, 16 * c) * ((mt + m - 1) / m) + 255) / 256) * t; };
    // A long chain of units over few columns: sixteen waves share it (by N and K alone, so that a row's bits do not depend on M). With eight
    // and with sixteen, 1, 16 and 64 rows: 12248 x 700 12.0 / 14.5 / 15.0 us against 10.3 / 15.5 / 15.9, 16384 x 256 11.5 / 18.6 / 18.9
    // against 10.3 / 19.4 / 20.0: a row or few gain what the longer sum over the waves costs many. At 8192 x 1024 they gain less than
    // that (7.0 / 11.0 / 11.1 against 6.6 / 12.2 / 12.4), at 4096 x 720 nothing (4.7 / 7.0 / 7.5 against 4.6 / 8.0 / 8.7), and more columns leave
    // workgroups of sixteen waves that do not fit at once (64 rows, 16264 x 1055 20.9 against 36.4).
    if constexpr (SU == 4)
        if (a.K > 8192 && a.N <= 1024) return launch_w4<1, 1, GS, SU, 16>(a, st);
    const uint64_t c24 = mt > 1 ? cost(2, 4, 115) : ~0ull, c14 = cost(1, 4, 70), c12 = cost(1, 2, 52), c11 = cost(1, 1, 45);
    const uint64_t best = std::min(std::min(c24, c14), std::min(c12, c11));
    if (best == c11) return launch_w4<1, 1, GS, SU>(a, st);
    if (best == c12) return launch_w4<1, 2, GS, SU>(a, st);
    if (best == c14) return launch_w4<1, 4, GS, SU>(a, st);
    return launch_w4<2, 4, GS, SU>(a, st);
}

// Units of 128 k keep the most words in flight (one row of 4096 x 14336, groups of 64: 10.9 us against 12.1 in units of 64); with
// fewer than eight of them (K < 1024) units of a group's own steps use every wave (one row of 720 x 2048, groups of 32: 3.6 against 4.1).
template <int GS>
bool launch_w4_unit(W4Args a, uint32_t group, hipStream_t st) {
    a.per = group / (32 * GS);
    return a.K < 1024 ? launch_w4_tile<GS, GS>(a, st) : launch_w4_tile<GS, 4>(a, st);
}

}  // namespace

extern "C" int sh_gemm_w4(uint64_t x, uint64_t w, uint64_t scale, uint64_t zero, uint64_t z, uint32_t M, uint32_t N, uint32_t K, uint32_t group,
                          uint32_t ldx, uint32_t ldw, uint32_t lds, uint32_t ldz, const sh_gemm_epi *epi) {
    if (!M || !N) return 0;
    if (!x || !w || !scale || !z) { sh_set_error(-1, "[sh_gemm_w4] NULL tensor address"); return -1; }
    if (!K || K % 8 || !group || group % 32) { sh_set_error(-1, "[sh_gemm_w4] K %u (a multiple of 8), group %u (a multiple of 32)", K, group); return -1; }
    if (ldx < K || ldw < N || lds < N || ldz < N) {
        sh_set_error(-1, "[sh_gemm_w4] leading dims %u %u %u %u for %ux%ux%u", ldx, ldw, lds, ldz, M, N, K);
        return -1;
    }
    if ((x | scale | z) % 2 || w % 4) { sh_set_error(-1, "[sh_gemm_w4] words must be 4-byte aligned, halves 2-byte aligned"); return -1; }
    if (M > (1u << 19) || N > (1u << 26)) { sh_set_error(-1, "[sh_gemm_w4] M=%u N=%u too large", M, N); return -1; }
    if (epi) {
        if (epi->act > SH_ACT_GELU) { sh_set_error(-1, "[sh_gemm_w4] unknown act %u", epi->act); return -1; }
        if (epi->bias && (epi->bias_fmt > SH_BIAS_FP32 || epi->bias % (epi->bias_fmt == SH_BIAS_FP32 ? 4 : 2))) {
            sh_set_error(-1, "[sh_gemm_w4] bias format %u or its alignment", epi->bias_fmt);
            return -1;
        }
        if (epi->residual && (epi->ldr < N || epi->residual % 2)) { sh_set_error(-1, "[sh_gemm_w4] ldr %u < N %u, or alignment", epi->ldr, N); return -1; }
        if (epi->splits > 1 || epi->ln_stats || epi->ln_c || epi->stats_out || epi->ln_parts) {
            sh_set_error(-1, "[sh_gemm_w4] no K split, LayerNorm fold or row partials");
            return -1;
        }
    }
    W4Args a{(const uint16_t *)x, (const uint16_t *)scale, (const uint32_t *)w, (const uint8_t *)zero, (uint16_t *)z, M, N, K, (K - 1) / group + 1, 0,
             ldx, ldw, lds, ldz, 0, nullptr, nullptr, 0, 0};
    if (epi) {
        a.bias = (const void *)epi->bias; a.bias_fp32 = epi->bias_fmt == SH_BIAS_FP32;
        a.act = epi->act;
        a.res = (const uint16_t *)epi->residual; a.ldr = epi->ldr;
    }
    const hipStream_t st = sh_stream();
    bool ok;
    if (group % 128 == 0) ok = launch_w4_unit<4>(a, group, st);
    else if (group % 64 == 0) ok = launch_w4_unit<2>(a, group, st);
    else ok = launch_w4_unit<1>(a, group, st);
    return ok ? 0 : SH_EHIP;
}
