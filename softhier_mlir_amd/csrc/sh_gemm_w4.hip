// Few rows times a weight of 4-bit codes (sh_gemm_w4).
//
// z[m][n] = sum_g s[g][n] sum_{k in g} x[m][k] (c[k][n] - z[g][n]): the inner sum on MFMA (v_mfma_f32_16x16x32_f16, 16 rows
// by 16 columns) with the integer c - z, which fp16 holds exactly; the scale multiplies the fp32 sum of its group. A word holds
// eight k of one column, which is one lane's operand of a step: lane (n, g) reads the word of column n and octet 4 step + g, so
// no operand is moved. In fp16 the number 1024 + c is 0x6400 | c: two codes of a word four apart are masked into a pair of
// halves at once, so the lane's k order is 0 4 1 5 2 6 3 7, and X's operand is put into the same order.
#include "sh_common.h"

namespace {

struct W4Args {
    const uint16_t *x, *scale;
    const uint32_t *w;
    const uint8_t *zero;
    uint16_t *z;
    uint32_t M, N, K, ugroup;          // ugroup: units of a group
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

// The eight codes of a word minus the zero: pairs (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ sh_h8 w4_half8(uint32_t w, sh_h2 z1024) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const sh_h2 v = __builtin_bit_cast(sh_h2, ((w >> (4 * i)) & 0x000F000Fu) | 0x64006400u) - z1024;
        r[i] = __builtin_bit_cast(uint32_t, v);
    }
    return __builtin_bit_cast(sh_h8, make_uint4(r[0], r[1], r[2], r[3]));
}
// Eight consecutive halves in that order.
__device__ __forceinline__ sh_h8 x_order(uint4 v) {
    return __builtin_bit_cast(sh_h8, make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                                                __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)));
}

__device__ __forceinline__ float gelu(float x) {          // x / (1 + 2^{x (k0 + k1 x^2)}), fp32
    return x * sh_fast_rcp(1.f + sh_fast_exp2(x * fmaf(SH_GELU_K1 * x, x, SH_GELU_K0)));
}

// A workgroup of NW waves: 16 CW columns (lane n has CW consecutive ones), 16 MT rows; wave i takes the units (32 SU values
// of k, all of one group) i, i + NW, ..., the next one's words in flight while it multiplies; the waves' sums are added in LDS in wave
// order. Columns and octets past the end are read from the last ones: their products are dropped or meet zeros of x.
template <int MT, int CW, int NW, int SU>
__global__ __launch_bounds__(64 * NW) void k_w4(W4Args a) {
    constexpr uint32_t LC = 16 * CW + 1;
    constexpr bool PX = MT == 1;                                    // x's next operands too
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
    struct Ops { Run<CW> w[SU]; uint4 x[PX ? SU : 1][MT]; float sc[CW]; uint32_t zr; };
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
        const uint64_t gi = (uint64_t)(u / a.ugroup) * a.lds + col;
        ld_scales<CW>(a.scale + gi, o.sc);
        o.zr = a.zero ? ld_zeros<CW>(a.zero + gi) : 0x08080808u;
    };
    const auto multiply = [&](uint32_t u, Ops &o) {
        uint4 x[SU][MT];
#pragma unroll
        for (int s = 0; s < SU; ++s)
            if constexpr (PX) x[s][0] = o.x[s][0]; else load_x(u, s, x[s]);
        sh_h2 z[CW];
#pragma unroll
        for (int j = 0; j < CW; ++j) {
            const uint32_t zz = 0x6400u | ((o.zr >> (8 * j)) & 15u);                     // the half 1024 + zero
            z[j] = __builtin_bit_cast(sh_h2, zz | zz << 16);
        }
        sh_f4v p[MT][CW];
        const bool tail = (u + 1) * 4 * SU > oct;
#pragma unroll
        for (int s = 0; s < SU; ++s) {
            sh_h8 wf[CW];
#pragma unroll
            for (int j = 0; j < CW; ++j) wf[j] = w4_half8(o.w[s].w[j], z[j]);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (tail && back(u, s)) x[s][i] = make_uint4(0, 0, 0, 0);
                const sh_h8 xf = x_order(x[s][i]);
#pragma unroll
                for (int j = 0; j < CW; ++j)
                    p[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf, wf[j], s ? p[i][j] : sh_f4v{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < CW; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(o.sc[j], p[i][j][e], acc[i][j][e]);
    };
    Ops o0, o1;
    uint32_t u = wave;
    if (u < units) load(u, o0);
    while (u < units) {
        if (u + NW < units) load(u + NW, o1);
        multiply(u, o0);
        u += NW;
        if (u >= units) break;
        if (u + NW < units) load(u + NW, o0);
        multiply(u, o1);
        u += NW;
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
        if (a.act == SH_ACT_GELU) v = gelu(v);
        uint16_t hz = sh_dev_f2h_rr(v);
        if (a.res) hz = sh_dev_f2h_rr(sh_dev_h2f(hz) + sh_dev_h2f(a.res[m * a.ldr + nn]));
        a.z[m * a.ldz + nn] = hz;
    }
}

template <int MT, int CW, int SU>
bool launch_w4(const W4Args &a, hipStream_t st) {
    constexpr uint32_t NW = 8, most = NW * 16 * MT * (16 * CW + 1) * 4;
    static bool set = false;
    if (!set && most > 65536) {
        if (!sh_hip_ok(hipFuncSetAttribute((const void *)k_w4<MT, CW, NW, SU>, hipFuncAttributeMaxDynamicSharedMemorySize, most),
                       "sh_gemm_w4 hipFuncSetAttribute")) return false;
        set = true;
    }
    const uint32_t lds = NW * (a.M < 16 * MT ? a.M : 16 * MT) * (16 * CW + 1) * 4;
    hipLaunchKernelGGL((k_w4<MT, CW, NW, SU>), dim3(sh_cdiv(a.N, 16 * CW), sh_cdiv(a.M, 16 * MT)), dim3(64 * NW), lds, st, a);
    return sh_launch_ok("sh_gemm_w4");
}
template <int SU>
bool launch_w4_tile(const W4Args &a, hipStream_t st) {
    const uint32_t mt = sh_cdiv(a.M, 16);
    const auto fills = [&](uint32_t m, uint32_t c) { return sh_cdiv(a.N, 16 * c) * sh_cdiv(mt, m) >= 192; };
    if (a.N < 4) return launch_w4<1, 1, SU>(a, st);
    if (fills(1, 4)) return launch_w4<1, 4, SU>(a, st);
    if (fills(1, 2)) return launch_w4<1, 2, SU>(a, st);
    return launch_w4<1, 1, SU>(a, st);
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
    if (M > (1u << 21) || N > (1u << 30)) { sh_set_error(-1, "[sh_gemm_w4] M=%u N=%u too large", M, N); return -1; }
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
    W4Args a{(const uint16_t *)x, (const uint16_t *)scale, (const uint32_t *)w, (const uint8_t *)zero, (uint16_t *)z, M, N, K, 0,
             ldx, ldw, lds, ldz, 0, nullptr, nullptr, 0, 0};
    if (epi) {
        a.bias = (const void *)epi->bias; a.bias_fp32 = epi->bias_fmt == SH_BIAS_FP32;
        a.act = epi->act;
        a.res = (const uint16_t *)epi->residual; a.ldr = epi->ldr;
    }
    const hipStream_t st = sh_stream();
    bool ok;
    if (group % 128 == 0) { a.ugroup = group / 128; ok = launch_w4_tile<4>(a, st); }
    else if (group % 64 == 0) { a.ugroup = group / 64; ok = launch_w4_tile<2>(a, st); }
    else { a.ugroup = group / 32; ok = launch_w4_tile<1>(a, st); }
    return ok ? 0 : SH_EHIP;
}
