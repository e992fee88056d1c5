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

typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
template <int CW> struct Vec { typedef uint32_t W; };
template <> struct Vec<2> { typedef u2v W; };
template <> struct Vec<4> { typedef u4v W; };

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
// of k, all of one group) i, i + NW, ...; their sums are added in LDS in wave order.
template <int MT, int CW, int NW, int SU>
__global__ __launch_bounds__(64 * NW) void k_w4(W4Args a) {
    typedef typename Vec<CW>::W W;
    __shared__ float s_z[NW][16 * MT][16 * CW + 1];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const uint32_t col0 = blockIdx.x * 16 * CW, m0 = blockIdx.y * 16 * MT;
    const uint32_t col = CW == 1 ? min(col0 + n, a.N - 1) : min(col0 + CW * n, a.N - CW);
    const uint32_t oct = a.K / 8, units = (a.K + 32 * SU - 1) / (32 * SU);
    sh_f4v acc[MT][CW];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < CW; ++j) acc[i][j] = sh_f4v{0.f, 0.f, 0.f, 0.f};
    for (uint32_t u = wave; u < units; u += NW) {
        W w[SU];
        uint4 x[SU][MT];
#pragma unroll
        for (int s = 0; s < SU; ++s) {
            const uint32_t o = (u * SU + s) * 4 + g, oc = min(o, oct - 1);
            w[s] = *(const W *)(a.w + oc * a.ldw + col);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                x[s][i] = sh_ld16_any(a.x + min(m0 + 16 * i + n, a.M - 1) * a.ldx + 8 * oc);
                if (o >= oct) x[s][i] = make_uint4(0, 0, 0, 0);
            }
        }
        const uint64_t gi = (uint64_t)(u / a.ugroup) * a.lds + col;
        float sc[CW];
        sh_h2 z[CW];
#pragma unroll
        for (int j = 0; j < CW; ++j) {
            sc[j] = sh_dev_h2f(a.scale[gi + j]);
            const _Float16 zz = (_Float16)(float)(1024 + (a.zero ? (a.zero[gi + j] & 15) : 8));
            z[j] = sh_h2{zz, zz};
        }
        sh_f4v p[MT][CW];
#pragma unroll
        for (int s = 0; s < SU; ++s) {
            sh_h8 xf[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) xf[i] = x_order(x[s][i]);
#pragma unroll
            for (int j = 0; j < CW; ++j) {
                uint32_t ww;
                if constexpr (CW == 1) ww = w[s]; else ww = w[s][j];
                const sh_h8 wf = w4_half8(ww, z[j]);
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    p[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[i], wf, s ? p[i][j] : sh_f4v{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < CW; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(sc[j], p[i][j][e], acc[i][j][e]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < CW; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s_z[wave][16 * i + 4 * g + e][CW * n + j] = acc[i][j][e];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 256 * MT * CW; i += 64 * NW) {
        const uint32_t r = i / (16 * CW), c = i % (16 * CW), m = m0 + r, nn = col0 + c;
        if (m >= a.M || nn >= a.N) continue;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < NW; ++k) v += s_z[k][r][c];
        if (a.bias) v += a.bias_fp32 ? ((const float *)a.bias)[nn] : sh_dev_h2f(((const uint16_t *)a.bias)[nn]);
        if (a.act == SH_ACT_GELU) v = gelu(v);
        uint16_t hz = sh_dev_f2h_rr(v);
        if (a.res) hz = sh_dev_f2h_rr(sh_dev_h2f(hz) + sh_dev_h2f(a.res[m * a.ldr + nn]));
        a.z[m * a.ldz + nn] = hz;
    }
}

template <int MT, int SU>
void launch_w4(const W4Args &a, bool vec, hipStream_t st) {
    hipLaunchKernelGGL((k_w4<MT, 1, 8, SU>), dim3(sh_cdiv(a.N, 16), sh_cdiv(a.M, 16 * MT)), dim3(512), 0, st, a);
}
template <int SU>
void launch_w4_rows(const W4Args &a, bool vec, hipStream_t st) {
    if (a.M <= 16) launch_w4<1, SU>(a, vec, st);
    else if (a.M <= 32) launch_w4<2, SU>(a, vec, st);
    else launch_w4<4, SU>(a, vec, st);
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
    const bool vec = false;
    if (group % 128 == 0) { a.ugroup = group / 128; launch_w4_rows<4>(a, vec, st); }
    else if (group % 64 == 0) { a.ugroup = group / 64; launch_w4_rows<2>(a, vec, st); }
    else { a.ugroup = group / 32; launch_w4_rows<1>(a, vec, st); }
    return sh_launch_ok("sh_gemm_w4") ? 0 : SH_EHIP;
}
