// Microscaled 4-bit floating point: rows to codes (sh_mx4_quant) and products of codes (sh_gemm_mx4, sh_gemm_mx4_f16).
//
// z[m][n] = sum_b 2^(sx[m][b] + sw[n][b]) sum_{k in b} x[m][k] w[n][k] over blocks b of 32 k: v_mfma_scale_f32_*_f8f6f4 takes the e2m1 codes
// and the scale bytes as they are stored. A lane's operand of a step is one block of one row (16 bytes), and one byte of a scale word
// that the instruction names, so no code is moved between lanes: of the 16 blocks that four steps of a 16 x 16 x 128 product take, lane (row, g) has the
// blocks 4 g .. 4 g + 3, in step j block 4 g + j, and their four scales in one aligned word. (Which blocks meet in a step does not
// matter, as long as both operands have the same.)
#include "sh_common.h"
#include <algorithm>
#include <type_traits>

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef uint16_t us2 __attribute__((ext_vector_type(2)));

constexpr int E2M1 = 4;                    // the instruction's number of the format
constexpr uint32_t ONES = 0x7F7F7F7Fu;     // four scales of 1

__device__ __forceinline__ v8i operand(sh_u4v c) { return v8i{(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0}; }
__device__ __forceinline__ us2 bits2(uint32_t w) { return __builtin_bit_cast(us2, w & 0x7FFF7FFFu); }     // a pair of halves without their signs

// The scale byte of a block whose largest |x| is the half `top`: amax = f 2^e with f in [0.5, 1), 6 = 0.75 2^3. 255 where it is not finite.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    const float amax = sh_dev_h2f((uint16_t)top);
    const int e = __builtin_amdgcn_frexp_expf(amax), p = top ? max(__builtin_amdgcn_frexp_mantf(amax) <= 0.75f ? e - 3 : e - 2, -32) : -32;
    return top >= 0x7C00u ? 255u : (uint32_t)(p + 127);
}
// Eight halves to eight codes, nearest, ties to even (|x| <= 6 scale).
__device__ __forceinline__ uint32_t codes8(uint4 v, float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(sh_h2, v.x), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(sh_h2, v.y), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(sh_h2, v.z), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(sh_h2, v.w), scale, 3);
}
__device__ __forceinline__ us2 top8(uint4 v) {
    return __builtin_elementwise_max(__builtin_elementwise_max(bits2(v.x), bits2(v.y)), __builtin_elementwise_max(bits2(v.z), bits2(v.w)));
}
// Halves [k, k + 8) of a row of K, zeros behind it.
__device__ __forceinline__ uint4 load8(const uint16_t *row, uint32_t k, uint32_t K) {
    if (k + 8 <= K) return sh_ld16_any(row + k);
    if (k >= K) return make_uint4(0, 0, 0, 0);
    if (K >= 8) return sh_ld8_row(row, k, K);
    uint32_t w[4] = {0, 0, 0, 0};
    for (uint32_t i = 0; i < K; ++i) w[i / 2] |= (uint32_t)row[i] << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- sh_mx4_quant -------------------------------------------------------------------------------------------------
struct QuantArgs {
    uint8_t *codes, *scales;
    const uint16_t *x;
    uint64_t ldc, lds, ldx, items;
    uint32_t cols, row0;
    ShDiv dch;                             // by a row's 16-byte pieces
};

// A lane has 8 columns, four lanes a block. Bound by HBM (8192 x 14336: 52 us, 5.7 TB/s), for a few rows by the launch (50 x 4096 4.8 us).
__global__ __launch_bounds__(256) void k_mx4_quant(QuantArgs a) {
    const uint32_t it = blockIdx.x * 256u + threadIdx.x;
    if (it >= a.items) return;
    const uint32_t r = sh_div(it, a.dch), c = it - r * a.dch.d;
    const uint64_t row = a.row0 + (uint64_t)r;
    const uint4 v = load8(a.x + row * a.ldx, 8 * c, a.cols);
    const us2 t = top8(v);
    float top = (float)max(t.x, t.y);                                          // (exact)
    top = fmaxf(top, sh_dpp<0xb1>(top, top));
    top = fmaxf(top, sh_dpp<0x4e>(top, top));
    const uint32_t e = scale_byte((uint32_t)top);
    const uint32_t w = e < 255u ? codes8(v, __uint_as_float(e << 23)) : 0u;
    *(uint32_t *)(a.codes + row * a.ldc + 4 * c) = w;
    if (!(c & 3)) a.scales[row * a.lds + c / 4] = (uint8_t)e;
}

// ---- products -----------------------------------------------------------------------------------------------------
struct MxArgs {
    const uint8_t *xc, *xs, *wc, *ws;
    const uint16_t *x;                     // fp16 rows in place of xc and xs
    uint16_t *z;
    uint32_t M, N, K, nb;
    uint64_t ldxc, ldxs, ldwc, ldws, ldx, ldz, ldr;
    const void *bias;
    const uint16_t *res;
    uint32_t bias_fp32, act;
};

__device__ __forceinline__ void store_one(const MxArgs &a, uint32_t m, uint32_t n, float v) {
    if (a.bias) v += a.bias_fp32 ? ((const float *)a.bias)[n] : sh_dev_h2f(((const uint16_t *)a.bias)[n]);
    if (a.act == SH_ACT_GELU) v = sh_gelu_f32(v);
    uint16_t h = sh_dev_f2h_rr(v);
    if (a.res) h = sh_dev_f2h_rr(sh_dev_h2f(h) + sh_dev_h2f(a.res[m * a.ldr + n]));
    a.z[m * a.ldz + n] = h;
}

// f(0), f(1), ..., f(N - 1) as compile-time numbers; and the part of them that falls to place E of P when they are spread evenly.
template <int N, int B = 0, typename F>
__device__ __forceinline__ void each(F f) {
    if constexpr (B < N) {
        f(std::integral_constant<int, B>{});
        each<N, B + 1>(f);
    }
}
template <int N, int P, typename E, typename F>
__device__ __forceinline__ void some(E, F f) {
    if constexpr (E::value < P) each<N * (E::value + 1) / P, N * E::value / P>(f);
}

__device__ __forceinline__ sh_u4v lds16(uint32_t addr) { return *(const __attribute__((address_space(3))) sh_u4v *)(uintptr_t)addr; }
__device__ __forceinline__ uint32_t lds4(uint32_t addr) { return *(const __attribute__((address_space(3))) uint32_t *)(uintptr_t)addr; }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// One global_load_lds_dword: each lane's word lands at lds_wave_base + 4 lane.
__device__ __forceinline__ void dma4_s(const void *base, uint32_t off, uint32_t lds_wave_base) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds_wave_base), "v"(off), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

constexpr int SU = 4;                      // steps of a unit of 512 k: four segments of 64 bytes of a row, four words of scales
// A row of halves as a lane's operands: block b0 + 4 g + j in step j, and the scales' word. WHOLE: all blocks of the unit are there.
template <bool WHOLE>
__device__ __forceinline__ uint32_t load_halves(const uint16_t *row, uint32_t b0, uint32_t g, uint32_t nb, uint32_t K, sh_u4v (&c)[SU]) {
    uint32_t s = 0;
    uint4 v[SU][4];
    const uint32_t k0 = 32 * (b0 + 4 * g), end = K - min(K, 8u);
    if (WHOLE || K >= 8)                                     // (no branch between the loads, what lies behind the row is put right below)
#pragma unroll
        for (int j = 0; j < SU; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t k = k0 + 32 * j + 8 * i;
                v[j][i] = sh_ld16_any(row + (WHOLE ? k : min(k, end)));
            }
    else
#pragma unroll
        for (int j = 0; j < SU; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j][i] = load8(row, k0 + 32 * j + 8 * i, K);
#pragma unroll
    for (int j = 0; j < SU; ++j) {
        if (!WHOLE && K >= 8 && k0 + 32 * j + 32 > K)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t k = k0 + 32 * j + 8 * i;
                if (k >= K) v[j][i] = make_uint4(0, 0, 0, 0);
                else if (k > end) v[j][i] = sh_fix8(v[j][i], k - end, 8 - (k - end));
            }
        if (!WHOLE && b0 + 4 * g + j >= nb) {
            c[j] = sh_u4v{0, 0, 0, 0};
            continue;
        }
        const us2 t = __builtin_elementwise_max(__builtin_elementwise_max(top8(v[j][0]), top8(v[j][1])), __builtin_elementwise_max(top8(v[j][2]), top8(v[j][3])));
        const uint32_t e = scale_byte(max(t.x, t.y));
        s |= e << (8 * j);
        const float f = __uint_as_float(e << 23);            // (255: infinity, whose codes are put right)
        c[j] = sh_u4v{codes8(v[j][0], f), codes8(v[j][1], f), codes8(v[j][2], f), codes8(v[j][3], f)};
        if (e == 255u) c[j] = sh_u4v{0, 0, 0, 0};
    }
    return s;
}

// Few rows: a workgroup has 16 CW columns and 16 MT rows of z; its waves take units of 512 k in turn, and their sums are added in LDS in wave order. A wave
// brings a unit's codes into LDS of its own by DMA, without a barrier: four lanes side by side read 64 bytes of a row, or its four words of scales, which
// change lanes afterwards. (Read straight into the operands' lanes, where neighbours are rows, each lane is an access of its own: 50 rows of 8192 x 4096 13.3 us, with
// DMAs 11.3; 64 of 16384 x 4096 25.5 and 15.2. With the scales alone read so, 20 of 16384 x 1024 9.2 us, 7.8 this way.) A workgroup begins at a unit of its own: where all begin
// with the same lines of x, they wait for each other's (50 rows 12.0 us, 9.2 so; 16 rows of 8192 x 4096 6.9 and 5.3). Seven waves would leave LDS for the scales too, and take
// a round more. In step j a lane has block 4 g + j. Behind the last block the codes are those of the last one again and both scales 2^-127.
template <int MT, int CW, int NW, bool F16>
struct Rows {
    static constexpr int GROUPS = CW + (F16 ? 0 : MT);                         // of 16 rows, of W and of x
    static constexpr uint32_t GROUP = SU * 1024, WAVE = GROUPS * GROUP, LC = 16 * CW + 1;
    static uint32_t lds(uint32_t nrow) { return std::max(NW * WAVE, NW * nrow * LC * 4); }
    static_assert(NW * WAVE <= 163840, "rows");
};
template <int MT, int CW, int NW, bool F16>
__global__ __launch_bounds__(64 * NW) void k_mx4_rows(MxArgs a) {
    using T = Rows<MT, CW, NW, F16>;
    constexpr uint32_t LC = T::LC;
    extern __shared__ __align__(128) uint8_t smem[];
    float *s_z = (float *)smem;                                                // [NW][rows][LC], after the products
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const uint32_t col0 = blockIdx.x * 16 * CW, m0 = blockIdx.y * 16 * MT, nrow = min(a.M - m0, 16u * MT);
    const uint32_t nb = a.nb, nd = (nb + 3) / 4, units = (nb + 4 * SU - 1) / (4 * SU);
    const uint32_t mine = sh_lds_addr(smem) + wave * T::WAVE;
    // DMAs: lane -> row, 16-byte chunk of a segment of 64; scales: lane -> row, word of the unit
    const uint32_t chunk = (lane & 3) ^ ((lane >> 3 ^ lane >> 5) & 3);
    const uint8_t *pc[T::GROUPS], *ps[T::GROUPS];
#pragma unroll
    for (int k = 0; k < T::GROUPS; ++k) {
        const uint32_t r = lane >> 2;
        if (k < CW) {
            pc[k] = a.wc + min(col0 + 16 * k + r, a.N - 1) * a.ldwc;
            ps[k] = a.ws + min(col0 + 16 * k + r, a.N - 1) * a.ldws;
        } else {
            pc[k] = a.xc + min(m0 + 16 * (k - CW) + r, a.M - 1) * a.ldxc;
            ps[k] = a.xs + min(m0 + 16 * (k - CW) + r, a.M - 1) * a.ldxs;
        }
    }
    uint32_t sc[T::GROUPS];
    const auto load = [&](uint32_t u) {
        const uint32_t b = 4 * (SU * u + g), left = b < nb ? nb - b : 0u, keep = left < 4 ? (1u << (8 * left)) - 1 : ~0u;
#pragma unroll
        for (int k = 0; k < T::GROUPS; ++k) sc[k] = *(const uint32_t *)(ps[k] + 4ull * min(SU * u + (lane & 3), nd - 1));
#pragma unroll
        for (int k = 0; k < T::GROUPS; ++k)
#pragma unroll
            for (int j = 0; j < SU; ++j) sh_lds_dma16(pc[k] + 16ull * min(4 * (SU * u + j) + chunk, nb - 1), mine + k * T::GROUP + j * 1024);
        return keep;
    };
    const auto scale = [&](int k, uint32_t keep) { return (int)(__builtin_amdgcn_ds_bpermute((int)(4 * n + g) * 4, (int)sc[k]) & keep); };
    const uint32_t code_at = g * 1024 + n * 64, swap = (n >> 1 ^ n >> 3) & 3;
    sh_f4v acc[CW][MT];
#pragma unroll
    for (int k = 0; k < CW; ++k)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[k][i] = sh_f4v{0.f, 0.f, 0.f, 0.f};
    const auto codes = [&](int k, sh_u4v (&c)[SU]) {
#pragma unroll
        for (int j = 0; j < SU; ++j) c[j] = lds16(mine + k * T::GROUP + code_at + 16 * (j ^ swap));
    };
    const uint32_t first = col0 / 64 % units;                                  // (by the column alone, whatever CW: a column's sums keep their order)
    for (uint32_t i = wave; i < units; i += NW) {
        const uint32_t u = i + first < units ? i + first : i + first - units, b0 = 4 * SU * u;
        sh_u4v x[MT][SU];
        int sx[MT];
        const uint32_t keep = load(u);
        // Halves are issued behind the codes' DMAs, and loads are counted off in order: the first wait for a half is one for all of the unit's codes, and
        // the conversion stands behind them. With few rows the lanes n repeat a row, and its conversion.
        if constexpr (F16)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const uint16_t *row = a.x + min(m0 + 16 * i + n, a.M - 1) * a.ldx;
                sx[i] = (int)(128 * SU * (u + 1) <= a.K ? load_halves<true>(row, b0, g, nb, a.K, x[i]) : load_halves<false>(row, b0, g, nb, a.K, x[i]));
            }
        sh_wait_vmcnt<0>();
        asm volatile("" ::: "memory");
        if constexpr (!F16)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                codes(CW + i, x[i]);
                sx[i] = scale(CW + i, keep);
            }
#pragma unroll
        for (int k = 0; k < CW; ++k) {
            sh_u4v w[SU];
            codes(k, w);
            const int sw = scale(k, keep);
#pragma unroll
            for (int i = 0; i < MT; ++i)
                each<SU>([&](auto j) {
                    constexpr int J = decltype(j)::value;
                    acc[k][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w[J]), operand(x[i][J]), acc[k][i], E2M1, E2M1, J, sw, J, sx[i]);
                });
        }
        sh_wait_lgkm0();                                                       // (the next unit's codes come into the same place)
        asm volatile("" ::: "memory");
    }
    __syncthreads();
    // lane (m, g): the columns 4 g .. 4 g + 3 of row m
#pragma unroll
    for (int i = 0; i < MT; ++i)
        if (16 * i + n < nrow)
#pragma unroll
            for (int k = 0; k < CW; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) s_z[(wave * nrow + 16 * i + n) * LC + 16 * k + 4 * g + e] = acc[k][i][e];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < nrow * 16 * CW; i += 64 * NW) {
        const uint32_t r = i / (16 * CW), c = i % (16 * CW);
        if (col0 + c >= a.N) continue;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < NW; ++k) v += s_z[(k * nrow + r) * LC + c];
        store_one(a, m0 + r, col0 + c, v);
    }
}

// Many rows. A workgroup has a BM x BN tile of z, a wave TM x TN blocks of 32 x 32 of it (W's rows are the instruction's rows, so a lane has one row
// of z and groups of four columns). Slices of 128 k (four blocks of a row: 64 bytes) go by DMA into a ring of four stages, three slices ahead; the scales of four
// slices (16 bytes of a row) into a ring of three. A slice is two steps of 64 k; a step's operands are read while the last step multiplies, and the barrier that frees
// a stage lies between the two, so that no wave meets it without products to issue. Chunk c of a row lies at c ^ ((row / 2 ^ row / 8 % 2) % 4) of its 64 bytes, so
// that neither eight nor sixteen lanes in a row meet in a bank (row / 2 % 4 alone: twice the conflicts). Behind the last block the codes are those of the last one again and both scales 2^-127: their product is 0 in fp32.
// Large problems are bound by power and by what the two waves of a SIMD wait: 8192^3, 290 to 300 us, 3.7 PFLOP/s at 1.78 GHz, matrix pipe busy 47 %; the pipe alone, fed
// from registers, gives 6.3 PFLOP/s of random codes and 9.7 of zeros. Eight waves share a 256 x 256 tile (four, with twice the registers each: 302 us); of the 73 us
// that a round of tiles takes there, 10 are its start and its end. One round of small tiles is bound by its start, its end and one workgroup of four waves a CU: 700 x 5000
// x 2880, 15.7 us, pipe busy 11 %. L2 bounds neither: a kernel of these DMAs alone gets 22 TB/s of whole lines, 17 to 19 of half lines and 14 of rows of 1440 bytes, every
// second half of which lies over two lines; the two take 7.6 (of 17) and 6.0 (of 14). 256 columns a slice in two stages, or a line of 128 bytes a row in four, were no faster.
template <int BM, int BN, int WGM, int WGN>
struct Tile {
    static constexpr int NW = WGM * WGN, TM = BM / WGM / 32, TN = BN / WGN / 32, NST = 4, ROWS = BM + BN;
    static constexpr int CPW = ROWS / 16 / NW;                                        // a wave's DMAs of a slice's codes (16 rows each)
    static constexpr int SG = ROWS / 64, SW = ROWS / 16;                              // DMAs of four slices' scales: one a wave (64 rows), or by words four (16 rows),
                                                                                      // one a slice; where there are fewer than waves, some are loaded twice
    static constexpr uint32_t CODE = ROWS * 64, SC = ROWS * 16, RING = NST * CODE, PITCH = BN * 4 + 16;
    static constexpr int PASSES = BM * PITCH <= 81920 ? 1 : 2;                        // of the sums through LDS
    static constexpr uint32_t STAGED = BM / PASSES * PITCH, LDS = RING + 3 * SC > STAGED ? RING + 3 * SC : STAGED;
    static_assert(ROWS % (16 * NW) == 0 && SG <= NW && SW <= 4 * NW && BN % 64 == 0 && TM % PASSES == 0 && BM % (32 * WGM) == 0 && BN % (32 * WGN) == 0 && LDS <= 163840, "tile");
};

template <int BM, int BN, int WGM, int WGN, int PER, bool A16>
__global__ __launch_bounds__(64 * WGM * WGN, PER) void k_mx4_tile(MxArgs a) {
    using T = Tile<BM, BN, WGM, WGN>;
    constexpr int NW = T::NW, TM = T::TM, TN = T::TN, NST = T::NST, CPW = T::CPW;
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t lds0 = sh_lds_addr(smem), sc0 = lds0 + T::RING;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % WGM, wn = wave / WGM;
    const uint32_t g = lane >> 5, r32 = lane & 31;
    // tiles in bands of eight of a column, a contiguous range of them for each XCD
    const uint32_t tm_all = (a.M + BM - 1) / BM, tn_all = (a.N + BN - 1) / BN, tiles = tm_all * tn_all;
    uint32_t id = blockIdx.x;
    {
        const uint32_t x = id & 7, per = tiles / 8, more = tiles % 8;
        id = x * per + min(x, more) + (id >> 3);
    }
    const uint32_t band = id / (8 * tn_all), in = id - band * 8 * tn_all, high = min(8u, tm_all - band * 8);
    const uint32_t m0 = (band * 8 + in % high) * BM, n0 = in / high * BN;
    const uint32_t nb = a.nb, nd = (nb + 3) / 4, n = nd;                               // slices
    const uint8_t *wc = a.wc + (uint64_t)n0 * a.ldwc, *xc = a.xc + (uint64_t)m0 * a.ldxc, *ws = a.ws + (uint64_t)n0 * a.ldws, *xs = a.xs + (uint64_t)m0 * a.ldxs;
    const uint32_t wlim = a.N - 1 - n0, xlim = a.M - 1 - m0;
    const uint32_t ldwc = (uint32_t)a.ldwc, ldxc = (uint32_t)a.ldxc, ldws = (uint32_t)a.ldws, ldxs = (uint32_t)a.ldxs;
    const uint32_t chunk = (lane & 3) ^ ((lane >> 3 ^ lane >> 5) & 3);
    uint32_t off[CPW];
#pragma unroll
    for (int i = 0; i < CPW; ++i) {
        const uint32_t first = (wave * CPW + i) * 16, row = first + (lane >> 2);
        off[i] = 16 * chunk + (first < BN ? min(row, wlim) * ldwc : min(row - BN, xlim) * ldxc);
    }
    // `part` of `parts` of a wave's DMAs
    const auto load_codes = [&](uint32_t u, int part = 0, int parts = 1) {
        const uint32_t slot = lds0 + (u % NST) * T::CODE;
        uint32_t back = 0;
        if (4 * u + 4 > nb && 4 * u + chunk >= nb) back = 16 * (4 * u + chunk + 1 - nb);
#pragma unroll
        for (int i = CPW * part / parts; i < CPW * (part + 1) / parts; ++i) {
            const uint32_t ins = wave * CPW + i;
            sh_lds_dma16_s((ins * 16 < BN ? wc : xc) + 64ull * u, off[i] - back, slot + ins * 1024);
        }
    };
    // Part `q` of the scales of slices 4 gr .. 4 gr + 3, of the last ones where there are none: rows of 16 bytes where these are aligned (A16), else words.
    uint32_t soff[A16 ? 1 : 4];
#pragma unroll
    for (int q = 0; q < (A16 ? 1 : 4); ++q) {
        const uint32_t row = A16 ? wave % T::SG * 64 + lane : (q * NW + wave) % T::SW * 16 + (lane >> 2);
        soff[q] = row < BN ? min(row, wlim) * ldws : min(row - BN, xlim) * ldxs;
    }
    const auto load_scales = [&](uint32_t gr, auto part) {
        constexpr int Q = decltype(part)::value;
        const uint32_t at = sc0 + gr % 3 * T::SC;
        if constexpr (!A16) {
            const uint32_t ins = (Q * NW + wave) % T::SW;
            dma4_s(ins * 16 < BN ? ws : xs, soff[Q] + 4 * min(4 * gr + (lane & 3), nd - 1), at + ins * 256);
        } else if constexpr (Q == 0) {
            const uint32_t ins = wave % T::SG;
            sh_lds_dma16_s((ins * 64 < BN ? ws : xs) + 16 * min(gr, (nd - 1) / 4), soff[0], at + ins * 1024);
        }
    };
    // What may be outstanding behind a slice that is waited for: two or three slices' codes, and by words the part of the scales that each slice brings behind
    // its codes (its own, still, is waited for). By 16 bytes a group's scales go behind one slice's codes in four, and none are counted.
    constexpr int W2 = 2 * CPW + (A16 ? 0 : 2), W3 = 3 * CPW + (A16 ? 0 : 3);
    const uint32_t lane_at = r32 * 64 + ((2 * g) ^ ((r32 >> 1 ^ (r32 >> 3 & 1)) & 3)) * 16;
    struct Ops { sh_u4v w[TN], x[TM]; };
    struct Scales { uint32_t w[TN], x[TM]; };
    // read i of a step's operands (w0, the x, the other w), and of a slice's scales
    const auto read = [&](uint32_t at, auto i, Ops &o) {
        constexpr int I = decltype(i)::value;
        if constexpr (I > 0 && I <= TM) o.x[I - 1] = lds16(at + BN * 64 + (wm * TM + I - 1) * 2048);
        else { constexpr int W = I ? I - TM : 0; o.w[W] = lds16(at + (wn * TN + W) * 2048); }
    };
    const auto read_scale = [&](uint32_t at, auto i, Scales &s) {
        constexpr int I = decltype(i)::value;
        if constexpr (I < TN) s.w[I] = lds4(at + (wn * TN + I) * 512);
        else s.x[I - TN] = lds4(at + BN * 16 + (wm * TM + I - TN) * 512);
    };
    const auto ops_at = [&](uint32_t t, int j) { return lds0 + (t % NST) * T::CODE + (lane_at ^ (16 * j)); };
    const auto scales_at = [&](uint32_t t) { return sc0 + t / 4 % 3 * T::SC + r32 * 16 + 4 * (t & 3); };
    const auto own_scales = [&](uint32_t t, Scales &s) {
        const uint32_t keep = 4 * t + 4 > nb ? (1u << (8 * (nb - 4 * t))) - 1 : ~0u;
#pragma unroll
        for (int i = 0; i < TN; ++i) s.w[i] = (s.w[i] & keep) >> (16 * g);
#pragma unroll
        for (int i = 0; i < TM; ++i) s.x[i] = (s.x[i] & keep) >> (16 * g);
    };
    struct Group { sh_u4v w[TN], x[TM]; };
    const auto read_group = [&](uint32_t at, auto i, Group &s) {
        constexpr int I = decltype(i)::value;
        if constexpr (I < TN) s.w[I] = lds16(at + (wn * TN + I) * 512);
        else s.x[I - TN] = lds16(at + BN * 16 + (wm * TM + I - TN) * 512);
    };
    const auto pick = [&](auto part, const Group &v, Scales &s) {
        constexpr int Q = decltype(part)::value;
        const auto word = [&](const sh_u4v &u) { return u[Q] >> (16 * g); };
#pragma unroll
        for (int i = 0; i < TN; ++i) s.w[i] = word(v.w[i]);
#pragma unroll
        for (int i = 0; i < TM; ++i) s.x[i] = word(v.x[i]);
    };
    sh_f16v acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int k = 0; k < TM; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][k][e] = 0.f;
    // A step's products, with `between(e)` before each: what it issues stays there (the compiler would put all reads first, and no product
    // is issued while LDS takes them).
    constexpr int P = TN * TM;
    const auto multiply = [&](auto j, const Ops &o, const Scales &s, auto between) {
        each<P>([&](auto e) {
            constexpr int E = decltype(e)::value, I = E / TM, K = E % TM;
            between(e);
            acc[I][K] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(o.w[I]), operand(o.x[K]), acc[I][K], E2M1, E2M1, decltype(j)::value, (int)s.w[I],
                                                                       decltype(j)::value, (int)s.x[K]);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    each<4>([&](auto q) { load_scales(0, q); });
    each<NST>([&](auto u) {
        if (decltype(u)::value < n) {
            load_codes(decltype(u)::value);
            load_scales(1, u);
        }
    });
    if (n >= NST) sh_wait_vmcnt<W3>();
    else sh_wait_vmcnt<0>();
    __syncthreads();
    constexpr int R = TN + TM, SPREAD = P > 1 ? P * 3 / 4 : 1;           // reads of a step, and the products that they are spread over
    Ops o0, o1;
    Scales s0, s1;
    {
        const uint32_t at = ops_at(0, 0);
        each<R>([&](auto i) { read(at, i, o0); });
    }
    // Between a slice's steps: the next slice has come, this one's operands are all in registers. (The barrier alone does not keep the compiler's
    // loads on their side; and a branch within a slice lets it move products past the barrier.)
    const auto turn = [&](auto waiting) {
        sh_wait_vmcnt<decltype(waiting)::value>();
        sh_wait_lgkm0();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    uint32_t t = 0;
    if (n >= 8) {                                            // four slices at a time, their scales in registers
        Group ga, gb;
        {
            const uint32_t at = sc0 + r32 * 16;
            each<R>([&](auto i) { read_group(at, i, ga); });
        }
        for (; t + 8 <= n; t += 4) {
            const uint32_t gat = sc0 + (t / 4 + 1) % 3 * T::SC + r32 * 16;
            each<4>([&](auto q) {
                constexpr int Q = decltype(q)::value;
                const uint32_t at1 = ops_at(Q, 1), at0 = ops_at(Q + 1, 0);
                pick(q, ga, s0);
                multiply(std::integral_constant<int, 0>{}, o0, s0, [&](auto e) {
                    some<R, SPREAD>(e, [&](auto i) {
                        read(at1, i, o1);
                        if constexpr (Q == 3) read_group(gat, i, gb);
                    });
                });
                turn(std::integral_constant<int, W2>{});
                multiply(std::integral_constant<int, 1>{}, o1, s0, [&](auto e) {
                    some<R, SPREAD>(e, [&](auto i) { read(at0, i, o0); });
                    load_codes(t + Q + NST, decltype(e)::value, P);
                    if constexpr (decltype(e)::value == P - 1) load_scales(t / 4 + 2, q);
                });
            });
            ga = gb;
        }
    }
    {
        const uint32_t at = scales_at(t);
        each<R>([&](auto i) { read_scale(at, i, s0); });
        own_scales(t, s0);
    }
    const auto slice = [&](auto more) {
        constexpr bool MORE = decltype(more)::value;
        const uint32_t at1 = ops_at(t, 1), nx = min(t + 1, n - 1), at0 = ops_at(nx, 0), sat = scales_at(nx);
        multiply(std::integral_constant<int, 0>{}, o0, s0, [&](auto e) { some<R, SPREAD>(e, [&](auto i) { read(at1, i, o1); }); });
        turn(std::integral_constant<int, MORE ? 2 * CPW : 0>{});      // (these load no scales)
        multiply(std::integral_constant<int, 1>{}, o1, s0, [&](auto e) {
            some<R, SPREAD>(e, [&](auto i) { read(at0, i, o0); read_scale(sat, i, s1); });
            if constexpr (MORE) load_codes(t + NST, decltype(e)::value, P);
        });
        s0 = s1;
        own_scales(nx, s0);
    };
    for (; t + NST < n; ++t) slice(std::true_type{});        // (up to three, whose loads need no further scales)
    for (; t < n; ++t) slice(std::false_type{});
    // The sums through LDS, in as many passes as they need room, to whole rows: a thread has the same eight columns of every row that it
    // finishes, in a short loop. (Finished where they are, 256 values a thread, 8192 x 8192 x 512 took 84.8 us, this way 70.8; both with four waves.)
    constexpr int PASSES = T::PASSES, KP = TM / PASSES;
    constexpr uint32_t CH = BN / 8, RS = 64 * NW / CH, RP = 32 * KP;
    const uint32_t c8 = threadIdx.x % CH * 8, nn = n0 + c8, left = nn < a.N ? min(a.N - nn, 8u) : 0u;
    float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (a.bias && a.bias_fp32)                                       // (loads at once; columns behind the last one are not stored)
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) bias[e] = ((const float *)a.bias)[min(nn + e, a.N - 1)];
    else if (a.bias)
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) bias[e] = sh_dev_h2f(((const uint16_t *)a.bias)[min(nn + e, a.N - 1)]);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KP; ++k)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const sh_f16v &v = acc[i][p * KP + k];
                    *(__attribute__((address_space(3))) sh_f4v *)(uintptr_t)(lds0 + ((wm * KP + k) * 32 + r32) * T::PITCH + ((wn * TN + i) * 32 + 8 * q + 4 * g) * 4) =
                        sh_f4v{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                }
        __syncthreads();
        const auto finish = [&](auto gelu) {
            constexpr uint32_t U = BM / PASSES / RS < 4 ? BM / PASSES / RS : 4;      // rows at a time
            static_assert(BM / PASSES % (U * RS) == 0, "rows");
            for (uint32_t r0 = threadIdx.x / CH; r0 < BM / PASSES; r0 += U * RS) {
                sh_f4v f[U][2];
#pragma unroll
                for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) f[u][e] = __builtin_bit_cast(sh_f4v, lds16(lds0 + (r0 + u * RS) * T::PITCH + c8 * 4 + 16 * e));
#pragma unroll
                for (uint32_t u = 0; u < U; ++u) {
                    const uint32_t r = r0 + u * RS, m = m0 + r / RP * (32 * TM) + p * RP + r % RP;
                    sh_u4v v;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        float x = f[u][e / 4][e % 4] + bias[e], y = f[u][e / 4][e % 4 + 1] + bias[e + 1];
                        if constexpr (decltype(gelu)::value) { x = sh_gelu_f32(x); y = sh_gelu_f32(y); }
                        asm("" : "+v"(x), "+v"(y));              // (rounded to fp32 before fp16, as sh_dev_f2h_rr)
                        v[e / 2] = __builtin_bit_cast(uint32_t, sh_h2{(_Float16)x, (_Float16)y});
                    }
                    if (m >= a.M) continue;
                    if (a.res) {
                        const uint4 q = load8(a.res + m * a.ldr, nn, a.N);
                        v = sh_u4v{sh_hadd2(v[0], q.x), sh_hadd2(v[1], q.y), sh_hadd2(v[2], q.z), sh_hadd2(v[3], q.w)};
                    }
                    sh_st8_any(a.z + m * a.ldz + nn, make_uint4(v[0], v[1], v[2], v[3]), left);
                }
            }
        };
        if (!left) continue;
        if (a.act == SH_ACT_GELU) finish(std::true_type{});
        else finish(std::false_type{});
    }
}

template <int BM, int BN, int WGM, int WGN, int PER, bool A16>
bool launch_tile_as(const MxArgs &a, hipStream_t st) {
    using T = Tile<BM, BN, WGM, WGN>;
    static bool set = false;
    if (!set && T::LDS > 65536) {
        if (!sh_hip_ok(hipFuncSetAttribute((const void *)k_mx4_tile<BM, BN, WGM, WGN, PER, A16>, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS),
                       "sh_gemm_mx4 hipFuncSetAttribute")) return false;
        set = true;
    }
    const uint64_t tiles = (uint64_t)sh_cdiv(a.M, BM) * sh_cdiv(a.N, BN);
    hipLaunchKernelGGL((k_mx4_tile<BM, BN, WGM, WGN, PER, A16>), dim3((uint32_t)tiles), dim3(64 * T::NW), T::LDS, st, a);
    return true;
}
template <int BM, int BN, int WGM, int WGN, int PER>
bool launch_tile(const MxArgs &a, hipStream_t st) {
    const bool a16 = !(((uint64_t)a.xs | (uint64_t)a.ws | a.ldxs | a.ldws) % 16);
    return a16 ? launch_tile_as<BM, BN, WGM, WGN, PER, true>(a, st) : launch_tile_as<BM, BN, WGM, WGN, PER, false>(a, st);
}

template <int MT, int CW, int NW, bool F16>
bool launch_rows_as(const MxArgs &a, hipStream_t st) {
    using T = Rows<MT, CW, NW, F16>;
    static bool set = false;
    const uint32_t lds = T::lds(std::min(a.M, 16u * MT)), most_rows = 65535 * 16 * MT;                         // (workgroups in y)
    if (!set && T::lds(16 * MT) > 65536) {
        if (!sh_hip_ok(hipFuncSetAttribute((const void *)k_mx4_rows<MT, CW, NW, F16>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)T::lds(16 * MT)),
                       "sh_gemm_mx4 hipFuncSetAttribute")) return false;
        set = true;
    }
    const uint32_t M = a.M;
    for (uint32_t m = 0; m < M; m += most_rows) {
        MxArgs b = a;
        b.M = std::min(M - m, most_rows);
        if (m) {
            b.xc += m * a.ldxc; b.xs += m * a.ldxs; b.z += m * a.ldz;
            if (b.res) b.res += m * a.ldr;
        }
        hipLaunchKernelGGL((k_mx4_rows<MT, CW, NW, F16>), dim3(sh_cdiv(a.N, 16 * CW), sh_cdiv(b.M, 16 * MT)), dim3(64 * NW), lds, st, b);
    }
    return true;
}
// Columns of a workgroup, by N alone. Wider ones read x (and bring it into codes) less often, but there have to be enough for 256 CUs. us with 16 / 32 / 64
// columns, K = 4096, fp16 rows: 1 x 4096 5.3 / 5.8 / 6.5, 1 x 5000 6.4 / 5.9 / 6.6, 1 x 10240 9.4 / 8.5 / 7.7, 1 x 28000 18.4 / 14.6 / 15.1, 16 x 4096 7.4 / 8.0 / 9.2,
// 16 x 5000 11.7 / 8.3 / 9.4, 16 x 10240 17.2 / 14.0 / 10.6; K = 2048, 16 x 20000 15.3 / 11.8 / 13.0. Rows of codes: 20 x 14336 12.4 / 10.5, 32 x 5000 6.9 / 5.6,
// 32 x 2048 level; up to 16 of them 16 columns (16 x 28000 12.9 / 15.7 / 14.9, 1 x 14336 7.9 / 8.3 / 7.8).
template <int MT, bool F16>
bool launch_rows(const MxArgs &a, hipStream_t st) {
    if constexpr (F16)
        if (a.N > 8192 && a.N <= 16384) return launch_rows_as<MT, 4, 8, F16>(a, st);
    if constexpr (MT == 2 || F16)
        if (a.N > 4096) return launch_rows_as<MT, 2, 8, F16>(a, st);
    return launch_rows_as<MT, 1, 8, F16>(a, st);
}

// The checks that both products make of the weight, the result and the epilogue.
int product_args(const char *name, uint64_t wc, uint64_t ws, uint64_t z, uint32_t M, uint32_t N, uint32_t K, uint32_t ldwc, uint32_t ldws, uint32_t ldz,
                 const sh_gemm_epi *epi, MxArgs *a) {
    if (!wc || !ws || !z) { sh_set_error(-1, "[%s] NULL tensor address", name); return -1; }
    if (!K || K > (1u << 31)) { sh_set_error(-1, "[%s] K %u", name, K); return -1; }
    if (M > (1u << 26) || N > (1u << 26)) { sh_set_error(-1, "[%s] M=%u N=%u too large", name, M, N); return -1; }
    const uint32_t nb = (K - 1) / 32 + 1;
    if (wc % 16 || ldwc % 16 || ldwc < 16 * (uint64_t)nb) { sh_set_error(-1, "[%s] weight codes: 16-byte aligned, leading dim %u for %u blocks", name, ldwc, nb); return -1; }
    if (ws % 4 || ldws % 4 || ldws < nb) { sh_set_error(-1, "[%s] weight scales: 4-byte aligned, leading dim %u for %u blocks", name, ldws, nb); return -1; }
    if (z % 2 || ldz < N) { sh_set_error(-1, "[%s] leading dim %u for %u columns, or alignment of z", name, ldz, N); return -1; }
    *a = MxArgs{};
    a->wc = (const uint8_t *)wc; a->ws = (const uint8_t *)ws;
    a->z = (uint16_t *)z;
    a->M = M; a->N = N; a->K = K; a->nb = nb;
    a->ldwc = ldwc; a->ldws = ldws; a->ldz = ldz;
    if (!epi) return 0;
    if (epi->act > SH_ACT_GELU) { sh_set_error(-1, "[%s] unknown act %u", name, epi->act); return -1; }
    if (epi->bias && (epi->bias_fmt > SH_BIAS_FP32 || epi->bias % (epi->bias_fmt == SH_BIAS_FP32 ? 4 : 2))) {
        sh_set_error(-1, "[%s] bias format %u or its alignment", name, epi->bias_fmt);
        return -1;
    }
    if (epi->residual && (epi->ldr < N || epi->residual % 2)) { sh_set_error(-1, "[%s] ldr %u < N %u, or alignment", name, epi->ldr, N); return -1; }
    if (epi->splits > 1 || epi->ln_stats || epi->ln_c || epi->stats_out || epi->ln_parts) {
        sh_set_error(-1, "[%s] no K split, LayerNorm fold or row partials", name);
        return -1;
    }
    a->bias = (const void *)epi->bias; a->bias_fp32 = epi->bias_fmt == SH_BIAS_FP32;
    a->act = epi->act;
    a->res = (const uint16_t *)epi->residual; a->ldr = epi->ldr;
    return 0;
}

}  // namespace

extern "C" {

int sh_mx4_quant(uint64_t codes, uint64_t scales, uint64_t x, uint32_t rows, uint32_t cols, uint32_t ldc, uint32_t lds, uint32_t ldx) {
    if (!rows || !cols) return 0;
    if (!codes || !scales || !x) { sh_set_error(-1, "[sh_mx4_quant] NULL address"); return -1; }
    const uint32_t nb = (cols - 1) / 32 + 1;
    if (codes % 16 || ldc % 16 || ldc < 16 * (uint64_t)nb) { sh_set_error(-1, "[sh_mx4_quant] codes: 16-byte aligned, leading dim %u for %u blocks", ldc, nb); return -1; }
    if (scales % 4 || lds % 4 || lds < nb) { sh_set_error(-1, "[sh_mx4_quant] scales: 4-byte aligned, leading dim %u for %u blocks", lds, nb); return -1; }
    if (x % 2 || ldx < cols) { sh_set_error(-1, "[sh_mx4_quant] leading dim %u for %u columns, or alignment of x", ldx, cols); return -1; }
    if (cols > (1u << 30)) { sh_set_error(-1, "[sh_mx4_quant] %u columns", cols); return -1; }
    QuantArgs a{(uint8_t *)codes, (uint8_t *)scales, (const uint16_t *)x, ldc, lds, ldx, 0, cols, 0, sh_make_div(4 * nb)};
    const uint32_t most = std::max(1u, (1u << 30) / (4 * nb));                  // rows of a launch
    for (uint64_t r = 0; r < rows; r += most) {
        a.row0 = (uint32_t)r;
        a.items = std::min<uint64_t>(rows - r, most) * 4 * nb;
        hipLaunchKernelGGL(k_mx4_quant, dim3((uint32_t)((a.items + 255) / 256)), dim3(256), 0, sh_stream(), a);
    }
    return sh_launch_ok("sh_mx4_quant") ? 0 : SH_EHIP;
}

int sh_gemm_mx4(uint64_t xc, uint64_t xs, uint64_t wc, uint64_t ws, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                uint32_t ldxc, uint32_t ldxs, uint32_t ldwc, uint32_t ldws, uint32_t ldz, const sh_gemm_epi *epi) {
    if (!M || !N) return 0;
    MxArgs a;
    if (int rc = product_args("sh_gemm_mx4", wc, ws, z, M, N, K, ldwc, ldws, ldz, epi, &a)) return rc;
    if (!xc || !xs) { sh_set_error(-1, "[sh_gemm_mx4] NULL tensor address"); return -1; }
    if (xc % 16 || ldxc % 16 || ldxc < 16 * (uint64_t)a.nb) { sh_set_error(-1, "[sh_gemm_mx4] codes: 16-byte aligned, leading dim %u for %u blocks", ldxc, a.nb); return -1; }
    if (xs % 4 || ldxs % 4 || ldxs < a.nb) { sh_set_error(-1, "[sh_gemm_mx4] scales: 4-byte aligned, leading dim %u for %u blocks", ldxs, a.nb); return -1; }
    a.xc = (const uint8_t *)xc; a.xs = (const uint8_t *)xs;
    a.ldxc = ldxc; a.ldxs = ldxs;
    const hipStream_t st = sh_stream();
    // Tiles by the rounds of workgroups that they take on 256 CUs, whatever K: a workgroup has all of it, so few tiles of a long K leave CUs idle (128 x 1024, 32 tiles:
    // K = 4096 6.8 us, 16384 24.4). Times (us, K = 4096, epilogue without residual) of the first round and of a further one: small
    // tiles' workgroups share a CU. 2048 x 4096: 47 / 40 / 30 / 27.5 / 31.5; 1000 x 2048: 14.4 / 13.6 / 15.0 / 21 / 29; 300 x 4096: 12.0 / 11.8 / 13.7 / 20 / 27;
    // 100 x 4096: 8.0 / 10.3 / 12.0 / 17 / 24; 700 x 5000 (K = 2880): 22 / 18.5 / 15.3 / 19.7 / 26; 4096 x 4096: 87 / 70 / 55 / 51 / 41.
    struct Shape { uint32_t bm, bn; double first, more; };
    static const Shape shapes[] = {{64, 64, 8, 6}, {64, 128, 11.5, 9.5}, {128, 128, 14.5, 14.5}, {128, 256, 26, 26}, {256, 256, 39, 39}};
    int pick = 0;
    double least = 0;
    for (int i = 0; i < 5; ++i) {
        const uint64_t tiles = (uint64_t)sh_cdiv(M, shapes[i].bm) * sh_cdiv(N, shapes[i].bn);
        const double c = shapes[i].first + shapes[i].more * (double)((tiles - 1) / 256);
        if (!i || c < least) { pick = i; least = c; }
    }
    const bool near = ldxc <= (1u << 24) && ldwc <= (1u << 24) && ldxs <= (1u << 24) && ldws <= (1u << 24);       // a tile's rows within 32-bit offsets
    bool ok = true;
    // Up to 64 rows the chain is shared by a workgroup's waves; more than 32 of many columns fill the GPU as tiles (64 rows of 4096 x 6144: 9.4 us, 10.7 so; 48 of
    // 2880 x 5000 7.1 and 8.6; but 64 of 4096 x 4096 9.1 and 5.9, of 8192 x 2048 13.8 and 7.9). Rows too far apart for a tile's offsets take the kernel for few rows
    // however many there are (700 x 1024 x 2880 7.1 us, 12.4 so).
    if (M <= 16) ok = launch_rows<1, false>(a, st);
    else if (M <= 32) ok = launch_rows<2, false>(a, st);
    else if ((M <= 64 && N <= 4096) || !near) ok = launch_rows<4, false>(a, st);
    else if (pick == 0) ok = launch_tile<64, 64, 2, 2, 2>(a, st);
    else if (pick == 1) ok = launch_tile<64, 128, 2, 2, 2>(a, st);
    else if (pick == 2) ok = launch_tile<128, 128, 2, 2, 2>(a, st);
    else if (pick == 3) ok = launch_tile<128, 256, 2, 4, 2>(a, st);
    else ok = launch_tile<256, 256, 4, 2, 2>(a, st);
    if (!ok) return SH_EHIP;
    return sh_launch_ok("sh_gemm_mx4") ? 0 : SH_EHIP;
}

int sh_gemm_mx4_f16(uint64_t x, uint64_t wc, uint64_t ws, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                    uint32_t ldx, uint32_t ldwc, uint32_t ldws, uint32_t ldz, const sh_gemm_epi *epi) {
    if (!M || !N) return 0;
    MxArgs a;
    if (int rc = product_args("sh_gemm_mx4_f16", wc, ws, z, M, N, K, ldwc, ldws, ldz, epi, &a)) return rc;
    if (!x || x % 2 || ldx < K) { sh_set_error(-1, "[sh_gemm_mx4_f16] x: NULL, not 2-byte aligned, or leading dim %u < %u", ldx, K); return -1; }
    if (M > 16) { sh_set_error(-1, "[sh_gemm_mx4_f16] %u rows (up to 16; more by sh_mx4_quant and sh_gemm_mx4)", M); return -1; }
    a.x = (const uint16_t *)x; a.ldx = ldx;
    if (!launch_rows<1, true>(a, sh_stream())) return SH_EHIP;
    return sh_launch_ok("sh_gemm_mx4_f16") ? 0 : SH_EHIP;
}

}  // extern "C"
