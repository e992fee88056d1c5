// The 8-bit paged key / value cache: block tables and slots of a step (sh_kv_slots) and the write of new rows
// (sh_kv_append). The attention over it is in sh_kv_attention.hip.
#include "sh_kv.h"
#include <math.h>

int sh_kv_check(const char *name, const sh_kv_cache *c, KvCache *out) {
    if (!c || !c->k || !c->v || !c->ks || !c->vs) { sh_set_error(-1, "[%s] NULL cache or cache address", name); return -1; }
    if (c->bs != 16 && c->bs != 32 && c->bs != 64) { sh_set_error(-1, "[%s] pages of %u tokens (16, 32 or 64)", name, c->bs); return -1; }
    if (!c->dh || c->dh > 256 || c->dh % 16) { sh_set_error(-1, "[%s] head width %u (a multiple of 16 up to 256)", name, c->dh); return -1; }
    if (!c->hkv || c->hkv > 1024) { sh_set_error(-1, "[%s] %u key / value heads (1 .. 1024)", name, c->hkv); return -1; }
    if (c->fmt != SH_INT8 && c->fmt != SH_FP8) { sh_set_error(-1, "[%s] fmt %u (SH_INT8 or SH_FP8)", name, c->fmt); return -1; }
    if (!c->pages || (uint64_t)c->pages * c->bs >= (1ull << 31)) { sh_set_error(-1, "[%s] %u pages of %u tokens", name, c->pages, c->bs); return -1; }
    const uint64_t pg = (uint64_t)c->hkv * c->bs * c->dh;
    const uint64_t pgk = c->pgk ? c->pgk : pg, pgv = c->pgv ? c->pgv : pg;
    const uint32_t pgs = c->pgs ? c->pgs : c->hkv;
    if (pgk < pg || pgv < pg || pgs < c->hkv) { sh_set_error(-1, "[%s] a page stride is smaller than a page", name); return -1; }
    if ((c->k | c->v | pgk | pgv) % 16 || (c->ks | c->vs) % 4) {
        sh_set_error(-1, "[%s] codes and page strides must be 16-byte aligned, scales 4-byte aligned", name);
        return -1;
    }
    uint32_t l = 0;
    while ((1u << l) < c->bs) ++l;
    *out = KvCache{(uint8_t *)c->k, (uint8_t *)c->v, (float *)c->ks, (float *)c->vs, pgk, pgv, pgs, c->pages, c->hkv, c->dh, c->bs, l};
    return 0;
}

namespace {

// ---- sh_kv_slots --------------------------------------------------------------------------------------------------
// Three prefix sums over the requests (rows, pages taken, pages given back) decide everything; the work behind them is
// one write for each new row, new page and returned page. Requests are scanned in chunks of the workgroup's threads; within a
// chunk the rows and pages are spread evenly over threads (a binary search in the chunk's sums finds a row's request), so
// one long prompt costs as much as many short requests.
struct SlotArgs {
    int32_t *table; uint32_t ld;
    const int32_t *lens, *add, *state;
    int32_t *lens_out, *state_out, *pool, *row_start, *slots, *pos, *kv_len;
    uint32_t B, lbs, pages, rows;
    uint32_t commit;     // this launch writes the new lengths and the ring's state
    uint32_t fill;       // this launch writes everything else
};

// Inclusive sum over the wave's lanes of a value split in 64 bits.
__device__ __forceinline__ int64_t wave_scan64(int64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// Inclusive sum over the workgroup, and its total; `part` holds one value a wave.
template <int T>
__device__ __forceinline__ int64_t group_scan64(int64_t v, int64_t *part, int64_t &total) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    v = wave_scan64(v);
    if (lane == 63) part[wave] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
        const int64_t p = part[w];
        before += w < wave ? p : 0;
        total += p;
    }
    __syncthreads();
    return v + before;
}

template <int T>
__global__ __launch_bounds__(T) void k_kv_slots(SlotArgs a) {
    __shared__ int64_t part[T / 64];
    __shared__ int32_t s_end[T], s_need[T], s_back[T], s_len[T], s_flag[T];     // sums within the chunk; flag: request is served
    __shared__ int32_t s_used, s_refused;
    const uint32_t tid = threadIdx.x, bs = 1u << a.lbs;
    const int64_t cap = (int64_t)a.ld << a.lbs;
    const int32_t head = a.state[0], count0 = a.state[1];
    const int64_t count = min(max(count0, 0), (int32_t)a.pages);
    const uint32_t h0 = (uint32_t)max(head, 0) % a.pages;
    if (tid == 0) s_used = s_refused = 0;
    int64_t rows0 = 0, need0 = 0, back0 = 0;                                    // the earlier chunks' sums
    for (uint32_t b0 = 0; b0 < a.B; b0 += T) {
        const uint32_t b = b0 + tid;
        const int32_t ad = b < a.B ? a.add[b] : 0;
        const int64_t raw = b < a.B ? a.lens[b] : 0, len = min(max(raw, (int64_t)0), cap), n = max(ad, 0);
        int64_t total_n, total_np;
        const int64_t end = rows0 + group_scan64<T>(n, part, total_n);
        bool ok = b < a.B && ad >= 0 && len + n <= cap && end <= (int64_t)a.rows;
        const int32_t have = (int32_t)((len + bs - 1) >> a.lbs);
        const int32_t need = ok ? (int32_t)((len + n + bs - 1) >> a.lbs) - have : 0, back = ad < 0 ? have : 0;
        // both page sums stay below B ld < 2^31: one scan of the pair
        const int64_t np = group_scan64<T>((int64_t)need << 32 | back, part, total_np);
        const int64_t upto = need0 + (np >> 32);
        ok = ok && (need == 0 || upto <= count);
        if (need && ok) atomicMax(&s_used, (int32_t)upto);
        if (b < a.B && ad >= 0 && !ok) atomicAdd(&s_refused, 1);
        if (b < a.B && a.commit) a.lens_out[b] = ok ? (int32_t)(len + n) : ad < 0 ? 0 : (int32_t)raw;
        if (a.fill) {
            if (b < a.B && blockIdx.x == 0) {
                a.row_start[b] = (int32_t)(end - n);
                a.kv_len[b] = ok ? (int32_t)(len + n) : 0;
                if (b == a.B - 1) a.row_start[a.B] = (int32_t)end;
            }
            s_end[tid] = (int32_t)min(end - rows0, (int64_t)a.rows);            // (only rows below a.rows are looked up)
            s_need[tid] = (int32_t)(np >> 32);
            s_back[tid] = (int32_t)(uint32_t)np;
            s_len[tid] = (int32_t)len;
            s_flag[tid] = ok;
            __syncthreads();
            const uint32_t stride = T * gridDim.x, first = blockIdx.x * T + tid;
            auto find = [&](const int32_t *s, int32_t i) {                      // first request whose sum exceeds i
                uint32_t lo = 0, hi = T - 1;
                while (lo < hi) {
                    const uint32_t m = (lo + hi) / 2;
                    if (s[m] > i) hi = m; else lo = m + 1;
                }
                return lo;
            };
            // the ring's ranges taken from and given back to do not meet: together they are at most `pages` long
            const uint32_t pages_new = (uint32_t)(total_np >> 32), pages_back = (uint32_t)total_np;
            for (uint32_t i = first; i < pages_new; i += stride) {
                const uint32_t f = find(s_need, (int32_t)i);
                if (!s_flag[f]) continue;
                const uint32_t j = i - (f ? (uint32_t)s_need[f - 1] : 0u), hv = ((uint32_t)s_len[f] + bs - 1) >> a.lbs;
                a.table[(uint64_t)(b0 + f) * a.ld + hv + j] = a.pool[(uint32_t)((h0 + (uint64_t)need0 + i) % a.pages)];
            }
            for (uint32_t i = first; i < pages_back; i += stride) {
                const uint32_t f = find(s_back, (int32_t)i);
                const uint32_t j = i - (f ? (uint32_t)s_back[f - 1] : 0u);
                a.pool[(uint32_t)((h0 + (uint64_t)count + back0 + i) % a.pages)] = a.table[(uint64_t)(b0 + f) * a.ld + j];
            }
            const int64_t rows_here = min(total_n, (int64_t)a.rows - min(rows0, (int64_t)a.rows));
            for (int64_t i = first; i < rows_here; i += stride) {
                const uint32_t f = find(s_end, (int32_t)i);
                const uint32_t at = (uint32_t)s_len[f] + (uint32_t)(i - (f ? s_end[f - 1] : 0)), j = at >> a.lbs;
                int32_t slot = -1, p = -1;
                if (s_flag[f]) {
                    // a page of this step is read from the ring: its table entry is being written
                    const uint32_t hv = ((uint32_t)s_len[f] + bs - 1) >> a.lbs, nb = f ? (uint32_t)s_need[f - 1] : 0u;
                    const int32_t page = j < hv ? a.table[(uint64_t)(b0 + f) * a.ld + j]
                                                : a.pool[(uint32_t)((h0 + (uint64_t)need0 + nb + (j - hv)) % a.pages)];
                    p = (int32_t)at;
                    if ((uint32_t)page < a.pages) slot = (int32_t)(((uint32_t)page << a.lbs) + (at & (bs - 1)));
                }
                a.slots[rows0 + i] = slot;
                a.pos[rows0 + i] = p;
            }
            __syncthreads();
        }
        rows0 += total_n; need0 += total_np >> 32; back0 += (uint32_t)total_np;
    }
    if (a.fill) {
        for (int64_t i = rows0 + (int64_t)blockIdx.x * T + tid; i < (int64_t)a.rows; i += (int64_t)T * gridDim.x) {
            a.slots[i] = -1;
            a.pos[i] = -1;
        }
        if (a.B == 0 && blockIdx.x == 0 && tid == 0) a.row_start[0] = 0;
    }
    __syncthreads();
    if (a.commit && tid == 0) {
        const int64_t left = count - s_used + back0;
        a.state_out[0] = (int32_t)((h0 + (uint64_t)s_used) % a.pages);
        a.state_out[1] = (int32_t)min(left, (int64_t)a.pages);
        a.state_out[2] = s_refused;
    }
}

// ---- sh_kv_append -------------------------------------------------------------------------------------------------
struct AppendArgs {
    KvCache c;
    const uint16_t *k, *v;
    uint64_t ldk, ldv;
    const int32_t *slots;
    uint32_t rows, rg;
    ShDiv dch;                             // by dh / 8
};

// |x| of a pair of halves as integers (monotone), NaN as 0, infinity as 65504.
__device__ __forceinline__ uint32_t abs_bits(uint32_t h) {
    const uint32_t a = h & 0x7FFFu;
    return a > 0x7C00u ? 0u : min(a, 0x7BFFu);
}
__device__ __forceinline__ float clean(uint16_t h) { return sh_dev_h2f((uint16_t)(abs_bits(h) | (h & 0x8000u))); }

// The smallest power of two s >= 2^-32 with amax <= s Q, Q = 127 or 448: amax = f 2^e with f in [0.5, 1), Q = q 2^x likewise.
template <bool FP8>
__device__ __forceinline__ float pow2_scale(float amax) {
    const float q = FP8 ? 0.875f : 0.9921875f;
    const int x = FP8 ? 9 : 7, e = __builtin_amdgcn_frexp_expf(amax);
    const float f = __builtin_amdgcn_frexp_mantf(amax);
    const int p = amax > 0.f ? max(f <= q ? e - x : e - x + 1, -32) : -32;
    return __uint_as_float((uint32_t)(p + 127) << 23);
}
// The codes of four values already divided by their scale, in a word: nearest, ties to even.
template <bool FP8>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    if constexpr (FP8) {
        const auto lim = [](float x) { return __builtin_amdgcn_fmed3f(x, -448.f, 448.f); };
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(lim(c), lim(d), __builtin_amdgcn_cvt_pk_fp8_f32(lim(a), lim(b), 0, false), true);
    } else {
        const auto q = [](float x) { return (uint32_t)(int)__builtin_amdgcn_fmed3f(__builtin_rintf(x), -127.f, 127.f); };
        const uint32_t lo = __builtin_amdgcn_perm(q(b), q(a), 0x0C0C0400u), hi = __builtin_amdgcn_perm(q(d), q(c), 0x04000C0Cu);
        return lo | hi;
    }
}
template <bool FP8>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
    if constexpr (FP8)
        return codes4<FP8>(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * ratio,
                           __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * ratio);
    else
        return codes4<FP8>((float)(int8_t)w * ratio, (float)(int8_t)(w >> 8) * ratio, (float)(int8_t)(w >> 16) * ratio, (float)(int8_t)(w >> 24) * ratio);
}

// A workgroup takes RG rows, one head and keys or values, and does the pages whose first new row is among its rows, one after
// the other. A thread holds four tokens by eight columns of the page (one such item), the tokens at the page's own multiples of
// four: four 16-byte loads; after the page's largest value is known, the codes of a key's eight columns are one 8-byte store a
// token, those of a value's four tokens one 4-byte store a column (a page of values has its tokens consecutive). At most 64 x 256
// values a page: 512 items. Bound by HBM: 2 bytes read and 1 written a value; written pages are whole lines in L2.
template <bool FP8, int NT>
__global__ __launch_bounds__(NT) void k_kv_append(AppendArgs a) {
    __shared__ uint32_t s_top[NT / 64];
    const KvCache &c = a.c;
    const uint32_t tid = threadIdx.x, lane = tid & 63, r0 = blockIdx.x * a.rg, h = blockIdx.y, isv = blockIdx.z;
    const uint32_t cap = c.pages << c.lbs, dh = c.dh, nch = dh / 8;
    // the first row of a page's run: it begins a page, or the row before does not precede it. Lane i: row r0 + i
    const uint32_t rl = r0 + lane;
    const uint32_t sl = rl < a.rows ? (uint32_t)a.slots[rl] : ~0u;
    const uint32_t sb = rl < a.rows && rl ? (uint32_t)a.slots[rl - 1] : ~0u;
    uint64_t lead = __ballot(lane < a.rg && sl < cap && (!(sl & (c.bs - 1)) || !rl || sb != sl - 1));
    const uint64_t ld = isv ? a.ldv : a.ldk;
    while (lead) {
        const uint32_t f = __builtin_ctzll(lead), r = r0 + f;
        lead &= lead - 1;
        const uint32_t s0 = (uint32_t)__builtin_amdgcn_readlane((int)sl, (int)f), off = s0 & (c.bs - 1), page = s0 >> c.lbs;
        // the run's rows, a page's rest of at most 64: among the rows read, or read again
        uint64_t has;
        if (f + c.bs - off <= 64) has = __ballot(lane >= f && lane - f < c.bs - off && sl == s0 + lane - f) >> f;
        else has = __ballot(lane < c.bs - off && r + lane < a.rows && (uint32_t)a.slots[min(r + lane, a.rows - 1)] == s0 + lane);
        const uint32_t n = ~has ? (uint32_t)__builtin_ctzll(~has) : 64u, end = off + n;
        const uint16_t *src = (isv ? a.v : a.k) + (uint64_t)r * ld + (uint64_t)h * dh;
        uint8_t *dst = (isv ? c.v + page * c.pgv : c.k + page * c.pgk) + (uint64_t)h * c.bs * dh;
        float *sp = (isv ? c.vs : c.ks) + (uint64_t)page * c.pgs + h;
        const float was = off ? *sp : 0.f;
        const uint32_t blk0 = off / 4, items = ((end + 3) / 4 - blk0) * nch;
        uint4 x[4];
        uint32_t top = 0;
        const uint32_t bl = sh_div(tid, a.dch), ch = tid - bl * nch, t0 = 4 * (blk0 + bl);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t t = t0 + j;
            x[j] = make_uint4(0, 0, 0, 0);
            if (tid < items && t >= off && t < end) x[j] = sh_ld16_any(src + (uint64_t)(t - off) * ld + 8 * ch);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(abs_bits(w[e] & 0xFFFFu), abs_bits(w[e] >> 16)));
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        if constexpr (NT > 64) {
            __syncthreads();                                        // the last page's maxima are read
            if (lane == 0) s_top[tid / 64] = top;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NT / 64; ++i) top = max(top, s_top[i]);
        }
        const float s = fmaxf(was, pow2_scale<FP8>(sh_dev_h2f((uint16_t)top)));
        if (off && s != was) {                                      // the page's older tokens: whole words, and the bytes beside the new ones
            const float ratio = was / s;
            uint32_t *d32 = (uint32_t *)dst;
            if (!isv) {
                for (uint32_t i = tid; i < off * dh / 4; i += NT) d32[i] = rescale4<FP8>(d32[i], ratio);
            } else {
                for (uint32_t i = tid; i < blk0 * dh; i += NT) {
                    uint32_t *p = d32 + (i / blk0) * (c.bs / 4) + i % blk0;
                    *p = rescale4<FP8>(*p, ratio);
                }
                for (uint32_t i = tid; i < (off & 3) * dh; i += NT) {
                    uint8_t *p = dst + (i % dh) * c.bs + 4 * blk0 + i / dh;
                    *p = (uint8_t)rescale4<FP8>(*p, ratio);
                }
            }
        }
        // x / s: the reciprocal of a power of two is exact (only a caller's own scales are not one)
        const bool p2 = (__float_as_uint(s) & 0x7FFFFFu) == 0;
        const float inv = 1.f / s;
        if (tid < items) {
            float v[4][8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = clean((uint16_t)(w[e / 2] >> (16 * (e & 1))));
            }
            if (p2) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j / 8][j % 8] *= inv;
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j / 8][j % 8] /= s;
            }
            if (!isv) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t t = t0 + j;
                    if (t >= off && t < end)
                        *(uint2 *)(dst + t * dh + 8 * ch) = make_uint2(codes4<FP8>(v[j][0], v[j][1], v[j][2], v[j][3]), codes4<FP8>(v[j][4], v[j][5], v[j][6], v[j][7]));
                }
            } else {
                const bool whole = t0 >= off && t0 + 4 <= end;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    uint8_t *p = dst + (8 * ch + e) * c.bs + t0;
                    const uint32_t w = codes4<FP8>(v[0][e], v[1][e], v[2][e], v[3][e]);
                    if (whole) *(uint32_t *)p = w;
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (t0 + j >= off && t0 + j < end) p[j] = (uint8_t)(w >> (8 * j));
                }
            }
        }
        if (tid == 0) *sp = s;
    }
}

template <bool FP8>
void launch_append(AppendArgs &a, hipStream_t st) {
    const dim3 grid(sh_cdiv(a.rows, a.rg), a.c.hkv, 2);
    const uint32_t items = a.c.bs * a.c.dh / 32;
    if (items <= 64) hipLaunchKernelGGL((k_kv_append<FP8, 64>), grid, dim3(64), 0, st, a);
    else if (items <= 128) hipLaunchKernelGGL((k_kv_append<FP8, 128>), grid, dim3(128), 0, st, a);
    else if (items <= 256) hipLaunchKernelGGL((k_kv_append<FP8, 256>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_kv_append<FP8, 512>), grid, dim3(512), 0, st, a);
}

}  // namespace

extern "C" {

int sh_kv_slots(uint64_t table, uint32_t ld, uint64_t lens, uint64_t lens_out, uint64_t add, uint64_t pool, uint64_t state, uint64_t state_out,
                uint64_t row_start, uint64_t slots, uint64_t pos, uint64_t kv_len, uint32_t B, uint32_t bs, uint32_t pages, uint32_t rows) {
    if (!table || !lens || !lens_out || !add || !pool || !state || !state_out || !row_start || !kv_len || (rows && (!slots || !pos))) {
        sh_set_error(-1, "[sh_kv_slots] NULL address");
        return -1;
    }
    if ((table | lens | lens_out | add | pool | state | state_out | row_start | slots | pos | kv_len) % 4) {
        sh_set_error(-1, "[sh_kv_slots] arrays must be 4-byte aligned");
        return -1;
    }
    if (bs != 16 && bs != 32 && bs != 64) { sh_set_error(-1, "[sh_kv_slots] pages of %u tokens (16, 32 or 64)", bs); return -1; }
    if (!B || B > 65536 || !ld || (uint64_t)B * ld >= (1ull << 31) || !pages || (uint64_t)pages * bs >= (1ull << 31) || rows >= (1u << 31) ||
        (uint64_t)ld * bs >= (1ull << 31)) {
        sh_set_error(-1, "[sh_kv_slots] bad B=%u ld=%u bs=%u pages=%u rows=%u", B, ld, bs, pages, rows);
        return -1;
    }
    SlotArgs a{(int32_t *)table, ld, (const int32_t *)lens, (const int32_t *)add, (const int32_t *)state, (int32_t *)lens_out,
               (int32_t *)state_out, (int32_t *)pool, (int32_t *)row_start, (int32_t *)slots, (int32_t *)pos, (int32_t *)kv_len,
               B, bs == 16 ? 4u : bs == 32 ? 5u : 6u, pages, rows, 1, 1};
    const hipStream_t st = sh_stream();
    const uint32_t groups = rows <= 4096 ? 1u : min(sh_cdiv(rows, 1024), 256u);
    if (groups == 1) {
        hipLaunchKernelGGL(k_kv_slots<1024>, dim3(1), dim3(1024), 0, st, a);
        return sh_launch_ok("sh_kv_slots") ? 0 : SH_EHIP;
    }
    a.commit = 0;
    hipLaunchKernelGGL(k_kv_slots<1024>, dim3(groups), dim3(1024), 0, st, a);
    a.commit = 1; a.fill = 0;
    hipLaunchKernelGGL(k_kv_slots<1024>, dim3(1), dim3(1024), 0, st, a);
    return sh_launch_ok("sh_kv_slots") ? 0 : SH_EHIP;
}

int sh_kv_append(const sh_kv_cache *c, uint64_t k, uint64_t v, uint32_t ldk, uint32_t ldv, uint64_t slots, uint32_t rows) {
    AppendArgs a;
    if (int rc = sh_kv_check("sh_kv_append", c, &a.c)) return rc;
    if (!rows) return 0;
    if (!k || !v || !slots) { sh_set_error(-1, "[sh_kv_append] NULL address"); return -1; }
    if ((k | v) % 2 || slots % 4) { sh_set_error(-1, "[sh_kv_append] rows must be 2-byte aligned, slots 4-byte aligned"); return -1; }
    if (ldk < c->hkv * c->dh || ldv < c->hkv * c->dh) {
        sh_set_error(-1, "[sh_kv_append] leading dim %u or %u < %u", ldk, ldv, c->hkv * c->dh);
        return -1;
    }
    if (rows >= (1u << 31)) { sh_set_error(-1, "[sh_kv_append] %u rows", rows); return -1; }
    a.k = (const uint16_t *)k; a.v = (const uint16_t *)v;
    a.ldk = ldk; a.ldv = ldv;
    a.slots = (const int32_t *)slots;
    a.rows = rows;
    a.dch = sh_make_div(c->dh / 8);
    // rows of a workgroup: one while all pages run at once, then few enough that most have a page to do in a prompt
    a.rg = rows <= 512 ? 1 : rows <= 4096 ? 4 : c->bs;
    if (c->fmt == SH_FP8) launch_append<true>(a, sh_stream());
    else launch_append<false>(a, sh_stream());
    return sh_launch_ok("sh_kv_append") ? 0 : SH_EHIP;
}

}  // extern "C"
