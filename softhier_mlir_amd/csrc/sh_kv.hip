// The 8-bit paged key / value cache: block tables and slots of a step (sh_kv_slots) and the write of new rows
// (sh_kv_append). The attention over it is in sh_kv_attention.hip.
#include "sh_kv.h"
#include <algorithm>

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
// one write for each new row, new page and returned page. Requests are scanned in chunks of the workgroup's threads. Where a chunk's
// requests add a few rows each, a thread writes its own; else rows and pages are spread evenly over the threads of all
// workgroups (a binary search in the chunk's sums finds a row's request), so one long prompt costs as much as many short requests.
// Bound by latency: a launch, the lengths, then a page, then the writes (64 single tokens 4.6 us, 1024 requests with 44 thousand rows 7.0).
struct SlotArgs {
    int32_t *table; uint32_t ld;
    const int32_t *lens, *add, *state;
    int32_t *lens_out, *state_out, *pool, *row_start, *slots, *pos, *kv_len;
    uint32_t B, lbs, pages, rows;
    uint32_t commit;     // this launch writes the new lengths and the ring's state
    uint32_t fill;       // this launch writes everything else
};
constexpr uint32_t OWN = 4;                // rows of a request up to which its thread writes them

// Inclusive sum over the workgroup, and its total; `part` holds one value a wave.
template <int T>
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t *part, uint32_t &total) {
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    v = kv_wave_scan(v);
    if (lane == 63) part[wave] = v;
    __syncthreads();
    const uint32_t p = kv_wave_scan(lane < T / 64 ? part[lane] : 0u);
    total = (uint32_t)__builtin_amdgcn_readlane((int)p, 63);
    return v + (wave ? (uint32_t)__builtin_amdgcn_readlane((int)p, (int)__builtin_amdgcn_readfirstlane(wave) - 1) : 0u);
}

template <int T>
__global__ __launch_bounds__(T) void k_kv_slots(SlotArgs a) {
    __shared__ uint32_t part[3][T / 64];
    __shared__ uint32_t s_end[T], s_need[T], s_back[T];              // sums within the chunk
    __shared__ int32_t s_len[T], s_flag[T];                          // flag: the request is served
    __shared__ uint32_t s_used, s_refused;
    const uint32_t tid = threadIdx.x, bs = 1u << a.lbs, cap = a.ld << a.lbs;
    const uint32_t count = (uint32_t)min(max(a.state[1], 0), (int32_t)a.pages), h0 = (uint32_t)max(a.state[0], 0) % a.pages;
    const auto ring = [&](uint32_t i) {                              // i < 2^31 places behind the ring's first entry
        const uint32_t x = h0 + i;
        return x < a.pages ? x : x - a.pages < a.pages ? x - a.pages : x % a.pages;
    };
    if (tid == 0) s_used = s_refused = 0;
    uint32_t rows0 = 0, need0 = 0, back0 = 0;                        // the earlier chunks' sums
    for (uint32_t b0 = 0; b0 < a.B; b0 += T) {
        const uint32_t b = b0 + tid;
        const int32_t ad = b < a.B ? a.add[b] : 0, raw = b < a.B ? a.lens[b] : 0;
        const uint32_t len = min((uint32_t)max(raw, 0), cap), n = (uint32_t)max(ad, 0);
        uint32_t total_n, total_need, total_back;
        const uint32_t in_n = group_scan<T>(n, part[0], total_n), end = rows0 + in_n;
        bool ok = b < a.B && ad >= 0 && n <= cap - len && end <= a.rows;
        const uint32_t have = (len + bs - 1) >> a.lbs, need = ok ? ((len + n + bs - 1) >> a.lbs) - have : 0, back = ad < 0 ? have : 0;
        const uint32_t in_need = group_scan<T>(need, part[1], total_need), in_back = group_scan<T>(back, part[2], total_back);
        const uint32_t upto = need0 + in_need, need_b = upto - need;
        ok = ok && (need == 0 || upto <= count);
        if (need && ok) atomicMax(&s_used, upto);
        if (b < a.B && ad >= 0 && !ok) atomicAdd(&s_refused, 1);
        const int32_t *row = a.table + (uint64_t)b * a.ld;
        // the ring's ranges taken from and given back to do not meet: together they are at most `pages` long
        if (a.fill) {
            const bool few = !__syncthreads_or(n > OWN || back);
            if (blockIdx.x == 0 && b < a.B) {
                a.row_start[b] = (int32_t)(end - n);
                a.kv_len[b] = ok ? (int32_t)(len + n) : 0;
                if (b == a.B - 1) a.row_start[a.B] = (int32_t)end;
            }
            if (few) {
                if (blockIdx.x == 0 && b < a.B && n) {
                    // n <= 4 rows lie in at most one page held and one page taken
                    const int32_t held = (len & (bs - 1)) && ok ? row[len >> a.lbs] : 0, taken = need && ok ? a.pool[ring(need_b)] : 0;
                    if (need && ok) a.table[(uint64_t)b * a.ld + have] = taken;
                    for (uint32_t i = 0; i < n; ++i) {
                        const uint32_t r = end - n + i, at = len + i;
                        const int32_t page = (at >> a.lbs) < have ? held : taken;
                        if (r >= a.rows) break;
                        a.slots[r] = ok && (uint32_t)page < a.pages ? (int32_t)(((uint32_t)page << a.lbs) + (at & (bs - 1))) : -1;
                        a.pos[r] = ok ? (int32_t)at : -1;
                    }
                }
            } else {
                s_end[tid] = in_n; s_need[tid] = in_need; s_back[tid] = in_back;
                s_len[tid] = (int32_t)len;
                s_flag[tid] = ok;
                __syncthreads();
                const uint32_t stride = T * gridDim.x, first = blockIdx.x * T + tid;
                const auto find = [&](const uint32_t *s, uint32_t i) {              // first request whose sum exceeds i
                    uint32_t lo = 0, hi = T - 1;
                    while (lo < hi) {
                        const uint32_t m = (lo + hi) / 2;
                        if (s[m] > i) hi = m; else lo = m + 1;
                    }
                    return lo;
                };
                const uint32_t rows_here = min(total_n, a.rows - min(rows0, a.rows));
                for (uint32_t i = first; i < rows_here; i += stride) {
                    const uint32_t f = find(s_end, i), fl = (uint32_t)s_len[f], at = fl + i - (f ? s_end[f - 1] : 0), j = at >> a.lbs;
                    int32_t slot = -1, p = -1;
                    if (s_flag[f]) {
                        // a page of this step is read from the ring: its table entry is being written
                        const uint32_t hv = (fl + bs - 1) >> a.lbs;
                        const int32_t page = j < hv ? a.table[(uint64_t)(b0 + f) * a.ld + j] : a.pool[ring(need0 + (f ? s_need[f - 1] : 0) + j - hv)];
                        p = (int32_t)at;
                        if ((uint32_t)page < a.pages) slot = (int32_t)(((uint32_t)page << a.lbs) + (at & (bs - 1)));
                    }
                    a.slots[rows0 + i] = slot;
                    a.pos[rows0 + i] = p;
                }
                for (uint32_t i = first; i < total_need; i += stride) {
                    const uint32_t f = find(s_need, i);
                    if (!s_flag[f]) continue;
                    const uint32_t j = i - (f ? s_need[f - 1] : 0), hv = ((uint32_t)s_len[f] + bs - 1) >> a.lbs;
                    a.table[(uint64_t)(b0 + f) * a.ld + hv + j] = a.pool[ring(need0 + i)];
                }
                for (uint32_t i = first; i < total_back; i += stride) {
                    const uint32_t f = find(s_back, i), j = i - (f ? s_back[f - 1] : 0);
                    a.pool[ring(count + back0 + i)] = a.table[(uint64_t)(b0 + f) * a.ld + j];
                }
            }
        }
        if (a.commit && blockIdx.x == 0 && b < a.B) a.lens_out[b] = ok ? (int32_t)(len + n) : ad < 0 ? 0 : raw;
        rows0 += total_n; need0 += total_need; back0 += total_back;
        if (b0 + T < a.B) __syncthreads();                           // the next chunk's sums
    }
    if (a.fill)
        for (uint64_t i = (uint64_t)rows0 + blockIdx.x * T + tid; i < a.rows; i += T * gridDim.x) {
            a.slots[i] = -1;
            a.pos[i] = -1;
        }
    __syncthreads();
    if (a.commit && blockIdx.x == 0 && tid == 0) {
        a.state_out[0] = (int32_t)ring(s_used);
        a.state_out[1] = (int32_t)min((uint64_t)count - s_used + back0, (uint64_t)a.pages);
        a.state_out[2] = (int32_t)s_refused;
    }
}

// ---- sh_kv_append -------------------------------------------------------------------------------------------------
struct AppendArgs {
    KvCache c;
    const uint16_t *k, *v;
    uint64_t ldk, ldv;
    const int32_t *slots;
    uint32_t rows, rg, row0;
    ShDiv dch, dheads;                     // by dh / 8, by 2 hkv
};

typedef uint16_t us2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ us2 bits2(uint32_t w) { return __builtin_bit_cast(us2, w & 0x7FFF7FFFu); }     // a pair of halves without their signs
// NaN as 0, infinity as the largest half.
__device__ __forceinline__ uint32_t clean1(uint32_t h) {
    const uint32_t a = h & 0x7FFFu;
    return a > 0x7C00u ? 0u : min(a, 0x7BFFu) | (h & 0x8000u);
}
__device__ __forceinline__ uint32_t clean2(uint32_t w) { return clean1(w & 0xFFFFu) | clean1(w >> 16) << 16; }

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
// values a page: 512 items. Bound by HBM: 2 bytes read and 1 written a value; written pages are whole lines in L2 (17 thousand rows of 8 heads
// of 64: 13.5 us, 3.9 TB/s; 64 single rows 4.8 us, one launch).
template <bool FP8, int NT>
__global__ __launch_bounds__(NT) void k_kv_append(AppendArgs a) {
    __shared__ uint32_t s_top[NT / 64];
    const KvCache &c = a.c;
    const uint32_t tid = threadIdx.x, lane = tid & 63, gr = sh_div(blockIdx.x, a.dheads), hv = blockIdx.x - gr * (2 * c.hkv), r0 = a.row0 + gr * a.rg;
    const uint32_t isv = hv >= c.hkv, h = isv ? hv - c.hkv : hv;
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
        const uint32_t bl = sh_div(tid, a.dch), ch = tid - bl * nch, t0 = 4 * (blk0 + bl);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t t = t0 + j;
            x[j] = make_uint4(0, 0, 0, 0);
            if (tid < items && t >= off && t < end) x[j] = sh_ld16_any(src + (uint64_t)(t - off) * ld + 8 * ch);
        }
        // the largest |x| as an integer (halves without their sign are ordered like their bits); only if a NaN or an infinity is
        // among them are these put right, and it is taken again
        uint32_t top;
        for (;;) {
            us2 t = {0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                t = __builtin_elementwise_max(t, __builtin_elementwise_max(bits2(x[j].x), bits2(x[j].y)));
                t = __builtin_elementwise_max(t, __builtin_elementwise_max(bits2(x[j].z), bits2(x[j].w)));
            }
            top = (uint32_t)sh_wave_max((float)max(t.x, t.y));      // (exact)
            if constexpr (NT > 64) {
                __syncthreads();                                    // the last maxima are read
                if (lane == 0) s_top[tid / 64] = top;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NT / 64; ++i) top = max(top, s_top[i]);
            }
            top = __builtin_amdgcn_readfirstlane(top);
            if (top < 0x7C00u) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = make_uint4(clean2(x[j].x), clean2(x[j].y), clean2(x[j].z), clean2(x[j].w));
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
        const bool p2 = !(__builtin_amdgcn_readfirstlane(__float_as_uint(s)) & 0x7FFFFFu);      // (only a caller's own scales are not)
        const float inv = 1.f / s;
        if (tid < items) {
            float v[4][8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = sh_dev_h2f((uint16_t)(w[e / 2] >> (16 * (e & 1))));
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                // the product, and what it lacks for the correctly rounded quotient (Markstein, "Computation of elementary functions on
                // the IBM RISC System/6000 processor", 1990): nothing where s is a power of two
                const float f = v[j / 8][j % 8], q = f * inv;
                v[j / 8][j % 8] = p2 ? q : fmaf(fmaf(-q, s, f), inv, q);
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

// Workgroups with the heads fastest, keys then values: those that run at one time read whole rows and write whole pages.
template <bool FP8, int NT>
void launch_append_nt(AppendArgs a, hipStream_t st) {
    const uint32_t heads = 2 * a.c.hkv, most = (1u << 31) / (heads * NT) * a.rg;            // (a launch has fewer than 2^32 threads)
    a.dheads = sh_make_div(heads);
    for (uint64_t r = 0; r < a.rows; r += most) {
        a.row0 = (uint32_t)r;
        hipLaunchKernelGGL((k_kv_append<FP8, NT>), dim3(sh_cdiv(std::min(a.rows - a.row0, most), a.rg) * heads), dim3(NT), 0, st, a);
    }
}
template <bool FP8>
void launch_append(const AppendArgs &a, hipStream_t st) {
    const uint32_t items = a.c.bs * a.c.dh / 32;
    if (items <= 64) launch_append_nt<FP8, 64>(a, st);
    else if (items <= 128) launch_append_nt<FP8, 128>(a, st);
    else if (items <= 256) launch_append_nt<FP8, 256>(a, st);
    else launch_append_nt<FP8, 512>(a, st);
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
    // One workgroup reads everything before it writes lengths and state in place; several do not, so these are then written by
    // a launch of their own unless they go elsewhere.
    if (rows <= 2048 && B <= 256) {
        hipLaunchKernelGGL(k_kv_slots<256>, dim3(1), dim3(256), 0, st, a);
    } else if (rows <= 4096) {
        hipLaunchKernelGGL(k_kv_slots<1024>, dim3(1), dim3(1024), 0, st, a);
    } else {
        const auto meet = [](uint64_t x, uint64_t y, uint64_t n) { return x < y + n && y < x + n; };
        const uint32_t groups = std::min(sh_cdiv(rows, 1024), 256u);
        const bool apart = !meet(lens, lens_out, (uint64_t)B * 4) && !meet(state, state_out, 12);
        a.commit = apart;
        hipLaunchKernelGGL(k_kv_slots<1024>, dim3(groups), dim3(1024), 0, st, a);
        a.commit = 1; a.fill = 0;
        if (!apart) hipLaunchKernelGGL(k_kv_slots<1024>, dim3(1), dim3(1024), 0, st, a);
    }
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
