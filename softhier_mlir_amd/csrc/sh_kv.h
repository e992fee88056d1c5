// What the 8-bit key / value cache's kernels share (not part of the C ABI).
#pragma once
#include "sh_common.h"

// A checked sh_kv_cache with its defaults filled in.
struct KvCache {
    uint8_t *k, *v;
    float *ks, *vs;
    uint64_t pgk, pgv;
    uint32_t pgs, pages, hkv, dh, bs, lbs;     // lbs = log2 bs
};
// 0 and *out, or -1 with the message set.
int sh_kv_check(const char *name, const sh_kv_cache *c, KvCache *out);

// Sum of the lanes up to this one (v_add with DPP moves: shifts within rows of 16, then the rows' last lanes broadcast).
__device__ __forceinline__ uint32_t kv_wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}

// The eight (four) bytes of two (one) words to fp16, exactly. INT8: with the sign bit flipped a byte u = code + 128 under
// the high byte 0x64 is the half 1024 + u; minus 1152. FP8: the hardware's e4m3 conversion.
template <bool FP8>
__device__ __forceinline__ void kv_half4(uint32_t w, sh_h2 &lo, sh_h2 &hi) {
    if constexpr (FP8) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        lo = __builtin_bit_cast(sh_h2, (h2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
        hi = __builtin_bit_cast(sh_h2, (h2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    } else {
        const uint32_t u = w ^ 0x80808080u;
        const sh_h2 b = {(_Float16)1152.0f, (_Float16)1152.0f};
        lo = __builtin_bit_cast(sh_h2, __builtin_amdgcn_perm(0x64646464u, u, 0x07010700u)) - b;
        hi = __builtin_bit_cast(sh_h2, __builtin_amdgcn_perm(0x64646464u, u, 0x07030702u)) - b;
    }
}
template <bool FP8>
__device__ __forceinline__ sh_h8 kv_half8(uint32_t w0, uint32_t w1) {
    sh_h2 a, b, c, d;
    kv_half4<FP8>(w0, a, b);
    kv_half4<FP8>(w1, c, d);
    return sh_h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
