// Quantising one row into the 8-bit KV cache, shared by the append kernels and the
// runtime's row kernel (kv8_append.cu has the definitions).
#pragma once

#include "kv8.h"

namespace n550 {

// Exponent e of the smallest power of two 2^e with amax <= 448 * 2^e, at least
// -126 (so that the scale and its reciprocal are normal numbers).
__device__ __forceinline__ int scale_exp(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u);
    return max(e, -126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// 1 / s of a power of two with exponent in [-126, 120]
__device__ __forceinline__ float inv_pow2(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// Four held codes at a scale 1 / shrink times larger.
__device__ __forceinline__ uint32_t shrink4(uint32_t c, float shrink) {
    const float2 a = e4m3x2_to_f32x2(c & 0xFFFFu), b = e4m3x2_to_f32x2(c >> 16);
    return f32x2_to_e4m3x2(a.x * shrink, a.y * shrink) | f32x2_to_e4m3x2(b.x * shrink, b.y * shrink) << 16;
}
// Codes with each NaN (0x7F, 0xFF) replaced by 0: what a NaN counts as in the bounds.
__device__ __forceinline__ uint32_t nan_to_zero(uint32_t c) {
    const uint32_t n = ((c & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;     // 0x80 at each NaN
    return n ? c & ~((n >> 7) * 0xFFu) : c;
}
__device__ __forceinline__ uint32_t hmin2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t hmax2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Appends one row of K or V (is_v) of a slot and KV head at `pos`, a warp with lane l
// holding the dimensions l + 32 j (BF16 values). The same codes, scales and bounds as
// the append kernels'. A row outside the cache is skipped.
__device__ __forceinline__ void kv8_put_row(const Kv8View &c, int slot, int kvh, bool is_v, int pos, const float (&x)[4],
                                            int lane) {
    if (slot < 0 || slot >= c.n_slots || pos < 0 || pos >= c.max_len) return;
    const int b = pos / KV8_BLOCK, held = pos % KV8_BLOCK;
    const size_t plane = c.plane(slot, kvh), blk = plane * c.nb + b;
    float *scale = (is_v ? c.vs : c.ks) + blk;
    uint8_t *bound = !is_v && c.kb ? c.kb + blk * 2 * KV8_HD + lane : nullptr;
    const float s_old = held ? *scale : 0.f;
    uint32_t lo = 0, hi = 0;
    if (held && bound)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            lo |= (uint32_t)bound[32 * j] << (8 * j);
            hi |= (uint32_t)bound[KV8_HD + 32 * j] << (8 * j);
        }
    uint32_t am = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t a = __float_as_uint(x[j]) & 0x7FFFFFFFu;
        if (a < 0x7F800000u) am = max(am, a);                 // infinities and NaN do not count
    }
    am = __reduce_max_sync(0xFFFFFFFFu, am);
    const float sc = fmaxf(s_old, pow2(scale_exp(am))), inv = inv_pow2(sc), shrink = s_old * inv;
    uint8_t *codes = (is_v ? c.v : c.k) + (plane * c.max_len + (size_t)b * KV8_BLOCK) * KV8_HD;
    if (held && shrink != 1.f) {                              // the scale grew
        uint32_t *w = (uint32_t *)codes + lane;
#pragma unroll 8
        for (int r = 0; r < held; r++) w[r * 32] = shrink4(w[r * 32], shrink);
    }
    const uint32_t code = f32x2_to_e4m3x2(x[0] * inv, x[1] * inv) | f32x2_to_e4m3x2(x[2] * inv, x[3] * inv) << 16;
#pragma unroll
    for (int j = 0; j < 4; j++) codes[held * KV8_HD + lane + 32 * j] = (uint8_t)(code >> (8 * j));
    if (lane == 0) *scale = sc;
    if (!bound) return;
    uint32_t mn = nan_to_zero(code), mx = mn;
    if (held) {
        lo = shrink4(lo, shrink);
        hi = shrink4(hi, shrink);
        mn = f16x2_to_e4m3x2(hmin2(e4m3x2_to_f16x2(mn & 0xFFFFu), e4m3x2_to_f16x2(lo & 0xFFFFu))) |
             f16x2_to_e4m3x2(hmin2(e4m3x2_to_f16x2(mn >> 16), e4m3x2_to_f16x2(lo >> 16))) << 16;
        mx = f16x2_to_e4m3x2(hmax2(e4m3x2_to_f16x2(mx & 0xFFFFu), e4m3x2_to_f16x2(hi & 0xFFFFu))) |
             f16x2_to_e4m3x2(hmax2(e4m3x2_to_f16x2(mx >> 16), e4m3x2_to_f16x2(hi >> 16))) << 16;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        bound[32 * j] = (uint8_t)(mn >> (8 * j));
        bound[KV8_HD + 32 * j] = (uint8_t)(mx >> (8 * j));
    }
}

}  // namespace n550
