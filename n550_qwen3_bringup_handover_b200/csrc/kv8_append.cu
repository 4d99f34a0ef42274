// Quantising append to the 8-bit KV cache.
//
// For each block of 64 positions that the new rows reach, and each KV head:
//   s_new = the smallest power of two with max |x| <= 448 s over the block's new
//           rows (finite values), s = max(s_old, s_new) when the block already
//           holds positions below the first new one, else s_new;
//   held codes  c' = e4m3(c s_old / s)   (only when the scale grew)
//   new codes   c  = e4m3(x / s)         round to nearest even.
// A power of two costs an e4m3 code nothing (its precision is relative) and makes
// every step above exact but for the one rounding; held codes lose bits only
// where they fall below 2^-6. Rounding is monotone, so the extreme codes of a
// block and channel, rescaled like the codes, stay its extreme codes.
#include "kv8.h"
#include "launch.h"

namespace n550 {
namespace {

constexpr int AP_THREADS = 256;
constexpr int AP_ROWS = AP_THREADS / 16;                  // rows in flight: 16 threads x 8 dims each
constexpr int AP_ITER = KV8_BLOCK / AP_ROWS;

template <bool F32>
__device__ __forceinline__ void load8(const void *base, size_t off, float (&x)[8]) {
    if constexpr (F32) {
        const float4 *p = (const float4 *)((const float *)base + off);
        const float4 a = p[0], b = p[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 a = *(const uint4 *)((const uint16_t *)base + off);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
}

// Exponent e of the smallest power of two 2^e with amax <= 448 * 2^e, at least
// -126 (so that the scale and its reciprocal are normal numbers).
__device__ __forceinline__ int scale_exp(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u);
    return max(e, -126);
}

// One CTA per (block the rows reach, K or V of a KV head, sequence).
template <bool F32>
__global__ void __launch_bounds__(AP_THREADS) kv8_append_kernel(const Kv8AppendArgs p) {
    __shared__ uint32_t wmax[AP_THREADS / 32];
    __shared__ float blo[AP_THREADS / 32][KV8_HD], bhi[AP_THREADS / 32][KV8_HD];
    dep_wait();
    dep_launch();
    const int s = blockIdx.z, kvh = blockIdx.y & 7;
    const bool is_v = blockIdx.y >= 8;
    const int slot = p.seq_ids[s], p0 = p.pos[s];
    if (slot < 0 || slot >= p.c.n_slots || p0 < 0 || p0 > p.c.max_len - p.L) return;
    const int b = p0 / KV8_BLOCK + blockIdx.x, t_blk = b * KV8_BLOCK;
    const int lo = max(p0, t_blk), hi = min(p0 + p.L, t_blk + KV8_BLOCK);
    if (lo >= hi) return;
    const size_t plane = p.c.plane(slot, kvh);
    uint8_t *codes = (is_v ? p.c.v : p.c.k) + (plane * p.c.max_len + t_blk) * KV8_HD;
    float *scale = (is_v ? p.c.vs : p.c.ks) + plane * p.c.nb + b;
    const void *src = is_v ? p.v : p.k;
    const int c8 = (threadIdx.x & 15) * 8, r0 = threadIdx.x >> 4, warp = threadIdx.x >> 5;

    float x[AP_ITER][8];
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < AP_ITER; i++) {
        const int t = t_blk + r0 + i * AP_ROWS;
        if (t < lo || t >= hi) continue;
        load8<F32>(src, ((size_t)s * p.L + (t - p0)) * p.ld + kvh * KV8_HD + c8, x[i]);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t a = __float_as_uint(x[i][j]) & 0x7FFFFFFFu;
            am = a < 0x7F800000u ? max(am, a) : am;
        }
    }
    am = __reduce_max_sync(0xFFFFFFFFu, am);
    if ((threadIdx.x & 31) == 0) wmax[warp] = am;
    const bool has_old = p0 > t_blk;
    const float s_old = has_old ? *scale : 0.f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < AP_THREADS / 32; w++) am = max(am, wmax[w]);
    const float s_new = __uint_as_float((uint32_t)(scale_exp(am) + 127) << 23);
    const float sc = fmaxf(s_old, s_new);
    const float inv = __uint_as_float((254u << 23) - __float_as_uint(sc));   // 1 / 2^e
    const float shrink = s_old * inv;

    float mn[8], mx[8];
#pragma unroll
    for (int j = 0; j < 8; j++) { mn[j] = INFINITY; mx[j] = -INFINITY; }
#pragma unroll
    for (int i = 0; i < AP_ITER; i++) {
        const int r = r0 + i * AP_ROWS, t = t_blk + r;
        uint8_t *dst = codes + (size_t)r * KV8_HD + c8;
        if (t >= lo && t < hi) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                w[j] = f32x2_to_e4m3x2(x[i][2 * j] * inv, x[i][2 * j + 1] * inv);
                const float2 f = e4m3x2_to_f32x2(w[j]);
                const float a = f.x == f.x ? f.x : 0.f, c = f.y == f.y ? f.y : 0.f;   // NaN counts as 0
                mn[2 * j] = fminf(mn[2 * j], a);
                mx[2 * j] = fmaxf(mx[2 * j], a);
                mn[2 * j + 1] = fminf(mn[2 * j + 1], c);
                mx[2 * j + 1] = fmaxf(mx[2 * j + 1], c);
            }
            *(uint2 *)dst = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
        } else if (t < lo && has_old && shrink != 1.f) {
            const uint2 o = *(const uint2 *)dst;
            uint32_t w[4] = {o.x & 0xFFFFu, o.x >> 16, o.y & 0xFFFFu, o.y >> 16};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = e4m3x2_to_f32x2(w[j]);
                w[j] = f32x2_to_e4m3x2(f.x * shrink, f.y * shrink);
            }
            *(uint2 *)dst = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
        }
    }
    if (threadIdx.x == 0) *scale = sc;
    if (is_v || !p.c.kb) return;
    // bounds: over the warp's two rows per pass, then over the warps
#pragma unroll
    for (int j = 0; j < 8; j++) {
        mn[j] = fminf(mn[j], __shfl_xor_sync(0xFFFFFFFFu, mn[j], 16));
        mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xFFFFFFFFu, mx[j], 16));
        if ((threadIdx.x & 31) < 16) { blo[warp][c8 + j] = mn[j]; bhi[warp][c8 + j] = mx[j]; }
    }
    __syncthreads();
    if (threadIdx.x < KV8_HD) {
        const int d = threadIdx.x;
        float l = blo[0][d], h = bhi[0][d];
#pragma unroll
        for (int w = 1; w < AP_THREADS / 32; w++) {
            l = fminf(l, blo[w][d]);
            h = fmaxf(h, bhi[w][d]);
        }
        uint8_t *kb = p.c.kb + (plane * p.c.nb + b) * 2 * KV8_HD + d;
        if (has_old) {
            const float2 o = e4m3x2_to_f32x2((uint32_t)kb[0] | ((uint32_t)kb[KV8_HD] << 8));
            const uint32_t r = f32x2_to_e4m3x2(o.x * shrink, o.y * shrink);
            const float2 q = e4m3x2_to_f32x2(r);
            l = fminf(l, q.x);
            h = fmaxf(h, q.y);
        }
        const uint32_t r = f32x2_to_e4m3x2(l, h);
        kb[0] = (uint8_t)r;
        kb[KV8_HD] = (uint8_t)(r >> 8);
    }
}

}  // namespace

int launch_kv8_append(cudaStream_t st, const Kv8AppendArgs &a, bool f32, int n_seqs) {
    const dim3 grid((a.L + KV8_BLOCK - 2) / KV8_BLOCK + 1, 2 * KV8_NKV, n_seqs);
    if (f32)
        N550_CUDA_TRY(launch_k(kv8_append_kernel<true>, grid, AP_THREADS, 0, st, a));
    else
        N550_CUDA_TRY(launch_k(kv8_append_kernel<false>, grid, AP_THREADS, 0, st, a));
    N550_LAUNCH_CHECK();
    return N550_OK;
}

}  // namespace n550
