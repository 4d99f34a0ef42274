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
#include "kv8_quant.cuh"
#include "launch.h"

namespace n550 {
namespace {

// FP32 bits of the largest magnitude of N words (FP32, or pairs of BF16), infinities
// and NaN being larger than all numbers; FINITE: of the numbers alone.
template <bool F32, bool FINITE, int N>
__device__ __forceinline__ uint32_t abs_max(const uint32_t (&w)[N]) {
    auto only = [](uint32_t a) { return !FINITE || a < 0x7F800000u ? a : 0u; };
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if constexpr (F32) m = max(m, only(w[i] & 0x7FFFFFFFu));
        else if constexpr (FINITE) m = max(m, max(only(w[i] << 16 & 0x7FFF0000u), only(w[i] & 0x7FFF0000u)));
        else m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    }
    return F32 || FINITE ? m : max(m << 16, m & 0xFFFF0000u);
}
// Four codes of four values (2 words of BF16 pairs, or 4 of FP32) times inv.
template <bool F32>
__device__ __forceinline__ uint32_t codes4(const uint32_t *w, float inv) {
    float x[4];
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[i]) * inv;
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16) * inv;
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u) * inv;
        }
    }
    return f32x2_to_e4m3x2(x[0], x[1]) | f32x2_to_e4m3x2(x[2], x[3]) << 16;
}
constexpr uint32_t kHInf = 0x7C007C00u, kHNegInf = 0xFC00FC00u;

// ---------------------------------------------------------------------------
// A few rows per sequence (a decode step, drafted tokens): one warp per (block the
// rows reach, KV head, sequence) does K and V, lane l the dimensions 4 l .. 4 l + 3.
// Bound: latency. All it reads besides ids and positions is requested at once. One
// CTA of 256 threads per (block, K or V head, sequence) took 19 us for 256 rows.
// ---------------------------------------------------------------------------
constexpr int FEW = 8;                                        // most rows per sequence
constexpr int FEW_WARPS = 4;

template <bool F32>
__global__ void __launch_bounds__(FEW_WARPS * 32) kv8_append_few_kernel(const Kv8AppendArgs p, int n_blk, int n_items) {
    constexpr int W = F32 ? 4 : 2;                            // words of a lane's four dimensions
    const int item = blockIdx.x * FEW_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    dep_wait();
    dep_launch();
    if (item >= n_items) return;
    const int kvh = item & 7, s = (item >> 3) / n_blk, nth = (item >> 3) % n_blk;
    const int slot = p.seq_ids[s], p0 = p.pos ? p.pos[s] : p.pos0;
    if (slot < 0 || slot >= p.c.n_slots || p0 < 0 || p0 > p.c.max_len - p.L) return;
    const int b = p0 / KV8_BLOCK + nth, t_blk = b * KV8_BLOCK;
    const int lo = max(p0, t_blk), hi = min(p0 + p.L, t_blk + KV8_BLOCK), n = hi - lo;
    if (n <= 0) return;
    const bool has_old = p0 > t_blk;
    const size_t plane = p.c.plane(slot, kvh), blk = plane * p.c.nb + b;
    uint32_t *bound = p.c.kb ? (uint32_t *)(p.c.kb + blk * 2 * KV8_HD) + lane : nullptr;
    float s_old[2] = {0.f, 0.f};
    uint32_t old_lo = 0, old_hi = 0;
    if (has_old) {
        s_old[0] = p.c.ks[blk];
        s_old[1] = p.c.vs[blk];
        if (bound) { old_lo = bound[0]; old_hi = bound[32]; }
    }
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const void *src = w ? p.v : p.k;
        uint32_t x[FEW][W], all[FEW * W];
#pragma unroll
        for (int i = 0; i < FEW; i++) {
            const size_t o = ((size_t)s * p.L + (lo - p0) + i) * p.ld + kvh * KV8_HD + 4 * lane;
#pragma unroll
            for (int j = 0; j < W; j++) x[i][j] = 0u;
            if (i < n) {
                if constexpr (F32) {
                    const uint4 q = *(const uint4 *)((const float *)src + o);
                    x[i][0] = q.x; x[i][1] = q.y; x[i][2] = q.z; x[i][3] = q.w;
                } else {
                    const uint2 q = *(const uint2 *)((const uint16_t *)src + o);
                    x[i][0] = q.x; x[i][1] = q.y;
                }
            }
#pragma unroll
            for (int j = 0; j < W; j++) all[i * W + j] = x[i][j];
        }
        uint32_t am = __reduce_max_sync(0xFFFFFFFFu, abs_max<F32, false>(all));
        if (am >= 0x7F800000u) am = __reduce_max_sync(0xFFFFFFFFu, abs_max<F32, true>(all));
        const float sc = fmaxf(s_old[w], pow2(scale_exp(am))), inv = inv_pow2(sc), shrink = s_old[w] * inv;
        uint32_t *codes = (uint32_t *)((w ? p.c.v : p.c.k) + (plane * p.c.max_len + t_blk) * KV8_HD) + lane;
        if (has_old && shrink != 1.f)                         // the scale grew
#pragma unroll 8
            for (int r = 0; r < p0 - t_blk; r++) codes[r * 32] = shrink4(codes[r * 32], shrink);
        uint32_t mn[2] = {kHInf, kHInf}, mx[2] = {kHNegInf, kHNegInf};
#pragma unroll
        for (int i = 0; i < FEW; i++) {
            if (i >= n) continue;
            const uint32_t c = codes4<F32>(x[i], inv);
            codes[(lo - t_blk + i) * 32] = c;
            if (w == 0) {
                const uint32_t z = nan_to_zero(c), h0 = e4m3x2_to_f16x2(z & 0xFFFFu), h1 = e4m3x2_to_f16x2(z >> 16);
                mn[0] = hmin2(mn[0], h0); mx[0] = hmax2(mx[0], h0);
                mn[1] = hmin2(mn[1], h1); mx[1] = hmax2(mx[1], h1);
            }
        }
        if (lane == 0) (w ? p.c.vs : p.c.ks)[blk] = sc;
        if (w == 0 && bound) {
            if (has_old) {
                const uint32_t l = shrink4(old_lo, shrink), h = shrink4(old_hi, shrink);
                mn[0] = hmin2(mn[0], e4m3x2_to_f16x2(l & 0xFFFFu)); mn[1] = hmin2(mn[1], e4m3x2_to_f16x2(l >> 16));
                mx[0] = hmax2(mx[0], e4m3x2_to_f16x2(h & 0xFFFFu)); mx[1] = hmax2(mx[1], e4m3x2_to_f16x2(h >> 16));
            }
            bound[0] = f16x2_to_e4m3x2(mn[0]) | f16x2_to_e4m3x2(mn[1]) << 16;
            bound[32] = f16x2_to_e4m3x2(mx[0]) | f16x2_to_e4m3x2(mx[1]) << 16;
        }
    }
}

// ---------------------------------------------------------------------------
// Prompts: one CTA per (block the rows reach, K or V of a KV head, sequence), the
// block's rows in registers between the maximum and the rounding. Bound: HBM, and
// instruction issue close behind it. Thread t takes 8 dimensions (t % 16) of rows
// t / 16, + 16, ..; rounding is monotone, so the bounds are the codes of the rows'
// minima and maxima, which for BF16 take one instruction for two values.
// ---------------------------------------------------------------------------
constexpr int AP_THREADS = 256;
constexpr int AP_WARPS = AP_THREADS / 32;
constexpr int AP_ROWS = AP_THREADS / 16;
constexpr int AP_ITER = KV8_BLOCK / AP_ROWS;

__device__ __forceinline__ uint32_t bmin2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t bmax2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool F32>
__device__ __forceinline__ uint32_t least(uint32_t a, uint32_t b) {
    return F32 ? __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b))) : bmin2(a, b);
}
template <bool F32>
__device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) {
    return F32 ? __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))) : bmax2(a, b);
}
// A word's values with each NaN replaced by 0.
template <bool F32>
__device__ __forceinline__ uint32_t no_nan(uint32_t w) {
    if (F32) return (w & 0x7FFFFFFFu) > 0x7F800000u ? 0u : w;
    if ((w & 0x7FFFu) > 0x7F80u) w &= 0xFFFF0000u;
    if ((w & 0x7FFF0000u) > 0x7F800000u) w &= 0x0000FFFFu;
    return w;
}

template <bool F32>
__global__ void __launch_bounds__(AP_THREADS, F32 ? 4 : 6) kv8_append_kernel(const Kv8AppendArgs p) {
    constexpr int W = F32 ? 8 : 4;                            // words of a thread's eight dimensions
    constexpr uint32_t kInf = F32 ? 0x7F800000u : 0x7F807F80u, kNegInf = F32 ? 0xFF800000u : 0xFF80FF80u;
    __shared__ uint32_t wmax[AP_WARPS];
    __shared__ __align__(16) uint32_t blo[AP_WARPS][16 * W], bhi[AP_WARPS][16 * W];
    dep_wait();
    dep_launch();
    const int s = blockIdx.z, kvh = blockIdx.y & 7;
    const bool is_v = blockIdx.y >= 8;
    const int slot = p.seq_ids[s], p0 = p.pos ? p.pos[s] : p.pos0;
    if (slot < 0 || slot >= p.c.n_slots || p0 < 0 || p0 > p.c.max_len - p.L) return;
    const int b = p0 / KV8_BLOCK + blockIdx.x, t_blk = b * KV8_BLOCK;
    const int lo = max(p0 - t_blk, 0), hi = min(p0 + p.L - t_blk, KV8_BLOCK);       // rows of the block
    if (lo >= hi) return;
    const size_t plane = p.c.plane(slot, kvh), blk = plane * p.c.nb + b;
    const int c16 = threadIdx.x & 15, r0 = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint2 *codes = (uint2 *)((is_v ? p.c.v : p.c.k) + (plane * p.c.max_len + t_blk + r0) * KV8_HD) + c16;
    float *scale = (is_v ? p.c.vs : p.c.ks) + blk;
    constexpr int E = F32 ? 4 : 2;                            // bytes of a value
    // (t_blk - p0 may be negative: rows below lo are not read)
    const char *src = (const char *)(is_v ? p.v : p.k) +
                      (((long long)s * p.L + (t_blk - p0) + r0) * p.ld + kvh * KV8_HD + 8 * c16) * E;
    const size_t step = (size_t)AP_ROWS * p.ld * E;

    uint32_t x[AP_ITER][W];
#pragma unroll
    for (int i = 0; i < AP_ITER; i++) {
        const int r = r0 + i * AP_ROWS;
#pragma unroll
        for (int j = 0; j < W; j++) x[i][j] = 0u;
        if (r < lo || r >= hi) continue;
        const uint4 *q = (const uint4 *)(src + i * step);
        const uint4 a = __ldcs(q);
        x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w;
        if constexpr (F32) {
            const uint4 d = __ldcs(q + 1);
            x[i][4] = d.x; x[i][5] = d.y; x[i][6] = d.z; x[i][7] = d.w;
        }
    }
    const bool has_old = lo > 0;
    const float s_old = has_old ? *scale : 0.f;
    const bool want = !is_v && p.c.kb;
    uint32_t am = 0, mn[W], mx[W];
#pragma unroll
    for (int j = 0; j < W; j++) { mn[j] = kInf; mx[j] = kNegInf; }
#pragma unroll
    for (int i = 0; i < AP_ITER; i++) am = max(am, abs_max<F32, false>(x[i]));
    am = __reduce_max_sync(0xFFFFFFFFu, am);
    const bool strange = am >= 0x7F800000u;                   // an infinity or a NaN in the warp's rows: a branch of its own
    if (strange) {
        am = 0;
#pragma unroll
        for (int i = 0; i < AP_ITER; i++) am = max(am, abs_max<F32, true>(x[i]));
        am = __reduce_max_sync(0xFFFFFFFFu, am);
    }
    if (want) {
#pragma unroll
        for (int i = 0; i < AP_ITER; i++) {
            const int r = r0 + i * AP_ROWS;
            if (r < lo || r >= hi) continue;
            if (strange) {
#pragma unroll
                for (int j = 0; j < W; j++) {
                    mn[j] = least<F32>(mn[j], no_nan<F32>(x[i][j]));
                    mx[j] = most<F32>(mx[j], no_nan<F32>(x[i][j]));
                }
            } else {
#pragma unroll
                for (int j = 0; j < W; j++) {
                    mn[j] = least<F32>(mn[j], x[i][j]);
                    mx[j] = most<F32>(mx[j], x[i][j]);
                }
            }
        }
    }
    if (lane == 0) wmax[warp] = am;
    if (want) {                                               // over the warp's two rows per step
#pragma unroll
        for (int j = 0; j < W; j++) {
            mn[j] = least<F32>(mn[j], __shfl_xor_sync(0xFFFFFFFFu, mn[j], 16));
            mx[j] = most<F32>(mx[j], __shfl_xor_sync(0xFFFFFFFFu, mx[j], 16));
        }
        if (lane < 16)
#pragma unroll
            for (int j = 0; j < W; j += 4) {
                *(uint4 *)&blo[warp][W * lane + j] = make_uint4(mn[j], mn[j + 1], mn[j + 2], mn[j + 3]);
                *(uint4 *)&bhi[warp][W * lane + j] = make_uint4(mx[j], mx[j + 1], mx[j + 2], mx[j + 3]);
            }
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < AP_WARPS; w++) am = max(am, wmax[w]);
    const float sc = fmaxf(s_old, pow2(scale_exp(am))), inv = inv_pow2(sc), shrink = s_old * inv;
#pragma unroll
    for (int i = 0; i < AP_ITER; i++) {
        const int r = r0 + i * AP_ROWS;
        uint2 *dst = codes + i * (AP_ROWS * KV8_HD / 8);
        if (r >= lo && r < hi) {
            *dst = make_uint2(codes4<F32>(x[i], inv), codes4<F32>(x[i] + W / 2, inv));
        } else if (r < lo && shrink != 1.f) {                 // held codes, and the scale grew
            const uint2 o = *dst;
            *dst = make_uint2(shrink4(o.x, shrink), shrink4(o.y, shrink));
        }
    }
    if (threadIdx.x == 0) *scale = sc;
    // the bounds of two channels per thread
    if (!want || threadIdx.x >= KV8_HD / 2) return;
    const int d = threadIdx.x;
    float lo2[2], hi2[2];
    if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            uint32_t l = blo[0][2 * d + e], h = bhi[0][2 * d + e];
#pragma unroll
            for (int w = 1; w < AP_WARPS; w++) {
                l = least<F32>(l, blo[w][2 * d + e]);
                h = most<F32>(h, bhi[w][2 * d + e]);
            }
            lo2[e] = __uint_as_float(l);
            hi2[e] = __uint_as_float(h);
        }
    } else {
        uint32_t l = blo[0][d], h = bhi[0][d];
#pragma unroll
        for (int w = 1; w < AP_WARPS; w++) {
            l = least<F32>(l, blo[w][d]);
            h = most<F32>(h, bhi[w][d]);
        }
        lo2[0] = __uint_as_float(l << 16); lo2[1] = __uint_as_float(l & 0xFFFF0000u);
        hi2[0] = __uint_as_float(h << 16); hi2[1] = __uint_as_float(h & 0xFFFF0000u);
    }
    uint32_t cl = f32x2_to_e4m3x2(lo2[0] * inv, lo2[1] * inv), ch = f32x2_to_e4m3x2(hi2[0] * inv, hi2[1] * inv);
    uint16_t *kb = (uint16_t *)(p.c.kb + blk * 2 * KV8_HD) + d;
    if (has_old) {
        cl = f16x2_to_e4m3x2(hmin2(e4m3x2_to_f16x2(cl), e4m3x2_to_f16x2(shrink4(kb[0], shrink) & 0xFFFFu)));
        ch = f16x2_to_e4m3x2(hmax2(e4m3x2_to_f16x2(ch), e4m3x2_to_f16x2(shrink4(kb[KV8_HD / 2], shrink) & 0xFFFFu)));
    }
    kb[0] = (uint16_t)cl;
    kb[KV8_HD / 2] = (uint16_t)ch;
}

}  // namespace

int launch_kv8_append(cudaStream_t st, const Kv8AppendArgs &a, bool f32, int n_seqs) {
    const int n_blk = (a.L + KV8_BLOCK - 2) / KV8_BLOCK + 1;  // blocks that L rows can touch
    if (a.L <= FEW) {
        const int items = n_blk * KV8_NKV * n_seqs;
        const dim3 grid((items + FEW_WARPS - 1) / FEW_WARPS);
        if (f32)
            N550_CUDA_TRY(launch_k(kv8_append_few_kernel<true>, grid, FEW_WARPS * 32, 0, st, a, n_blk, items));
        else
            N550_CUDA_TRY(launch_k(kv8_append_few_kernel<false>, grid, FEW_WARPS * 32, 0, st, a, n_blk, items));
    } else {
        const dim3 grid(n_blk, 2 * KV8_NKV, n_seqs);
        if (f32)
            N550_CUDA_TRY(launch_k(kv8_append_kernel<true>, grid, AP_THREADS, 0, st, a));
        else
            N550_CUDA_TRY(launch_k(kv8_append_kernel<false>, grid, AP_THREADS, 0, st, a));
    }
    N550_LAUNCH_CHECK();
    return N550_OK;
}

}  // namespace n550
