// Attention over the 8-bit KV cache: for query position p and head h (KV head
// h / 2), s_t = (q . k_t) * 0.08838834764831845 over t = 0..p (or over the
// positions of the listed blocks), softmax over t, out = sum_t softmax_t * v_t,
// with k_t and v_t the codes times their block's scale.
#include "kv8.h"
#include "launch.h"

namespace n550 {
namespace {

constexpr int AT_THREADS = 128;
constexpr int AT_WARPS = AT_THREADS / 32;

// One CTA per (query, KV head, sequence); a warp takes one position at a time,
// lane l the dimensions 4 l .. 4 l + 3 of both query heads.
__global__ void __launch_bounds__(AT_THREADS) kv8_prefill_kernel(const Kv8AttnArgs p) {
    __shared__ float wm[AT_WARPS][2], wl[AT_WARPS][2];
    __shared__ float wo[AT_WARPS][2][KV8_HD];
    dep_wait();
    dep_launch();
    const int j = blockIdx.x, kvh = blockIdx.y, s = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slot = p.seq_ids[s];
    const int len = kv8_ctx(p.c, slot, p.pos ? p.pos[s] : p.pos0 + j);
    const size_t row = (size_t)s * p.L + j, plane = len ? p.c.plane(slot, kvh) : 0;
    const uint8_t *kc = p.c.k + plane * p.c.max_len * KV8_HD, *vc = p.c.v + plane * p.c.max_len * KV8_HD;
    float q[2][4], o[2][4], m[2], l[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        m[h] = -INFINITY;
        l[h] = 0.f;
#pragma unroll
        for (int d = 0; d < 4; d++) {
            q[h][d] = bf16_bits_to_f32(p.q[row * p.ldq + (2 * kvh + h) * KV8_HD + 4 * lane + d]);
            o[h][d] = 0.f;
        }
    }
    const int n_items = p.n_select >= 0 ? p.n_select : (len + KV8_BLOCK - 1) / KV8_BLOCK;
    for (int i = 0; i < n_items; i++) {
        const int b = p.n_select >= 0 ? p.blocks[((size_t)s * KV8_NKV + kvh) * p.n_select + i] : i;
        if (b < 0 || (long long)b * KV8_BLOCK >= len) continue;
        const float ks = p.c.ks[plane * p.c.nb + b] * kKv8ScaleLog2, vs = p.c.vs[plane * p.c.nb + b];
        const int end = min(len, (b + 1) * KV8_BLOCK);
        for (int t = b * KV8_BLOCK + warp; t < end; t += AT_WARPS) {
            const uint32_t kw = *(const uint32_t *)(kc + (size_t)t * KV8_HD + 4 * lane);
            const uint32_t vw = *(const uint32_t *)(vc + (size_t)t * KV8_HD + 4 * lane);
            const float2 k0 = e4m3x2_to_f32x2(kw & 0xFFFFu), k1 = e4m3x2_to_f32x2(kw >> 16);
            const float2 v0 = e4m3x2_to_f32x2(vw & 0xFFFFu), v1 = e4m3x2_to_f32x2(vw >> 16);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float d = q[h][0] * k0.x + q[h][1] * k0.y + q[h][2] * k1.x + q[h][3] * k1.y;
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) d += __shfl_xor_sync(0xFFFFFFFFu, d, x);
                d *= ks;
                const float mn = fmaxf(m[h], d);
                const float c = m[h] == -INFINITY ? 0.f : exp2f(m[h] - mn);
                const float e = mn == -INFINITY ? 0.f : exp2f(d - mn);
                m[h] = mn;
                l[h] = l[h] * c + e;
                const float w = e * vs;
                o[h][0] = o[h][0] * c + w * v0.x;
                o[h][1] = o[h][1] * c + w * v0.y;
                o[h][2] = o[h][2] * c + w * v1.x;
                o[h][3] = o[h][3] * c + w * v1.y;
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (lane == 0) { wm[warp][h] = m[h]; wl[warp][h] = l[h]; }
#pragma unroll
        for (int d = 0; d < 4; d++) wo[warp][h][4 * lane + d] = o[h][d];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * KV8_HD; i += AT_THREADS) {
        const int h = i >> 7, d = i & 127;
        float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < AT_WARPS; w++) M = fmaxf(M, wm[w][h]);
#pragma unroll
        for (int w = 0; w < AT_WARPS; w++) {
            const float f = wm[w][h] == -INFINITY ? 0.f : exp2f(wm[w][h] - M);
            L += wl[w][h] * f;
            O += wo[w][h][d] * f;
        }
        p.out[row * p.ldo + (2 * kvh + h) * KV8_HD + d] = f32_to_bf16_rne(L > 0.f ? O / L : L == 0.f ? 0.f : L);
    }
}

}  // namespace


int launch_kv8_prefill(cudaStream_t st, const Kv8AttnArgs &a) {
    N550_CUDA_TRY(launch_k(kv8_prefill_kernel, dim3(a.L, KV8_NKV, a.n_seqs), AT_THREADS, 0, st, a));
    N550_LAUNCH_CHECK();
    return N550_OK;
}

}  // namespace n550
