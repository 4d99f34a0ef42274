// Block selection over the 8-bit KV cache: the blocks of 64 positions whose K
// bounds promise the largest scores for a query.
//
//   score_b = s_b * max over the KV head's two query heads of
//             sum_d max(q_d lo_bd, q_d hi_bd)
// with lo / hi the block's smallest / largest code of channel d and s_b its K
// scale: no q . k_t of the block is larger. The first n_sink and the last
// n_recent blocks of the context are always taken, then the largest scores, the
// lower index first among equals. Scores are summed in binary64: they decide an
// order, so a result must not depend on the order of the sum.
#include "kv8.h"
#include "launch.h"

namespace n550 {
namespace {

constexpr int SL_THREADS = 256;

// One CTA per (KV head, sequence); scores in shared memory, a block's rank is
// the number of blocks before it.
__global__ void __launch_bounds__(SL_THREADS) kv8_select_kernel(const Kv8SelectArgs p) {
    extern __shared__ double sc[];
    __shared__ int n_out, wcnt[SL_THREADS / 32];
    dep_wait();
    dep_launch();
    const int kvh = blockIdx.x, s = blockIdx.y;
    const int slot = p.seq_ids[s];
    const int nb = (kv8_ctx(p.c, slot, p.pos[s]) + KV8_BLOCK - 1) / KV8_BLOCK;
    int32_t *out = p.blocks + ((size_t)s * KV8_NKV + kvh) * p.n_select;
    const size_t plane = nb ? p.c.plane(slot, kvh) : 0;
    const uint16_t *q = p.q + (size_t)s * p.ldq + 2 * kvh * KV8_HD;
    for (int b = threadIdx.x; b < nb; b += SL_THREADS) {
        const uint8_t *kb = p.c.kb + (plane * p.c.nb + b) * 2 * KV8_HD;
        double a[2] = {0., 0.};
        for (int d = 0; d < KV8_HD; d += 2) {
            const float2 lo = e4m3x2_to_f32x2(*(const uint16_t *)(kb + d));
            const float2 hi = e4m3x2_to_f32x2(*(const uint16_t *)(kb + KV8_HD + d));
            for (int h = 0; h < 2; h++) {
                const double q0 = bf16_bits_to_f32(q[h * KV8_HD + d]), q1 = bf16_bits_to_f32(q[h * KV8_HD + d + 1]);
                a[h] += fmax(q0 * lo.x, q0 * hi.x);
                a[h] += fmax(q1 * lo.y, q1 * hi.y);
            }
        }
        double v = fmax(a[0], a[1]) * p.c.ks[plane * p.c.nb + b];
        if (!(v == v)) v = -INFINITY;
        if (b < p.n_sink || b >= nb - p.n_recent) v = INFINITY;
        sc[b] = v;
    }
    if (threadIdx.x == 0) n_out = 0;
    __syncthreads();
    for (int base = 0; base < nb; base += SL_THREADS) {
        const int b = base + threadIdx.x;
        bool take = false;
        if (b < nb) {
            int rank = 0;
            for (int i = 0; i < nb; i++) rank += sc[i] > sc[b] || (sc[i] == sc[b] && i < b);
            take = rank < p.n_select;
        }
        // ascending output: the taken blocks before this one
        const uint32_t bal = __ballot_sync(0xFFFFFFFFu, take);
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) wcnt[warp] = __popc(bal);
        __syncthreads();
        int at = n_out + __popc(bal & ((1u << lane) - 1u));
        for (int w = 0; w < warp; w++) at += wcnt[w];
        if (take) out[at] = b;
        __syncthreads();
        if (threadIdx.x == 0)
            for (int w = 0; w < SL_THREADS / 32; w++) n_out += wcnt[w];
        __syncthreads();
    }
    for (int i = min(nb, p.n_select) + threadIdx.x; i < p.n_select; i += SL_THREADS) out[i] = -1;
}

}  // namespace

int launch_kv8_select(cudaStream_t st, const Kv8SelectArgs &a) {
    const size_t smem = (size_t)a.c.nb * sizeof(double);
    N550_CUDA_TRY(cudaFuncSetAttribute(kv8_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)smem));
    N550_CUDA_TRY(launch_k(kv8_select_kernel, dim3(KV8_NKV, a.n_seqs), SL_THREADS, smem, st, a));
    N550_LAUNCH_CHECK();
    return N550_OK;
}

}  // namespace n550
