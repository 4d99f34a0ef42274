// Block selection over the 8-bit KV cache: the blocks of 64 positions whose K
// bounds promise the largest scores for a query.
//
//   score_b = s_b * max over the KV head's two query heads of
//             sum_d max(q_d lo_bd, q_d hi_bd)
// with lo / hi the block's smallest / largest code of channel d and s_b its K
// scale: no q . k_t of the block is larger. The maximum takes hi where q_d is
// positive and lo elsewhere. The first n_sink and the last n_recent blocks of the
// context are always taken, then the largest scores, the lower index first among
// equals. Scores are summed in binary64, where products of 8 and 4 significant
// bits add without rounding as long as their exponents stay within 34 binades:
// they decide an order, so a result must not depend on the order of a sum.
//
// Bound: HBM for long contexts (256 bytes of bounds per block and KV head) and
// latency below that: a cluster of CTAs scores the blocks of one (sequence, KV
// head), 8 lanes a block, and sends the scores to its first CTA's shared memory,
// which takes the n_select-th largest by radix (8 bits a pass, from the first bit
// in which the scores differ) and writes the taken indices in order.
#include "kv8.h"
#include "launch.h"

namespace n550 {
namespace {

constexpr int SL_THREADS = 512;                 // one CTA per SM by registers: 32 doubles of query a lane
constexpr int SL_WARPS = SL_THREADS / 32;
constexpr int SL_STEP = 16;                     // blocks a warp scores at a time

// e4m3 codes enter binary64 through FP16: its bits under a binary64 exponent
// field are the value times 2^-1008 (e4m3's subnormal numbers are normal in
// FP16), so queries are taken times 2^512 and sums times 2^496.
__device__ __forceinline__ double widen(uint32_t h_top) {     // FP16 in the upper half, anything in the lower
    return __hiloint2double((int)h_top >> 6 & 0x81FFFC00, 0);
}

// Binary64 -> unsigned with the same order.
__device__ __forceinline__ unsigned long long order_key(double x) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);   // one zero
    return b >> 63 ? ~b : b | 1ull << 63;
}

__device__ __forceinline__ void min_cluster_u32(uint32_t addr, unsigned int v) {
    asm volatile("red.relaxed.cluster.shared::cluster.min.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void max_cluster_u32(uint32_t addr, unsigned int v) {
    asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// One cluster per (KV head, sequence).
__global__ void __launch_bounds__(SL_THREADS) kv8_select_kernel(const Kv8SelectArgs p) {
    extern __shared__ unsigned long long key[];                // [nb] in the cluster's first CTA
    __shared__ unsigned int hist[256];
    __shared__ unsigned int range[2];                          // upper halves of the least and largest key that is not forced
    __shared__ unsigned long long found;                       // digit and counts
    __shared__ int wgt[SL_WARPS], weq[SL_WARPS];
    dep_wait();
    dep_launch();
    const int rank = cluster_ctarank(), cs = cluster_nctarank();
    const int kvh = blockIdx.y, s = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slot = p.seq_ids[s];
    const int nb = (kv8_ctx(p.c, slot, p.pos[s]) + KV8_BLOCK - 1) / KV8_BLOCK;
    int32_t *out = p.blocks + ((size_t)s * KV8_NKV + kvh) * p.n_select;
    if (nb <= p.n_select) {                                    // the same in all CTAs of the cluster
        if (rank == 0)
            for (int i = threadIdx.x; i < p.n_select; i += SL_THREADS) out[i] = i < nb ? i : -1;
        return;
    }
    const size_t plane = p.c.plane(slot, kvh);
    if (threadIdx.x == 0) { range[0] = ~0u; range[1] = 0u; }
    cluster_arrive();                                          // the first CTA is there before it is written to
    const int f0 = p.n_sink, f1 = nb - p.n_recent;             // forced: b < f0 or b >= f1 (n_sink + n_recent <= n_select < nb)

    // ---------------- scores: lane l the dimensions 16 (l % 8) .. of block l / 8 of 4 ----------------
    {
        const int d0 = (lane & 7) * 16;
        double q[2][16];
        uint32_t sel[2][4];                                    // byte selectors: 0-3 lo, 4-7 hi
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint4 *src = (const uint4 *)(p.q + (size_t)s * p.ldq + (2 * kvh + h) * KV8_HD + d0);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint4 x = src[i];
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    q[h][8 * i + 2 * j] = (double)__uint_as_float(w[j] << 16) * 0x1p512;
                    q[h][8 * i + 2 * j + 1] = (double)__uint_as_float(w[j] & 0xFFFF0000u) * 0x1p512;
                    const uint32_t a = w[j] >> 15 & 1, b = w[j] >> 31;
                    const uint32_t n = (2 * (j & 1)) + (a ? 0 : 4) | ((2 * (j & 1) + 1) + (b ? 0 : 4)) << 4;
                    if (j & 1) sel[h][2 * i + (j >> 1)] |= n << 8;
                    else sel[h][2 * i + (j >> 1)] = n;
                }
            }
        }
        const uint32_t dst = mapa_shared(smem_u32(key), 0);
        cluster_wait();
        unsigned int least = ~0u, most = 0u;
        const uint8_t *kb = p.c.kb + plane * p.c.nb * 2 * KV8_HD;
        const float *ks = p.c.ks + plane * p.c.nb;
        for (int b0 = (rank * SL_WARPS + warp) * SL_STEP; b0 < nb; b0 += cs * SL_WARPS * SL_STEP) {
            uint4 lo[4], hi[4];
            float sc[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int b = b0 + 4 * j + (lane >> 3);
                const uint8_t *src = kb + (size_t)min(b, nb - 1) * 2 * KV8_HD + d0;
                lo[j] = __ldcg((const uint4 *)src);
                hi[j] = __ldcg((const uint4 *)(src + KV8_HD));
                sc[j] = __ldcg(ks + min(b, nb - 1));
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t l[4] = {lo[j].x, lo[j].y, lo[j].z, lo[j].w}, g[4] = {hi[j].x, hi[j].y, hi[j].z, hi[j].w};
                double a[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    double e = 0., o = 0.;
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const uint32_t c = __byte_perm(l[w], g[w], sel[h][w]);
                        const uint32_t f = e4m3x2_to_f16x2(c & 0xFFFFu), t = e4m3x2_to_f16x2(c >> 16);
                        e = fma(q[h][4 * w], widen(f << 16), e);
                        o = fma(q[h][4 * w + 1], widen(f), o);
                        e = fma(q[h][4 * w + 2], widen(t << 16), e);
                        o = fma(q[h][4 * w + 3], widen(t), o);
                    }
                    a[h] = e + o;
                }
#pragma unroll
                for (int x = 1; x < 8; x <<= 1) {
                    a[0] += __shfl_xor_sync(0xFFFFFFFFu, a[0], x);
                    a[1] += __shfl_xor_sync(0xFFFFFFFFu, a[1], x);
                }
                const int b = b0 + 4 * j + (lane >> 3);
                if ((lane & 7) == 0 && b < nb) {
                    double v = fmax(a[0], a[1]) * 0x1p496 * (double)sc[j];
                    if (!(v == v)) v = -INFINITY;
                    const unsigned long long x = order_key(v);
                    st_cluster_u64(dst + 8u * b, x);
                    if (b >= f0 && b < f1) {
                        least = min(least, (unsigned int)(x >> 32));
                        most = max(most, (unsigned int)(x >> 32));
                    }
                }
            }
        }
        if ((lane & 7) == 0 && least <= most) {
            const uint32_t r = mapa_shared(smem_u32(range), 0);
            min_cluster_u32(r, least);
            max_cluster_u32(r + 4, most);
        }
    }
    cluster_sync();
    if (rank) return;

    // ---------------- the n_rest largest of the blocks that are not forced ----------------
    const unsigned int lo = range[0], hi = range[1];           // (some block is not forced: nb > n_select)
    int k = p.n_select - p.n_sink - p.n_recent;                // still to take among those equal to `at` above `bits`
    int bits = 64 - __clz(lo ^ hi);                            // key bits not decided yet (32 when the halves are equal)
    unsigned long long at = bits == 64 ? 0 : (unsigned long long)hi << 32 >> bits;   // the decided bits of the k-th largest key
    bool done = k == 0;
    while (bits > 0 && !done) {
        const int take = min(bits, 8), rest = bits - take;
        if (threadIdx.x < 256) hist[threadIdx.x] = 0;
        __syncthreads();
        for (int b = f0 + threadIdx.x; b < f1; b += SL_THREADS) {
            const unsigned long long x = key[b];
            if (bits == 64 || x >> bits == at) atomicAdd(&hist[x >> rest & ((1u << take) - 1u)], 1u);
        }
        __syncthreads();
        if (warp == 0) {
            // lane l: digits 255 - 8 l .. 248 - 8 l, from the largest down
            unsigned int n[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) sum += n[i] = hist[255 - 8 * lane - i];
            unsigned int before = sum;
#pragma unroll
            for (int x = 1; x < 32; x <<= 1) {
                const unsigned int t = __shfl_up_sync(0xFFFFFFFFu, before, x);
                if (lane >= x) before += t;
            }
            before -= sum;                                     // keys with larger digits
            if ((int)before < k && (int)(before + sum) >= k) {
                int i = 0;                                     // the first digit that reaches k
                unsigned int above = before, c = n[0];
#pragma unroll
                for (int m = 1; m < 8; m++)
                    if ((int)(above + c) < k) {
                        above += c;
                        c = n[m];
                        i = m;
                    }
                found = (unsigned long long)(255 - 8 * lane - i) | (unsigned long long)above << 8 | (unsigned long long)c << 32;
            }
        }
        __syncthreads();
        const unsigned long long f = found;
        at = (bits == 64 ? 0 : at << take) | (f & 255);
        bits = rest;
        k -= (int)(f >> 8 & 0xFFFFFFu);
        done = k == (int)(f >> 32);                            // all of that digit: nothing left to decide
    }
    // taken: forced, key above `at`, and the first k equal to it (all of them when done)
    const int per = ((nb + SL_WARPS - 1) / SL_WARPS + 31) & ~31, b_lo = warp * per, b_hi = min(nb, b_lo + per);
    auto side = [&](int b, bool &gt, bool &eq) {
        gt = eq = false;
        if (b >= b_hi) return;
        const unsigned long long x = bits == 64 ? 0 : key[b] >> bits;
        const bool forced = b < f0 || b >= f1;
        gt = forced || x > at;
        eq = !forced && x == at && k > 0;
    };
    int ngt = 0, neq = 0;
    for (int b = b_lo; b < b_hi; b += 32) {
        bool gt, eq;
        side(b + lane, gt, eq);
        ngt += __popc(__ballot_sync(0xFFFFFFFFu, gt));
        neq += __popc(__ballot_sync(0xFFFFFFFFu, eq));
    }
    if (lane == 0) { wgt[warp] = ngt; weq[warp] = neq; }
    __syncthreads();
    int n_gt = 0, n_eq = 0;
    for (int w = 0; w < warp; w++) { n_gt += wgt[w]; n_eq += weq[w]; }
    for (int b = b_lo; b < b_hi; b += 32) {
        bool gt, eq;
        side(b + lane, gt, eq);
        const uint32_t bg = __ballot_sync(0xFFFFFFFFu, gt), be = __ballot_sync(0xFFFFFFFFu, eq), under = (1u << lane) - 1u;
        const int e = n_eq + __popc(be & under);
        if (gt || (eq && e < k)) out[n_gt + __popc(bg & under) + min(e, k)] = b + lane;
        n_gt += __popc(bg);
        n_eq += __popc(be);
    }
}

}  // namespace

int launch_kv8_select(cudaStream_t st, const Kv8SelectArgs &a) {
    const size_t smem = (size_t)a.c.nb * sizeof(unsigned long long);
    static bool attr[64];
    int dev = 0;
    N550_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && !attr[dev]) {
        N550_CUDA_TRY(cudaFuncSetAttribute(kv8_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           N550_KV8_SELECT_MAX_BLOCKS * (int)sizeof(unsigned long long)));
        attr[dev] = true;
    }
    const int pairs = a.n_seqs * KV8_NKV;
    // as many CTAs as fit the 148 SMs at once, up to the portable 8 per cluster (128 pairs:
    // 13 us in clusters of 1, 21 in clusters of 4; 8 pairs: 37 us in clusters of 1, 13 of 8)
    const int cs = pairs <= 18 ? 8 : pairs <= 37 ? 4 : pairs <= 74 ? 2 : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cs, KV8_NKV, a.n_seqs);
    cfg.blockDim = dim3(SL_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cs;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = g_pdl ? 2 : 1;
    N550_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv8_select_kernel, a));
    N550_LAUNCH_CHECK();
    return N550_OK;
}

}  // namespace n550
