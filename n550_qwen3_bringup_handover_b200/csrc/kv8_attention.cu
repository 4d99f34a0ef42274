// Attention of a few queries per sequence over the 8-bit KV cache (decode,
// sparse decode, verification of drafted tokens): for query position p and head
// h (KV head h / 2), s_t = (q . k_t) * 0.08838834764831845 over t = 0..p (or over
// the positions of the listed blocks), softmax over t, out = sum_t softmax_t v_t,
// with k_t and v_t the codes times their block's scale.
//
// Bound: HBM, 256 bytes of codes per position and KV head against 1024 flop per
// query. The work is the list of 64-position blocks of all (sequence, KV head)
// pairs, cut into equal runs, one per CTA: contexts of any mix of lengths load
// the SMs evenly, where one CTA per pair waits for the longest. A run that ends
// inside a pair leaves a partial (max, sum, out) that the combine kernel merges.
//
// The codes are tensor-core operands as they lie in the cache: tiles of 128
// positions (two blocks) go from HBM by TMA into shared memory and from there
// into tcgen05.mma kind::f8f6f4, K as the 128-row side of S^T = K q^T, V (MN-major)
// as the 128-row side of O^T = V^T P^T. No code passes through a register; the
// mma.sync form of this kernel, which turned codes into FP16 there, issued about
// 390 instructions per warp and 16 positions and stopped at 4.7 TB/s (256
// sequences x 1152 positions, 114 us; now 103, 5.2 TB/s). The 16-column side has room for
// queries and weights in e4m3 parts, four bits a part:
//   q = 2^a (h + l / 16): two parts hold a BF16 value whole if it is at least 2^-13 of
//       its head's largest, and a smaller one as a multiple of 2^-20 of that at worst;
//   w = 2^-8 (w1 + w2 / 16 + w3 / 256): a softmax weight is rounded to FP16's 11 bits
//       (2^-12 of it at most), which three parts hold whole, or as a multiple of
//       2^-25 of the tile's largest where it is small.
// Weights are relative to the largest score of their own tile, so each tile's O is
// finished by its MMAs and added up, scaled, in registers: an O that stays in
// TMEM over the tiles has to be scaled there whenever a maximum grows (in 4 of 10
// tiles at 1152 positions). Sums, scores and the softmax state are FP32.
//
//   warp 0     producer: walks the run, 32 blocks a batch (one per lane: list entry,
//              slot, scales), and fills a ring of 32 KB stages
//   warp 1     issues the MMAs, S of the next tile before P.V of this one
//   warps 2-5  softmax, a thread per position, and O, a thread per dimension (of
//              the tile before, once its MMAs are done); they agree on a tile's maximum through shared memory.
//              With more query tokens more such groups share the columns.
//   last warp  splits the queries of each new pair
#include <cuda.h>
#include <float.h>

#include "kv8.h"
#include "launch.h"
#include "tmap.h"

namespace n550 {
namespace {

constexpr int BLK = KV8_BLOCK * KV8_HD;         // 8 KB of K or V codes
constexpr int STAGE = 4 * BLK;                  // K of two blocks | V of two blocks

// What the producer says about a ring stage: one or two blocks of one pair.
struct __align__(16) Rec {
    int blk[2], ctx, flags;                     // blk[0] < 0: nothing to read, blk[1] < 0: one block
    float ks[2], vs[2];
    int s, kvh, slot, pad;                      // partial slot, or -1: the whole pair
};
enum { R_FIRST = 1, R_LAST = 2, R_END = 4, R_Q = 8 };   // of a piece, of the run; the piece's first tile

// How the blocks are laid out along the run axis.
enum { LAY_RAGGED = 0, LAY_EVEN = 1, LAY_PAIR = 2 };
struct Lay {
    int kind;
    int upp;                                    // LAY_EVEN: units per pair
};

// LT: most query tokens (2 heads each) of an instance. S has 4 columns a token, O
// (and P) 6, at most 12 of 16 for each softmax group. A group's P is [128 positions]
// [16 columns] bytes, an MN-major operand without swizzle, so that a position's
// weights are one 16-byte store: column 6 j + 2 k + h is part k of token j, head h.
template <int LT> constexpr int groups() { return LT == 1 ? 1 : LT / 2; }       // of four softmax warps
template <int LT> constexpr int s_cols() { return LT == 1 ? 16 : 4 * LT; }
template <int LT> constexpr int p_cols() { return 16 * groups<LT>(); }
template <int LT> constexpr int tmem_cols() {
    return 2 * (s_cols<LT>() + p_cols<LT>()) <= 64 ? 64 : 2 * (s_cols<LT>() + p_cols<LT>()) <= 128 ? 128 : 256;
}
template <int LT> constexpr int op_bytes() { return 2 * 128 * (s_cols<LT>() + p_cols<LT>()); }
// Ring stages and CTAs per SM: HBM latency takes about 4000 cycles under load and a
// tile's way from full to empty about 2000, so an SM needs some 150 KB of ring; 3 x 2
// stages beat 2 x 3 (256 x 1152 decode 107 against 113 us), because the softmax of
// one CTA alone keeps 13 bytes per cycle of the 23 that HBM gives an SM.
template <int LT> constexpr int stages() { return LT == 8 ? 4 : 2; }
template <int LT> constexpr int per_sm() { return LT == 1 ? 3 : LT == 4 ? 2 : 1; }
template <int LT> constexpr int smem_bytes(int L) { return stages<LT>() * (STAGE + L * 512) + op_bytes<LT>() + 1024; }
template <int LT> constexpr int threads() { return (3 + 4 * groups<LT>()) * 32; }

// The pair that a run leaves to the merge: its pieces are in runs c .. c + n - 1.
struct Cross {
    int s, kvh, n, slot;                        // n = 0: none; slot: the first piece's (2 c or 2 c + 1)
};
// Whether run c's record names a pair of the call and pieces of its runs. Records are
// read from a workspace that nothing initialises; what is merged for one that no run
// wrote has to stay inside it and inside out.
__device__ __forceinline__ bool cross_ok(const Cross &x, int c, int n_runs, int n_seqs) {
    return x.n > 0 && x.n <= n_runs - c && x.s >= 0 && x.s < n_seqs && x.kvh >= 0 && x.kvh < KV8_NKV;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// D[tmem] (+)= A[smem] . B[smem]^T, e4m3 x e4m3 -> FP32, M = 128, K = 32.
__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Instruction descriptor: D FP32, A and B e4m3 (format 0), M = 128; mn: both MN-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int N, int mn) {
    return (1u << 4) | ((uint32_t)mn << 15) | ((uint32_t)mn << 16) | ((uint32_t)(N >> 3) << 17) | ((128u >> 4) << 24);
}

// Shared-memory descriptor of an MN-major 8-bit operand without swizzle: 16 MN
// elements x 8 K rows are 128 bytes in one piece, the next 8 K rows `k_step` and the
// next 16 MN elements `mn_step` bytes on.
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t smem_addr, uint32_t k_step, uint32_t mn_step) {
    return (uint64_t)(smem_addr >> 4 & 0x3FFFu) | (uint64_t)(k_step >> 4) << 16 | (uint64_t)(mn_step >> 4) << 32 |
           (uint64_t)1 << 46;
}

__device__ __forceinline__ void tmem_ld_x4(uint32_t taddr, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
// N columns (2 to 24, loads rounded up to a multiple of 4) of this thread's TMEM lane.
template <int N>
__device__ __forceinline__ void load_cols(uint32_t t, uint32_t (&r)[(N + 3) / 4 * 4]) {
    int at = 0;
    if constexpr (N >= 16) { tmem_ld_32x32b_x16(t, *reinterpret_cast<uint32_t(*)[16]>(&r[0])); at = 16; }
    if constexpr (N % 16 > 4) { tmem_ld_x8(t + at, r + at); at += 8; }
    if constexpr (N % 8 > 0 && N % 8 <= 4) tmem_ld_x4(t + at, r + at);
    tmem_ld_wait();
}
// Maximum over the warp; a NaN counts as nothing.
__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(y) : "f"(x));
    return y;
}
// Whether the phase has completed, without waiting (try_wait may suspend the thread).
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// 2 or 4 consecutive floats in shared memory, aligned to their size.
template <int N>
__device__ __forceinline__ void get_row(const float *p, float (&x)[N]) {
    if constexpr (N == 2) {
        const float2 v = *(const float2 *)p;
        x[0] = v.x; x[1] = v.y;
    } else {
        const float4 v = *(const float4 *)p;
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    }
}
template <int N>
__device__ __forceinline__ void put_row(float *p, const float (&x)[N]) {
    if constexpr (N == 2) *(float2 *)p = make_float2(x[0], x[1]);
    else *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]);
}
// Byte offset of byte k of row n in an operand of 128-byte rows, 128-byte swizzle.
__device__ __forceinline__ uint32_t sw(int n, int k) { return n * 128 + ((((k >> 4) ^ n) & 7) << 4) + (k & 15); }

// Units (blocks; one empty unit for an empty context) of a pair of sequence s.
__device__ __forceinline__ int seq_ctx(const Kv8AttnArgs &p, int s) {
    const int slot = p.seq_ids[s], pos = p.pos ? p.pos[s] : p.pos0 + p.L - 1;   // through L1: every CTA reads them all
    return kv8_ctx(p.c, slot, pos);
}
__device__ __forceinline__ int ctx_blocks(int ctx) { return max(1, (ctx + KV8_BLOCK - 1) / KV8_BLOCK); }

// Cursor into the run axis: sequence s, unit x of its 8 pairs, upp units per pair.
struct Cur {
    int s, upp, ctx, x;
};

// One converged warp. Returns the total number of units and places *cur at unit
// first(total). LAY_RAGGED needs the prefix sums of the sequences' block counts,
// which every CTA forms itself: 256 sequences take one round of loads.
template <class First>
__device__ __forceinline__ long long locate(const Kv8AttnArgs &p, const Lay lay, First first, Cur *cur) {
    if (lay.kind == LAY_EVEN) {
        const long long per = (long long)lay.upp * KV8_NKV, total = per * p.n_seqs, u = first(total);
        if (u >= total) return total;
        cur->s = total >> 31 ? (int)(u / per) : (int)((uint32_t)u / (uint32_t)per);
        cur->x = (int)(u - cur->s * per);
        cur->upp = lay.upp;
        return total;
    }
    // Rounds of 256 sequences, lane l holds l, 32 + l, .. of them: their sums by 32 find the
    // group of 32 that holds the unit, a scan of that group the sequence. (The code
    // runs once, from a cold instruction cache: eight unrolled scans cost 2000 cycles
    // more, and a lane's loads from 8 consecutive sequences 3000.)
    constexpr int ROUND = 8;
    const int lane = threadIdx.x & 31;
    int ctx[ROUND], sum[ROUND];
    auto round = [&](int s0) -> long long {      // returns the round's units
        long long all = 0;
#pragma unroll
        for (int i = 0; i < ROUND; i++) ctx[i] = s0 + 32 * i + lane < p.n_seqs ? seq_ctx(p, s0 + 32 * i + lane) : -KV8_BLOCK;
#pragma unroll
        for (int i = 0; i < ROUND; i++) {
            sum[i] = s0 + 32 * i < p.n_seqs ? __reduce_add_sync(0xFFFFFFFFu, ctx[i] < 0 ? 0 : ctx_blocks(ctx[i])) * KV8_NKV : 0;
            all += sum[i];
        }
        return all;
    };
    long long total = 0;
    for (int s0 = 0; s0 < p.n_seqs; s0 += 32 * ROUND) total += round(s0);
    const long long u = first(total);
    if (u >= total) return total;
    int s0 = 0;
    long long base = 0;                          // units before the round that holds u
    if (p.n_seqs > 32 * ROUND)
        for (;; s0 += 32 * ROUND) {
            const long long n = round(s0);
            if (u < base + n) break;
            base += n;
        }
    long long rest = u - base;
    int mine = ctx[0];
    bool found = rest < sum[0];
#pragma unroll
    for (int i = 1; i < ROUND; i++)
        if (!found) {
            rest -= sum[i - 1];
            s0 += 32;
            mine = ctx[i];
            found = rest < sum[i];
        }
    const int x = (int)rest, n = mine < 0 ? 0 : ctx_blocks(mine) * KV8_NKV;
    int end = n;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xFFFFFFFFu, end, o);
        if (lane >= o) end += t;
    }
    const int l = __ffs(__ballot_sync(0xFFFFFFFFu, x < end)) - 1;
    cur->s = s0 + l;
    cur->ctx = __shfl_sync(0xFFFFFFFFu, mine, l);
    cur->x = x - __shfl_sync(0xFFFFFFFFu, end - n, l);
    cur->upp = ctx_blocks(cur->ctx);
    return total;
}

// Floats before the partials of n runs: the runs' Cross records.
__host__ __device__ __forceinline__ size_t part_base(int n) { return (size_t)n * (sizeof(Cross) / sizeof(float)); }

// `total` units cut into n runs that differ by at most one unit: as many runs as
// CTAs, but none shorter than kMinRun units (a run's blocks are in flight
// together, and each piece costs the merge a partial; one 1152-position context takes
// 12.1, 11.4, 12.8, 13.5 us with runs of at least 1, 2, 4, 6).
constexpr int kMinRun = 2;
struct Cut {
    long long q;
    int n, r;                                   // run c: q units, the first r runs one more
    __device__ __forceinline__ Cut(long long total, int n_max) {
        const long long most = (total + kMinRun - 1) / kMinRun;
        n = most < n_max ? (int)most : n_max;
        q = total >> 31 ? total / n : (long long)((uint32_t)total / (uint32_t)n);
        r = (int)(total - q * n);
    }
    __device__ __forceinline__ long long start(int c) const { return q * c + min(c, r); }
    __device__ __forceinline__ int run_of(long long u) const {
        const long long big = (q + 1) * r;
        return (int)(u < big ? u / (q + 1) : r + (u - big) / q);
    }
};

template <int LT>
__global__ void __launch_bounds__(threads<LT>(), per_sm<LT>())
kv8_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const Kv8AttnArgs p, const Lay lay) {
    constexpr int NS = s_cols<LT>(), NP = p_cols<LT>(), NC = 2 * LT, G = groups<LT>(), ST = stages<LT>();
    extern __shared__ uint8_t dsm[];
    uint8_t *ring = (uint8_t *)(((uintptr_t)dsm + 1023) & ~(uintptr_t)1023);      // [ST][STAGE]
    uint8_t *sQ = ring + ST * STAGE;                                               // [2][NS][128]
    uint8_t *sP = sQ + 2 * NS * 128;                                               // [2][NP][128]
    uint8_t *sraw = sP + 2 * NP * 128;                                             // [ST][L][2 heads x 128 BF16]
    __shared__ Rec rec[ST];
    __shared__ __align__(8) uint64_t full[ST], empty[ST], q_ready[4], q_free[2], s_full[2], p_full[2], pv_done[2], done;
    __shared__ float q_scale[4][NC];            // power of two of each query row, by piece modulo 4
    __shared__ __align__(16) float xmax[2][4][NC], xsum[2][4][NC];
    __shared__ int xdead[G][2][4];
    __shared__ uint32_t tmem_slot;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) { mbar_init(&full[i], 1); mbar_init(&empty[i], 2 + 4 * G); }
        for (int i = 0; i < 2; i++) {
            mbar_init(&q_ready[i], 1);
            mbar_init(&q_ready[2 + i], 1);
            mbar_init(&q_free[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4 * G);
            mbar_init(&pv_done[i], 1);
        }
        mbar_init(&done, 1);
        fence_mbar_init();
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 1) { tmem_alloc(&tmem_slot, tmem_cols<LT>()); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, tS = tmem, tO = tmem + 2 * NS;
    dep_launch();
    // Block lists, positions, scales, codes and queries all come from earlier kernels, and
    // out and the workspace may be in use by them; what every CTA reads first may be on
    // its way to L2 before they end. (All warps wait here: the limits of the waits below
    // do not count the time of earlier kernels.)
    if (warp == 0 && lay.kind == LAY_RAGGED && lane * 32 < p.n_seqs) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.pos + lane * 32));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.seq_ids + lane * 32));
    }
    dep_wait();
    if (warp == 0) {
        Cur cur{};
        int n_units;
        long long u0 = 0, total = 0;
        if (lay.kind == LAY_PAIR) {
            cur.s = blockIdx.x / KV8_NKV;
            cur.ctx = seq_ctx(p, cur.s);
            cur.upp = p.n_select >= 0 ? max(1, p.n_select) : ctx_blocks(cur.ctx);
            cur.x = (int)(blockIdx.x % KV8_NKV) * cur.upp;
            n_units = cur.upp;
        } else {
            long long u1 = 0;
            total = locate(p, lay, [&](long long all) {
                const Cut cut(all, gridDim.x);
                u0 = u1 = all;
                if ((int)blockIdx.x < cut.n) {
                    u0 = cut.start(blockIdx.x);
                    u1 = cut.start(blockIdx.x + 1);
                }
                return u0;
            }, &cur);
            n_units = (int)(u1 - u0);
            // An empty merge record until batch() has the run's last unit: a run whose waits
            // expire before that leaves this one.
            if (lane == 0) ((Cross *)p.part)[blockIdx.x] = Cross{};
            __syncwarp();
        }
        // ---------------- producer: lane i takes unit 32 k + i ----------------
        bool seen = false;                       // the piece that reaches into this batch had a tile
        // The records of the batch of 32 units at `base` (the next one is read while the
        // ring still takes this one: its loads depend on one another three deep).
        auto batch = [&](int base, Rec &me, int &plane, uint32_t &sends) {
            const int i = base + lane;
            me = Rec{};
            bool send = false;
            int ps = i;                          // the run's unit with which the piece begins
            // walk to this lane's unit: whole sequences first
            Cur c = cur;
            if (base + 31 < n_units || i < n_units) {
                c.x += lane;
                while (c.x >= c.upp * KV8_NKV && c.s + 1 < p.n_seqs) {
                    c.x -= c.upp * KV8_NKV;
                    c.s++;
                    if (lay.kind == LAY_RAGGED) {
                        c.ctx = seq_ctx(p, c.s);
                        c.upp = ctx_blocks(c.ctx);
                    }
                }
            }
            me.blk[0] = me.blk[1] = -1;
            plane = 0;
            if (i < n_units) {
                const int slot = p.seq_ids[c.s];
                if (lay.kind == LAY_EVEN) c.ctx = seq_ctx(p, c.s);
                const int kvh = c.x / c.upp, j = c.x - kvh * c.upp;
                int b = j;
                if (p.n_select >= 0)
                    b = p.n_select > 0 ? __ldcg(p.blocks + ((size_t)c.s * KV8_NKV + kvh) * p.n_select + j) : -1;
                if (b < 0 || b > (c.ctx - 1) >> 6) b = -1;      // ctx 0: -1 >> 6 = -1
                me.s = c.s; me.kvh = kvh; me.blk[0] = b; me.ctx = c.ctx;
                me.flags = (i == 0 || j == 0 ? R_FIRST : 0) | (i == n_units - 1 || j == c.upp - 1 ? R_LAST : 0) |
                           (i == n_units - 1 ? R_END : 0);
                // a piece [first unit here .. last unit here] that is not the whole pair
                // is a partial; the one that begins this CTA's run takes slot 2 c
                ps = max(0, i - j);
                const bool head = i - j < 0;                     // the pair begins before this run
                const bool tail = i - j + c.upp > n_units;       // and here ends behind it
                me.slot = head || tail ? 2 * (int)blockIdx.x + (i - j > 0) : -1;
                // tell the merge about the pair that crosses this run's end, if it begins in it
                if (i == n_units - 1 && lay.kind != LAY_PAIR) {
                    Cross x{};
                    if (tail && !head) {
                        x.s = c.s;
                        x.kvh = kvh;
                        x.n = Cut(total, gridDim.x).run_of(u0 + (i - j) + c.upp - 1) - (int)blockIdx.x + 1;
                        x.slot = me.slot;
                    }
                    ((Cross *)p.part)[blockIdx.x] = x;
                }
                if (b >= 0) {
                    plane = (int)p.c.plane(slot, kvh);
                    // the ring's first blocks need not wait for the scales
                    if (i < 2 * ST) {
                        tma_prefetch_3d(&tmK, 0, b * KV8_BLOCK, plane);
                        tma_prefetch_3d(&tmV, 0, b * KV8_BLOCK, plane);
                    }
                    me.ks[0] = __ldcg(p.c.ks + (size_t)plane * p.c.nb + b);
                    me.vs[0] = __ldcg(p.c.vs + (size_t)plane * p.c.nb + b);
                }
                // an unlisted block needs no stage unless its pair begins or ends with it
                send = b >= 0 || (me.flags & (R_FIRST | R_LAST));
            }
            // the queries travel with the piece's first tile
            {
                const bool tile = me.blk[0] >= 0;
                const uint32_t before = __ballot_sync(0xFFFFFFFFu, tile) & ((1u << lane) - 1u) & ~0u << max(0, ps - base);
                const bool earlier = before != 0 || (ps < base && seen);
                if (tile && !earlier) me.flags |= R_Q;
                seen = __shfl_sync(0xFFFFFFFFu, earlier || tile, 31);
            }
            // Lanes 2 i and 2 i + 1 share a stage where both hold a block of one piece
            // and V's scales are near enough for weights in one scale (a factor 8: the
            // small weights of one are then multiples of 2^-22 of its largest instead of 2^-25).
            const int blk = __shfl_down_sync(0xFFFFFFFFu, me.blk[0], 1), fl = __shfl_down_sync(0xFFFFFFFFu, me.flags, 1);
            const float ks = __shfl_down_sync(0xFFFFFFFFu, me.ks[0], 1), vs = __shfl_down_sync(0xFFFFFFFFu, me.vs[0], 1);
            bool two = false;
            if (!(lane & 1) && i + 1 < n_units && me.blk[0] >= 0 && blk >= 0 && !(fl & R_FIRST) &&
                fmaxf(vs, me.vs[0]) <= 8.f * fminf(vs, me.vs[0])) {
                two = true;
                me.blk[1] = blk;
                me.ks[1] = ks;
                me.vs[1] = vs;
                me.flags |= fl;
            }
            if (__shfl_up_sync(0xFFFFFFFFu, (int)two, 1) && (lane & 1)) send = false;
            sends = __ballot_sync(0xFFFFFFFFu, send);
            // the next batch starts behind lane 31's unit
            cur.s = __shfl_sync(0xFFFFFFFFu, c.s, 31);
            cur.upp = __shfl_sync(0xFFFFFFFFu, c.upp, 31);
            cur.ctx = __shfl_sync(0xFFFFFFFFu, c.ctx, 31);
            cur.x = __shfl_sync(0xFFFFFFFFu, c.x, 31) + 1;
        };
        Rec me, nxt;
        int plane, nplane;
        uint32_t sends, nsends;
        if (n_units > 0) {
            batch(0, me, plane, sends);
        } else {                                 // an empty run: one record says so
            me = Rec{};
            me.blk[0] = me.blk[1] = -1;
            me.flags = R_END;
            sends = 1;
            plane = 0;
        }
        int r = 0;                               // records issued
        bool ok = true;
        for (int base = 0; ok; base += 32) {
            bool more = false;
            for (; sends; sends &= sends - 1) {
                const int l = __ffs(sends) - 1, st = r % ST;
                if (lane == l) {
                    ok = mbar_wait(&empty[st], ((r / ST) & 1) ^ 1);
                    if (ok) {
                        rec[st] = me;
                        const int qn = me.flags & R_Q ? p.L : 0;
                        const uint32_t tx = (me.blk[0] >= 0 ? 2 * BLK : 0) + (me.blk[1] >= 0 ? 2 * BLK : 0) + qn * 512;
                        if (tx) mbar_arrive_expect_tx(&full[st], tx);
                        else mbar_arrive(&full[st]);
                        uint8_t *t = ring + st * STAGE;
                        for (int j = 0; j < qn; j++)
                            bulk_load(sraw + (st * p.L + j) * 512,
                                      p.q + ((size_t)me.s * p.rows + p.row0 + j) * p.ldq + me.kvh * 2 * KV8_HD, 512, &full[st]);
                        for (int j = 0; j < 2; j++)
                            if (me.blk[j] >= 0) {
                                tma_load_3d(t + j * BLK, &tmK, &full[st], 0, me.blk[j] * KV8_BLOCK, plane);
                                tma_load_3d(t + (2 + j) * BLK, &tmV, &full[st], 0, me.blk[j] * KV8_BLOCK, plane);
                            }
                    }
                }
                ok = __shfl_sync(0xFFFFFFFFu, ok, l);
                if (!ok) break;
                r++;
                if (!more && base + 32 < n_units) {   // once the batch's first records are on their way
                    more = true;
                    batch(base + 32, nxt, nplane, nsends);
                }
            }
            if (!ok || base + 32 >= n_units) break;
            if (!more) batch(base + 32, nxt, nplane, nsends);
            me = nxt;
            plane = nplane;
            sends = nsends;
        }
        // every load must have landed before the CTA exits: the last ST records
        if (lane == 0)
            for (int i = max(0, r - ST); i < r; i++) mbar_wait(&full[i % ST], (i / ST) & 1);
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMAs ----------------
        constexpr uint32_t id_s = idesc_e4m3(NS, 0), id_o = idesc_e4m3(NP, 1);
        const uint32_t aR = smem_u32(ring), aQ = smem_u32(sQ), aP = smem_u32(sP);
        int t = 0, piece = -1;                   // tiles whose S was issued; this piece with tiles
        int w_st = 0, w_half = 0;                // the tile whose P.V is due
        bool due = false, ok = true;
        // (The softmax has read the O of tile u - 2, this one's columns, before its weights of tile u.)
        auto issue_pv = [&]() -> bool {
            const int u = t - 1, b = u & 1;
            due = false;
            if (!warp_wait(&p_full[b], (u >> 1) & 1)) return false;
            tc_fence_after();
            const uint32_t v = aR + w_st * STAGE + 2 * BLK, pp = aP + b * NP * 128, d = tO + b * NP;
            const int steps = w_half ? 2 : 4;
            for (int k = 0; k < steps; k++)
                if (elect_one_sync())
                    umma_e4m3(d, umma_desc_sw128_mn(v + k * 4096, 0), umma_desc_mn(pp + k * 512, 128, 2048), id_o,
                              k > 0 ? 1u : 0u);
            if (elect_one_sync()) { umma_commit(&empty[w_st]); umma_commit(&pv_done[b]); }
            __syncwarp();
            return true;
        };
        for (int r = 0;; r++) {
            const int st = r % ST;
            // nothing to issue S for yet: the due P.V frees its stage
            if (due && !__all_sync(0xFFFFFFFFu, mbar_test(&full[st], (r / ST) & 1)) && !(ok = issue_pv())) break;
            if (!(ok = warp_wait(&full[st], (r / ST) & 1))) break;
            const Rec w = rec[st];
            if (w.flags & R_Q) {
                // every S of the piece before has been issued
                if (piece >= 0 && elect_one_sync()) umma_commit(&q_free[piece & 1]);
                __syncwarp();
                piece++;
                if (!(ok = warp_wait(&q_ready[piece & 3], (piece >> 2) & 1))) break;
            }
            if (w.blk[0] < 0) {
                if (lane == 0) mbar_arrive(&empty[st]);
            } else {
                tc_fence_after();
                const uint32_t q = aQ + (piece & 1) * NS * 128, k = aR + st * STAGE, d = tS + (t & 1) * NS;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (elect_one_sync())
                        umma_e4m3(d, umma_desc_sw128(k + i * 32), umma_desc_sw128(q + i * 32), id_s, i > 0 ? 1u : 0u);
                if (elect_one_sync()) umma_commit(&s_full[t & 1]);
                __syncwarp();
                // P.V of the tile before, then this one is due
                if (due && !(ok = issue_pv())) break;
                t++;
                due = true;
                w_st = st;
                w_half = w.blk[1] < 0;
            }
            if (w.flags & R_END) break;
        }
        if (ok && due) issue_pv();
        // all MMAs of this warp are done before TMEM is released
        if (elect_one_sync()) umma_commit(&done);
        __syncwarp();
        warp_wait(&done, 0);
    } else if (warp == 2 + 4 * G) {
        // ---------------- query parts: lane i takes dimensions 4 i .. 4 i + 3 ----------------
        int piece = -1;
        for (int r = 0;; r++) {
            const int st = r % ST;
            if (!warp_wait(&full[st], (r / ST) & 1)) break;
            const int flags = rec[st].flags;
            if (flags & R_Q) {
                piece++;
                // the buffer's last piece but one has been multiplied
                if (piece >= 2 && !warp_wait(&q_free[piece & 1], ((piece >> 1) - 1) & 1)) break;
                uint8_t *dst = sQ + (piece & 1) * NS * 128;
#pragma unroll 2
                for (int c = 0; c < 2 * p.L; c++) {
                    const uint2 x2 = *(const uint2 *)(sraw + (st * p.L) * 512 + c * 256 + lane * 8);
                    uint32_t am = max(max(x2.x & 0x7FFFu, x2.x >> 16 & 0x7FFFu), max(x2.y & 0x7FFFu, x2.y >> 16 & 0x7FFFu));
                    am = __reduce_max_sync(0xFFFFFFFFu, am);
                    // the row's largest magnitude to [128, 256)
                    const int e = min(max((int)(am >> 7), 8), 254);
                    const float f = __uint_as_float((uint32_t)(261 - e) << 23);
                    float x[4] = {__uint_as_float(x2.x << 16), __uint_as_float(x2.x & 0xFFFF0000u),
                                  __uint_as_float(x2.y << 16), __uint_as_float(x2.y & 0xFFFF0000u)};
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int k = 0; k < 4; k++) x[k] = fabsf(x[k]) == INFINITY ? NAN : x[k] * f;   // e4m3 has no infinity
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        hi[k] = f32x2_to_e4m3x2(x[2 * k], x[2 * k + 1]);
                        const float2 h = e4m3x2_to_f32x2(hi[k]);
                        lo[k] = f32x2_to_e4m3x2((x[2 * k] - h.x) * 16.f, (x[2 * k + 1] - h.y) * 16.f);
                    }
                    *(uint32_t *)(dst + sw(2 * c, 4 * lane)) = hi[0] | hi[1] << 16;
                    *(uint32_t *)(dst + sw(2 * c + 1, 4 * lane)) = lo[0] | lo[1] << 16;
                    if (lane == 0) q_scale[piece & 3][c] = __uint_as_float((uint32_t)max(e - 7, 1) << 23);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_ready[piece & 3]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
            if (flags & R_END) break;
        }
    } else {
        // ---------------- softmax and output: a group's columns c0 .. c0 + NG - 1 ----------------
        constexpr int NG = NC / G;
        const int grp = (warp - 2) >> 2, c0 = grp * NG, ng = min(NG, 2 * p.L - c0);     // ng <= 0: nothing to do but keep step
        const int qw = warp & 3, row = qw * 32 + lane, half = row >> 6;
        const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
        int t = 0, piece = -1, bars = 0, ends = 0;                 // tiles, pieces with tiles, meetings, ended pieces
        float qf[NG] = {};
        bool dead = false;
        // A group's four warps pass here together, and leave together: after the last
        // record, or when a wait of one of them ran out.
        auto meet = [&](bool mine) -> bool {
            int *d = xdead[grp][bars & 1];
            if (lane == 0) d[qw] = mine;
            named_bar_sync(1 + grp, 128);
            bars++;
            return d[0] | d[1] | d[2] | d[3];
        };
        // The piece so far: maximum, this lane's part of the sum, this lane's dimension of O.
        float m[NG], l[NG], o[NG];
        auto reset = [&]() {
#pragma unroll
            for (int c = 0; c < NG; c++) { m[c] = -INFINITY; l[c] = 0.f; o[c] = 0.f; }
        };
        reset();
        // The last tile whose weights are out: its maximum and sum, V's scale, whether it is owed to the piece.
        float tm[NG], tl[NG], tv = 0.f;
        bool owed = false;
        auto collect = [&]() {
            const int u = t - 1;
            owed = false;
            if (dead || (dead = !warp_wait(&pv_done[u & 1], (u >> 1) & 1))) return;
            uint32_t x[(3 * NG + 3) / 4 * 4];
            tc_fence_after();
            load_cols<3 * NG>(tO + lane_off + (u & 1) * NP + 16 * grp, x);
            tc_fence_before();
#pragma unroll
            for (int c = 0; c < NG; c++) {
                const int n = 6 * (c >> 1) + (c & 1);
                const float part = fmaf(fmaf(__uint_as_float(x[n + 4]), 0.0625f, __uint_as_float(x[n + 2])), 0.0625f,
                                        __uint_as_float(x[n]));
                const float mn = fmaxf(m[c], tm[c]), ref = mn == -INFINITY ? 0.f : mn;
                const float a = ex2(m[c] - ref), b = ex2(tm[c] - ref);
                o[c] = o[c] * a + part * (b * tv);
                l[c] = l[c] * a + tl[c] * b;
                m[c] = mn;
            }
        };
        // Output of the piece that ended: divided by the sum of its weights, or as a
        // partial. False: some warp's wait ran out, all leave.
        bool ending = false;
        int old_s = 0, old_kvh = 0, old_slot = 0;
        auto finish = [&]() -> bool {
            ending = false;
            ends++;
#pragma unroll
            for (int c = 0; c < NG; c++) {
#pragma unroll
                for (int k = 16; k > 0; k >>= 1) l[c] += __shfl_xor_sync(0xFFFFFFFFu, l[c], k);
                if (lane == 0) xsum[ends & 1][qw][c0 + c] = l[c];
            }
            if (meet(dead)) return false;
            const float (*xs)[NC] = xsum[ends & 1];
#pragma unroll
            for (int c = 0; c < NG; c++) {
                if (c >= ng) break;
                const int col = c0 + c;
                const float L = (xs[0][col] + xs[1][col]) + (xs[2][col] + xs[3][col]);
                if (old_slot < 0) {
                    const size_t orow = (size_t)old_s * p.rows + p.row0 + (col >> 1);
                    // no position at all: zero
                    p.out[orow * p.ldo + (2 * old_kvh + (col & 1)) * KV8_HD + row] =
                        f32_to_bf16_rne(L == 0.f ? 0.f : o[c] * (1.f / L));
                } else {
                    float *part = p.part + part_base(gridDim.x) + (size_t)old_slot * (2 * p.L) * (KV8_HD + 2);
                    part[col * KV8_HD + row] = o[c];
                    if (row == 0) {
                        part[2 * p.L * KV8_HD + 2 * col] = m[c];
                        part[2 * p.L * KV8_HD + 2 * col + 1] = L;
                    }
                }
            }
            reset();
            return true;
        };
        for (int r = 0;; r++) {
            const int st = r % ST;
            if (dead || (dead = !warp_wait(&full[st], (r / ST) & 1))) {
                meet(true);
                break;
            }
            const Rec w = rec[st];
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
            if (w.flags & R_Q) {
                piece++;
                dead = !warp_wait(&q_ready[piece & 3], (piece >> 2) & 1);
#pragma unroll
                for (int c = 0; c < NG; c++) qf[c] = c < ng ? q_scale[piece & 3][c0 + c] : 0.f;
            }
            const bool tile = w.blk[0] >= 0;
            float x[NG], sum[NG], vmax = 0.f;                      // this tile's maximum and sum
            if (tile && !dead) {
                const int blk = half ? w.blk[1] : w.blk[0], pos = blk * KV8_BLOCK + (row & 63);
                const float kf = half ? w.ks[1] : w.ks[0];
                float s[NG];
                dead = !warp_wait(&s_full[t & 1], (t >> 1) & 1);
                if (!dead) {
                    uint32_t v[(2 * NG + 3) / 4 * 4];
                    tc_fence_after();
                    load_cols<2 * NG>(tS + lane_off + (t & 1) * NS + 2 * c0, v);
                    const int lim = blk < 0 ? -1 : w.ctx - p.L + c0 / 2;   // last position of this group's token j: lim + j
#pragma unroll
                    for (int c = 0; c < NG; c++) {
                        s[c] = -INFINITY;
                        if (c < ng) {
                            const float q = fmaf(__uint_as_float(v[2 * c + 1]), 0.0625f, __uint_as_float(v[2 * c]));
                            // The scales of q and k make one factor: q times its own could pass FP32's
                            // largest number where the score does not. (A factor that does is taken as
                            // that number: a sum of 0 stays 0.)
                            const float f = qf[c] * kf;
                            if (blk >= 0 && pos <= lim + c / 2) s[c] = q * ((f > FLT_MAX ? FLT_MAX : f) * kKv8ScaleLog2);
                        }
                        x[c] = warp_max(s[c]);
                    }
                    if (lane == 0) put_row<NG>(&xmax[bars & 1][qw][c0], x);
                }
                const float (*xm)[NC] = xmax[bars & 1];            // [warp][column]
                if (meet(dead)) break;
                vmax = w.blk[1] < 0 ? w.vs[0] : fmaxf(w.vs[0], w.vs[1]);
                uint8_t *dst = sP + (t & 1) * NP * 128 + grp * 2048;     // (P.V of tile t - 2 was collected)
                const float ratio = blk < 0 || vmax == 0.f ? 0.f : 256.f * ((half ? w.vs[1] : w.vs[0]) / vmax);
                float xw[4][NG];
#pragma unroll
                for (int k = 0; k < 4; k++) get_row<NG>(&xm[k][c0], xw[k]);
                uint32_t part[8] = {};                             // columns in pairs of two heads, 16 bits each
#pragma unroll
                for (int c = 0; c < NG; c++) {
                    x[c] = fmaxf(fmaxf(xw[0][c], xw[1][c]), fmaxf(xw[2][c], xw[3][c]));
                    sum[c] = ex2(s[c] - (x[c] == -INFINITY ? 0.f : x[c]));
                }
#pragma unroll
                for (int c = 0; c < NG; c += 2) {
                    uint32_t a = pack_f16x2(sum[c] * ratio, sum[c + 1] * ratio);
#pragma unroll
                    for (int k = 0; k < 3; k++) {
                        part[3 * (c / 2) + k] = f16x2_to_e4m3x2(a);
                        // what is left, times 16 (both steps exact)
                        if (k < 2) a = hfma2(e4m3x2_to_f16x2(part[3 * (c / 2) + k]), 0xCC00CC00u, hmul2(a, 0x4C004C00u));
                    }
                }
                *(uint4 *)(dst + row * 16) = make_uint4(part[0] | part[1] << 16, part[2] | part[3] << 16,
                                                        part[4] | part[5] << 16, part[6] | part[7] << 16);
                // codes of V behind the context may be anything, NaN too: a weight of 0 needs a 0
                if (grp == 0 && blk >= 0 && pos >= w.ctx) {
                    uint4 *z = (uint4 *)(ring + st * STAGE + 2 * BLK + row * 128);
#pragma unroll
                    for (int k = 0; k < 8; k++) z[k] = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t & 1]);
            }
            // Meanwhile the tile before this one: its O, and the output if its piece is over. A
            // piece ends with a record that says so; the next record collects its last tile.
            if (owed) collect();
            if (ending) {
                if (!finish()) break;
            }
            if (tile) {
                t++;
                owed = true;
                tv = vmax * 0.00390625f;
#pragma unroll
                for (int c = 0; c < NG; c++) { tm[c] = x[c]; tl[c] = sum[c]; }
            }
            if (w.flags & R_LAST) {
                ending = true;
                old_s = w.s; old_kvh = w.kvh; old_slot = w.slot;
            }
            if (w.flags & R_END) {
                if (owed) collect();
                if (ending) finish();
                else meet(dead);
                break;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, tmem_cols<LT>());
    }
}

// Merges the pair that begins in run c = blockIdx.x and ends behind it (at most
// one). A warp takes one column (128 dimensions, 4 per lane); with 2 or 4 columns
// the 8 warps share each column's pieces.
constexpr int CMB_WARPS = 8;
__global__ void __launch_bounds__(CMB_WARPS * 32) kv8_combine_kernel(const Kv8AttnArgs p, int n_runs) {
    __shared__ float red[CMB_WARPS][KV8_HD + 1];
    dep_wait();
    dep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int4 x4 = __ldcg((const int4 *)p.part + blockIdx.x);
    const Cross x = *(const Cross *)&x4;
    const int pieces = x.n;
    if (!cross_ok(x, blockIdx.x, n_runs, p.n_seqs)) return;
    const int n_col = 2 * p.L, wpc = max(1, CMB_WARPS / n_col), sub = warp % wpc;
    const size_t stride = (size_t)n_col * (KV8_HD + 2);
    // piece k: slot 2 (c + k), but the first one's is given
    const float *own = p.part + part_base(n_runs) + 2 * (size_t)blockIdx.x * stride;
    const size_t own_off = (x.slot & 1) * stride;
    for (int col = warp / wpc; col < n_col; col += CMB_WARPS / wpc) {
        const size_t ml = (size_t)n_col * KV8_HD + 2 * col;
        auto state = [&](int k) { return __ldcg((const float2 *)(own + 2 * k * stride + (k ? 0 : own_off) + ml)); };
        // lane i holds piece i's (max, sum); pieces beyond 32 are read again below
        const float2 mine = lane < pieces ? state(lane) : make_float2(-INFINITY, 0.f);
        float M = mine.x;
        for (int k = lane + 32; k < pieces; k += 32) M = fmaxf(M, state(k).x);
        M = warp_max(M);
        float L = 0.f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < pieces; k0 += 32) {
            const float2 v = k0 == 0 ? mine : k0 + lane < pieces ? state(k0 + lane) : make_float2(-INFINITY, 0.f);
            const float f = v.x == M ? 1.f : ex2(v.x - M);
            if (lane % wpc == sub) L += v.y * f;
            const int n = min(32, pieces - k0);
#pragma unroll 8
            for (int i = sub; i < n; i += wpc) {
                const float w = __shfl_sync(0xFFFFFFFFu, f, i);
                const float4 o = __ldcg((const float4 *)(own + 2 * (k0 + i) * stride + (k0 + i ? 0 : own_off) + col * KV8_HD) + lane);
                O.x += o.x * w; O.y += o.y * w; O.z += o.z * w; O.w += o.w * w;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xFFFFFFFFu, L, o);
        if (wpc > 1) {                                         // one round: every warp comes here once
            float *d = red[warp] + 4 * lane;
            d[0] = O.x; d[1] = O.y; d[2] = O.z; d[3] = O.w;
            if (lane == 0) red[warp][KV8_HD] = L;
            __syncthreads();
            if (sub) continue;
            for (int w = 1; w < wpc; w++) {
                const float *q = red[warp + w] + 4 * lane;
                O.x += q[0]; O.y += q[1]; O.z += q[2]; O.w += q[3];
                L += red[warp + w][KV8_HD];
            }
        }
        const size_t row = (size_t)x.s * p.rows + p.row0 + (col >> 1);
        const float inv = L == 0.f ? 0.f : 1.f / L;
        uint2 *dst = (uint2 *)(p.out + row * p.ldo + (2 * x.kvh + (col & 1)) * KV8_HD) + lane;
        *dst = make_uint2(pack_bf16x2(O.x * inv, O.y * inv), pack_bf16x2(O.z * inv, O.w * inv));
    }
}

constexpr int kSms = 148;
template <int LT>
int ctas() { return kSms * per_sm<LT>(); }
static_assert(3 * (smem_bytes<1>(1) + 2048) <= 233472 && 2 * (smem_bytes<4>(4) + 2560) <= 233472 &&
                  smem_bytes<8>(8) + 3 * 1024 <= 233472,
              "shared memory of an SM: 228 KB, 1 KB a CTA reserved, the rest of the sum static");
static_assert(3 * tmem_cols<1>() <= 512 && 2 * tmem_cols<4>() <= 512 && tmem_cols<8>() <= 512, "TMEM of an SM");
int max_ctas(int L) { return L == 1 ? ctas<1>() : L <= 4 ? ctas<4>() : ctas<8>(); }

template <int LT>
int launch(cudaStream_t st, const CUtensorMap &tk, const CUtensorMap &tv, const Kv8AttnArgs &a) {
    static bool attr[64];
    int dev = 0;
    N550_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && !attr[dev]) {
        N550_CUDA_TRY(cudaFuncSetAttribute(kv8_attn_kernel<LT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           smem_bytes<LT>(LT)));
        attr[dev] = true;
    }
    const size_t smem = smem_bytes<LT>(a.L);
    Lay lay{};
    const long long pairs = (long long)a.n_seqs * KV8_NKV;
    if (!a.part) {
        lay.kind = LAY_PAIR;
        N550_CUDA_TRY(launch_k(kv8_attn_kernel<LT>, dim3((unsigned)pairs), threads<LT>(), smem, st, tk, tv, a, lay));
        N550_LAUNCH_CHECK();
        return N550_OK;
    }
    if (a.n_select >= 0) {
        lay.kind = LAY_EVEN;
        lay.upp = a.n_select > 0 ? a.n_select : 1;
    } else if (!a.pos) {
        lay.kind = LAY_EVEN;
        lay.upp = (a.pos0 + a.L + KV8_BLOCK - 1) / KV8_BLOCK;
    }
    // no more runs than there can be (the kernels cut by the units there are)
    const long long most = (pairs * (lay.kind == LAY_EVEN ? lay.upp : a.c.nb) + kMinRun - 1) / kMinRun;
    const int n = (int)(most < ctas<LT>() ? most : ctas<LT>());
    N550_CUDA_TRY(launch_k(kv8_attn_kernel<LT>, dim3(n), threads<LT>(), smem, st, tk, tv, a, lay));
    N550_LAUNCH_CHECK();
    if (n > 1) {
        N550_CUDA_TRY(launch_k(kv8_combine_kernel, dim3(n - 1), CMB_WARPS * 32, 0, st, a, n));
        N550_LAUNCH_CHECK();
    }
    return N550_OK;
}

}  // namespace

// For calls of up to L queries: the instances differ in their number of runs, so the
// largest need of all of them.
size_t kv8_attn_workspace(int n_seqs, int L) {
    if (n_seqs <= 0 || L <= 0) return 0;
    size_t most = 0;
    for (int l = 1; l <= L; l++) {
        const size_t n = max_ctas(l), need = n * sizeof(Cross) + n * 2 * (2 * l) * (KV8_HD + 2) * sizeof(float);
        most = need > most ? need : most;
    }
    return most;
}

int launch_kv8_merge(cudaStream_t st, const Kv8AttnArgs &a) {
    const int n = max_ctas(a.L);
    N550_CUDA_TRY(launch_k(kv8_combine_kernel, dim3(n - 1), CMB_WARPS * 32, 0, st, a, n));
    N550_LAUNCH_CHECK();
    return N550_OK;
}

int launch_kv8_attn(cudaStream_t st, const Kv8AttnArgs &a) {
    CUtensorMap tk, tv;
    // a row of 128 codes as 64 16-bit columns: one 128-byte swizzle row
    const uint64_t planes = (uint64_t)a.c.n_slots * a.c.n_layers * KV8_NKV;
    int rc = tmap_bf16_sw128_3d(&tk, a.c.k, a.c.max_len, 64, 64, KV8_BLOCK, planes, (uint64_t)a.c.max_len * 64);
    if (!rc) rc = tmap_bf16_sw128_3d(&tv, a.c.v, a.c.max_len, 64, 64, KV8_BLOCK, planes, (uint64_t)a.c.max_len * 64);
    if (rc) return rc;
    return a.L == 1 ? launch<1>(st, tk, tv, a) : a.L <= 4 ? launch<4>(st, tk, tv, a) : launch<8>(st, tk, tv, a);
}

}  // namespace n550
