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
// In a CTA one warp reads block lists and scales and streams K and V blocks (8
// KB each) through a ring of TMA loads, and four warps take 16 positions of every
// block each. Codes become FP16 in registers, exactly (e4m3 is a subset), on
// their way from shared memory into mma.sync fragments with the positions (for
// q . k) and the dimensions (for P . v) as the 16-row side and the query columns
// as the 8-column side: 2 heads x 4 tokens fill a tile that a decode leaves 3/4
// empty, at a tenth of the tensor rate either way. The 128-byte swizzle and the
// row permutation tok_of() let every shared-memory access read 8 different
// 16-byte columns per phase.
#include <cuda.h>

#include "kv8.h"
#include "launch.h"
#include "tmap.h"

namespace n550 {
namespace {

constexpr int CW = 4;                           // consumer warps
constexpr int THREADS = (CW + 1) * 32;
constexpr int TILE = KV8_BLOCK * KV8_HD;        // 8 KB of K or V codes
constexpr float kLazy = 8.0f;                   // a maximum may be 8 (a factor 256) stale

// What the producer says about a ring stage: one block of one pair.
struct Rec {
    int s, kvh, blk, ctx;                       // blk < 0: nothing to read
    float ks, vs;
    int flags, slot;                            // partial slot, or -1: the whole pair
};
enum { R_FIRST = 1, R_LAST = 2, R_END = 4 };

// How the blocks are laid out along the run axis.
enum { LAY_RAGGED = 0, LAY_EVEN = 1, LAY_PAIR = 2 };
struct Lay {
    int kind;
    int upp;                                    // LAY_EVEN: units per pair
};

template <int NT> constexpr int stages() { return NT == 1 ? 4 : 3; }

__device__ __forceinline__ int tok_of(int g) { return (g & 1) ? (g & 6) ^ 5 : g; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Transposes an 8 x 8 matrix of 16-bit values held one row per four lanes.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// D (16 x 8, FP32) += A (16 x 16 FP16) . B (16 x 8 FP16)
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

// Units (blocks; one empty unit for an empty context) of a pair of sequence s.
__device__ __forceinline__ int seq_ctx(const Kv8AttnArgs &p, int s) {
    const int slot = __ldcg(p.seq_ids + s);
    if (!p.pos) return kv8_ctx(p.c, slot, p.pos0 + p.L - 1);
    return kv8_ctx(p.c, slot, __ldcg(p.pos + s));
}
__device__ __forceinline__ int ctx_blocks(int ctx) { return max(1, (ctx + KV8_BLOCK - 1) / KV8_BLOCK); }

// Cursor into the run axis: sequence s, unit x of its 8 pairs, upp units per pair.
struct Cur {
    int s, upp, ctx;
    long long x;
};

// All threads of the CTA. Returns the total number of units and places *cur at
// unit first(total): LAY_RAGGED needs the prefix sums of the sequences' block
// counts, which every CTA forms itself (n_seqs loads, two barriers).
template <class First>
__device__ __forceinline__ long long locate(const Kv8AttnArgs &p, const Lay lay, First first, Cur *cur) {
    if (lay.kind == LAY_EVEN) {
        const long long total = (long long)lay.upp * KV8_NKV * p.n_seqs, u = first(total);
        if (u >= total) return total;
        cur->s = (int)(u / ((long long)lay.upp * KV8_NKV));
        cur->x = u - (long long)cur->s * lay.upp * KV8_NKV;
        cur->upp = lay.upp;
        return total;
    }
    __shared__ long long wsum[32];
    __shared__ int found_s;
    __shared__ long long found_x;
    const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (p.n_seqs + nt - 1) / nt, s0 = min(tid * per, p.n_seqs), s1 = min(s0 + per, p.n_seqs);
    long long mine = 0;
    for (int s = s0; s < s1; s++) mine += (long long)ctx_blocks(seq_ctx(p, s)) * KV8_NKV;
    long long pre = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xFFFFFFFFu, pre, o);
        if (lane >= o) pre += t;
    }
    if (lane == 31) wsum[warp] = pre;
    __syncthreads();
    long long base = 0, total = 0;
    for (int w = 0; w < nt / 32; w++) {
        if (w < warp) base += wsum[w];
        total += wsum[w];
    }
    const long long u = first(total);
    pre += base - mine;                          // units before this thread's sequences
    if (u >= pre && u < pre + mine) {
        int s = s0;
        long long x = u - pre;
        for (;; s++) {
            const long long n = (long long)ctx_blocks(seq_ctx(p, s)) * KV8_NKV;
            if (x < n) break;
            x -= n;
        }
        found_s = s;
        found_x = x;
    }
    __syncthreads();
    if (u < total) {
        cur->s = found_s;
        cur->x = found_x;
        cur->ctx = seq_ctx(p, found_s);
        cur->upp = ctx_blocks(cur->ctx);
    }
    return total;
}

// `total` units cut into n runs that differ by at most one unit: as many runs as
// CTAs, but none shorter than kMinRun units (a run's blocks are in flight
// together, and each piece costs the merge a partial).
constexpr int kMinRun = 2;
struct Cut {
    long long q;
    int n, r;                                   // run c: q units, the first r runs one more
    __device__ __forceinline__ Cut(long long total, int n_max) {
        const long long most = (total + kMinRun - 1) / kMinRun;
        n = most < n_max ? (int)most : n_max;
        q = total / n;
        r = (int)(total - q * n);
    }
    __device__ __forceinline__ long long start(int c) const { return q * c + min(c, r); }
    __device__ __forceinline__ int run_of(long long u) const {
        const long long big = (q + 1) * r;
        return (int)(u < big ? u / (q + 1) : r + (u - big) / q);
    }
};

// NT column tiles of 8: column 8 i + c is query token (8 i + c) / 2 and head
// 2 kvh + (c & 1).
template <int NT>
__global__ void __launch_bounds__(THREADS)
kv8_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const Kv8AttnArgs p, const Lay lay) {
    constexpr int ST = stages<NT>();
    extern __shared__ uint8_t dsm[];
    uint8_t *ring = (uint8_t *)(((uintptr_t)dsm + 1023) & ~(uintptr_t)1023);     // [ST][K | V]
    const int q_stride = p.L * 512;                                               // 2 heads x 128 BF16 per token
    uint8_t *sq = ring + ST * 2 * TILE;                                           // [ST][L][256]
    float *wo = (float *)(sq + ST * q_stride);                                    // [CW][2 L][128]
    __shared__ __align__(16) Rec rec[ST];
    __shared__ __align__(8) uint64_t full[ST], empty[ST], merge[2];
    __shared__ float wm[CW][8 * NT], wl[CW][8 * NT], wscale[CW];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) { mbar_init(&full[i], 1); mbar_init(&empty[i], CW); }
        mbar_init(&merge[0], CW);
        mbar_init(&merge[1], CW);
        fence_mbar_init();
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    // block lists, positions, scales, codes and queries all come from earlier kernels
    dep_wait();
    dep_launch();
    Cur cur{};
    int n_units;
    if (lay.kind == LAY_PAIR) {
        cur.s = blockIdx.x / KV8_NKV;
        cur.ctx = seq_ctx(p, cur.s);
        cur.upp = p.n_select >= 0 ? max(1, p.n_select) : ctx_blocks(cur.ctx);
        cur.x = (long long)(blockIdx.x % KV8_NKV) * cur.upp;
        n_units = cur.upp;
        __syncthreads();
    } else {
        long long u0 = 0, u1 = 0;
        locate(p, lay, [&](long long total) {
            const Cut cut(total, gridDim.x);
            u0 = u1 = total;
            if ((int)blockIdx.x < cut.n) {
                u0 = cut.start(blockIdx.x);
                u1 = cut.start(blockIdx.x + 1);
            }
            return u0;
        }, &cur);
        n_units = (int)(u1 - u0);
        if (lay.kind == LAY_EVEN) __syncthreads();
    }
    if (n_units == 0) return;

    if (warp == CW) {
        // ---------------- producer: lane i takes unit 32 k + i ----------------
        int r = 0;                                                 // records issued
        bool ok = true;
        for (int base = 0; base < n_units && ok; base += 32) {
            const int i = base + lane;
            Rec me{};
            bool send = false;
            // walk to this lane's unit: whole sequences first
            Cur c = cur;
            if (base + 31 < n_units || i < n_units) {
                c.x += lane;
                while (c.x >= (long long)c.upp * KV8_NKV && c.s + 1 < p.n_seqs) {
                    c.x -= (long long)c.upp * KV8_NKV;
                    c.s++;
                    if (lay.kind == LAY_RAGGED) {
                        c.ctx = seq_ctx(p, c.s);
                        c.upp = ctx_blocks(c.ctx);
                    }
                }
            }
            if (i < n_units) {
                if (lay.kind == LAY_EVEN) c.ctx = seq_ctx(p, c.s);
                const int kvh = (int)(c.x / c.upp), j = (int)(c.x % c.upp);
                int b = j;
                if (p.n_select >= 0)
                    b = p.n_select > 0 ? __ldcg(p.blocks + ((size_t)c.s * KV8_NKV + kvh) * p.n_select + j) : -1;
                if (b < 0 || b > (c.ctx - 1) >> 6) b = -1;      // ctx 0: -1 >> 6 = -1
                me.s = c.s; me.kvh = kvh; me.blk = b; me.ctx = c.ctx;
                me.flags = (i == 0 || j == 0 ? R_FIRST : 0) | (i == n_units - 1 || j == c.upp - 1 ? R_LAST : 0) |
                           (i == n_units - 1 ? R_END : 0);
                // a piece [first unit here .. last unit here] that is not the whole pair
                // is a partial; the one that begins this CTA's run takes slot 2 c
                const bool head = i - j < 0;                     // the pair begins before this run
                const bool tail = i - j + c.upp > n_units;       // and here ends behind it
                me.slot = head || tail ? 2 * (int)blockIdx.x + (i - j > 0) : -1;
                if (b >= 0) {
                    const size_t o = p.c.plane(__ldcg(p.seq_ids + c.s), kvh) * p.c.nb + b;
                    me.ks = __ldcg(p.c.ks + o);
                    me.vs = __ldcg(p.c.vs + o);
                }
                // an unlisted block needs no stage unless its pair begins or ends with it
                send = b >= 0 || (me.flags & (R_FIRST | R_LAST));
            }
            const int n = min(32, n_units - base);
            const uint32_t sends = __ballot_sync(0xFFFFFFFFu, send);
            for (int l = 0; l < n; l++) {
                if (!(sends >> l & 1)) continue;
                const int st = r % ST;
                if (lane == l) {
                    ok = mbar_wait(&empty[st], ((r / ST) & 1) ^ 1);
                    if (ok) {
                        rec[st] = me;
                        const int qn = me.flags & R_FIRST ? p.L : 0;
                        const uint32_t tx = (me.blk >= 0 ? 2 * TILE : 0) + qn * 512;
                        if (tx) mbar_arrive_expect_tx(&full[st], tx);
                        else mbar_arrive(&full[st]);
                        if (me.blk >= 0) {
                            const int plane = (int)p.c.plane(__ldcg(p.seq_ids + me.s), me.kvh);
                            uint8_t *t = ring + st * 2 * TILE;
                            tma_load_3d(t, &tmK, &full[st], 0, me.blk * KV8_BLOCK, plane);
                            tma_load_3d(t + TILE, &tmV, &full[st], 0, me.blk * KV8_BLOCK, plane);
                        }
                        for (int j = 0; j < qn; j++)
                            bulk_load(sq + st * q_stride + j * 512,
                                      p.q + ((size_t)me.s * p.L + j) * p.ldq + me.kvh * 2 * KV8_HD, 512, &full[st]);
                    }
                }
                ok = __shfl_sync(0xFFFFFFFFu, ok, l);
                if (!ok) break;
                r++;
            }
            // the next batch starts behind lane 31's unit
            cur.s = __shfl_sync(0xFFFFFFFFu, c.s, 31);
            cur.upp = __shfl_sync(0xFFFFFFFFu, c.upp, 31);
            cur.ctx = __shfl_sync(0xFFFFFFFFu, c.ctx, 31);
            cur.x = __shfl_sync(0xFFFFFFFFu, c.x, 31) + 1;
        }
        // every load must have landed before the CTA exits: the last ST records
        if (lane == 0)
            for (int i = max(0, r - ST); i < r; i++) mbar_wait(&full[i % ST], (i / ST) & 1);
        __syncwarp();
        return;
    }

    // ---------------- consumers: positions 16 warp .. 16 warp + 15 of every block ----------------
    const int g = lane >> 2, tq = lane & 3, p0 = warp * 16;
    const int n_col = 2 * p.L;
    uint32_t qa[NT][16];                        // q of column g: dims 16 tq + 2 e (+1), then 64 + 16 tq ..
    float qs[NT][2];                            // score factor of columns 2 tq, 2 tq + 1
    float m[NT][2], l[NT][2], o[NT][8][4], vref = 0.f, vinv = INFINITY;
    int jlim[NT][2];                            // last position of the columns' queries
    int merged = 0;
    // addresses of this lane's 16-byte chunks in a tile (row r at 128 r, chunk c at c ^ (r & 7))
    const int kr = p0 + tok_of(g), va = p0 + 2 * tq, vb = p0 + ((2 * tq) ^ 5);
    const uint32_t k_off[2] = {(uint32_t)(kr * 128 + ((tq ^ (kr & 7)) << 4)),
                               (uint32_t)(kr * 128 + (((tq + 4) ^ (kr & 7)) << 4))};
    const uint32_t v_off[2] = {(uint32_t)(va * 128 + ((g ^ (va & 7)) << 4)),
                               (uint32_t)(vb * 128 + ((g ^ (vb & 7)) << 4))};
    for (int r = 0;; r++) {
        const int st = r % ST;
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(&full[st], (r / ST) & 1))) return;
        const Rec w = rec[st];
        if (w.flags & R_FIRST) {
            // queries: FP16 with the column's largest magnitude brought into [1, 2) by
            // a power of two, which BF16 values survive whole (down to 2^-14 of it)
            const uint32_t qb = smem_u32(sq + st * q_stride);
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const int col = 8 * i + g;
                uint32_t x[16];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint4 t = make_uint4(0u, 0u, 0u, 0u);
                    if (col < n_col)
                        t = lds128(qb + col * 256 + (e >> 1) * 128 + tq * 32 + (e & 1) * 16);
                    x[4 * e] = t.x; x[4 * e + 1] = t.y; x[4 * e + 2] = t.z; x[4 * e + 3] = t.w;
                }
                uint32_t am = 0;
#pragma unroll
                for (int e = 0; e < 16; e++) am = max(am, max(x[e] & 0x7FFFu, x[e] >> 16 & 0x7FFFu));
                am = max(am, __shfl_xor_sync(0xFFFFFFFFu, am, 1));
                am = max(am, __shfl_xor_sync(0xFFFFFFFFu, am, 2));
                const int e2 = min(max((int)(am >> 7) - 127, -126), 126);
                const float inv = __uint_as_float((uint32_t)(127 - e2) << 23);
                const float up = __uint_as_float((uint32_t)(127 + e2) << 23);
#pragma unroll
                for (int e = 0; e < 16; e++)
                    qa[i][e] = pack_f16x2(__uint_as_float(x[e] << 16) * inv,
                                          __uint_as_float(x[e] & 0xFFFF0000u) * inv);
                qs[i][0] = __shfl_sync(0xFFFFFFFFu, up, 8 * tq);
                qs[i][1] = __shfl_sync(0xFFFFFFFFu, up, 8 * tq + 4);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    m[i][c] = -INFINITY;
                    l[i][c] = 0.f;
                    // both columns of a lane are heads of one token
                    jlim[i][c] = w.ctx - p.L + 4 * i + tq;
                }
#pragma unroll
                for (int d = 0; d < 8; d++) o[i][d][0] = o[i][d][1] = o[i][d][2] = o[i][d][3] = 0.f;
            }
            vref = 0.f;                            // O is zero: the first block sets the scale
            vinv = INFINITY;
        }
        if (w.blk >= 0) {
            const uint32_t kb = smem_u32(ring + st * 2 * TILE), vbase = kb + TILE;
            const int t0 = w.blk * KV8_BLOCK + p0;                 // this warp's first position
            // S (positions x columns): 16 dims per thread and load, 4 steps each
            float s[NT][4];
#pragma unroll
            for (int i = 0; i < NT; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint4 ra = lds128(kb + k_off[h]), rb = lds128(kb + k_off[h] + 8 * 128);
                const uint32_t a[4] = {ra.x, ra.y, ra.z, ra.w}, b[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t a0 = e4m3x2_to_f16x2(a[e] & 0xFFFFu), a2 = e4m3x2_to_f16x2(a[e] >> 16);
                    const uint32_t a1 = e4m3x2_to_f16x2(b[e] & 0xFFFFu), a3 = e4m3x2_to_f16x2(b[e] >> 16);
#pragma unroll
                    for (int i = 0; i < NT; i++)
                        mma_f16(s[i], a0, a1, a2, a3, qa[i][8 * h + 2 * e], qa[i][8 * h + 2 * e + 1]);
                }
            }
            // online softmax; position of s[.][0], [1]: row g, of [2], [3]: row g + 8
            const int ta = t0 + tok_of(g), tb = ta + 8;
            bool grow = false;
            const float kf = w.ks * kKv8ScaleLog2;
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float f = qs[i][c] * kf;
                    s[i][c] = ta <= jlim[i][c] ? s[i][c] * f : -INFINITY;
                    s[i][2 + c] = tb <= jlim[i][c] ? s[i][2 + c] * f : -INFINITY;
                    grow |= s[i][c] > m[i][c] + kLazy || s[i][2 + c] > m[i][c] + kLazy;
                }
            if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float x = fmaxf(m[i][c], fmaxf(s[i][c], s[i][2 + c]));
                        x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 16));
                        const float corr = m[i][c] == x ? 1.f : ex2(m[i][c] - x);
                        m[i][c] = x;
                        l[i][c] *= corr;
#pragma unroll
                        for (int d = 0; d < 8; d++) { o[i][d][c] *= corr; o[i][d][2 + c] *= corr; }
                    }
            }
            // V's block scale joins the weights as a ratio to the scale O is held in;
            // O moves to the new scale when the ratio leaves [2^-6, 2^6] (FP16 weights
            // reach 2^8 * 2^6)
            float ratio = w.vs * vinv;
            if (!(ratio >= 0.015625f && ratio <= 64.f)) {
                const float move = vref / w.vs;
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int d = 0; d < 8; d++)
#pragma unroll
                        for (int c = 0; c < 4; c++) o[i][d][c] *= move;
                vref = w.vs;
                vinv = 1.f / vref;
                ratio = 1.f;
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int i = 0; i < NT; i++) {
                float e[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float mm = m[i][c & 1] == -INFINITY ? 0.f : m[i][c & 1];
                    e[c] = ex2(s[i][c] - mm);
                    l[i][c & 1] += e[c];
                    e[c] *= ratio;
                }
                // rows g / g + 8 of P become the k pairs of the B fragment of column g
                pb[i][0] = transpose8(pack_f16x2(e[0], e[1]));
                pb[i][1] = transpose8(pack_f16x2(e[2], e[3]));
            }
            // O (dimensions x columns) += V^T P^T: positions va, vb (k = 2 tq, 2 tq + 1) and + 8
            uint4 q4[4];
            q4[0] = lds128(vbase + v_off[0]);
            q4[1] = lds128(vbase + v_off[1]);
            q4[2] = lds128(vbase + v_off[0] + 8 * 128);
            q4[3] = lds128(vbase + v_off[1] + 8 * 128);
            if (t0 + 16 > w.ctx) {
                // codes behind the context may be anything, NaN too: a weight of 0 needs a 0
                const int pv[4] = {va - p0, vb - p0, va - p0 + 8, vb - p0 + 8};
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (t0 + pv[e] >= w.ctx) q4[e] = make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t x0 = e == 0 ? q4[0].x : e == 1 ? q4[0].y : e == 2 ? q4[0].z : q4[0].w;
                const uint32_t x1 = e == 0 ? q4[1].x : e == 1 ? q4[1].y : e == 2 ? q4[1].z : q4[1].w;
                const uint32_t x2 = e == 0 ? q4[2].x : e == 1 ? q4[2].y : e == 2 ? q4[2].z : q4[2].w;
                const uint32_t x3 = e == 0 ? q4[3].x : e == 1 ? q4[3].y : e == 2 ? q4[3].z : q4[3].w;
                const uint32_t lo = __byte_perm(x0, x1, 0x5140), hi = __byte_perm(x0, x1, 0x7362);
                const uint32_t lo8 = __byte_perm(x2, x3, 0x5140), hi8 = __byte_perm(x2, x3, 0x7362);
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const uint32_t u = half ? hi : lo, v = half ? hi8 : lo8;
                    const uint32_t a0 = e4m3x2_to_f16x2(u & 0xFFFFu), a1 = e4m3x2_to_f16x2(u >> 16);
                    const uint32_t a2 = e4m3x2_to_f16x2(v & 0xFFFFu), a3 = e4m3x2_to_f16x2(v >> 16);
#pragma unroll
                    for (int i = 0; i < NT; i++)
                        mma_f16(o[i][2 * e + half], a0, a1, a2, a3, pb[i][0], pb[i][1]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
        if (!(w.flags & R_LAST)) continue;

        // ---------------- the piece ends: merge the four warps ----------------
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[i][c] += __shfl_xor_sync(0xFFFFFFFFu, l[i][c], x);
                const int col = 8 * i + 2 * tq + c;
                if (g == 0) { wm[warp][col] = m[i][c]; wl[warp][col] = l[i][c]; }
                if (col < n_col) {
                    float *d = wo + ((size_t)warp * n_col + col) * KV8_HD + 16 * g;
#pragma unroll
                    for (int x = 0; x < 8; x++)
                        *(float2 *)(d + 2 * x) = make_float2(o[i][x][c], o[i][x][2 + c]);
                }
            }
        if (lane == 0) wscale[warp] = vref;
        __syncwarp();
        if (lane == 0) mbar_arrive(&merge[0]);
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(&merge[0], merged & 1))) return;
        for (int i = threadIdx.x; i < n_col * KV8_HD; i += CW * 32) {
            const int col = i >> 7, d = i & 127;
            float M = -INFINITY;
#pragma unroll
            for (int x = 0; x < CW; x++) M = fmaxf(M, wm[x][col]);
            float L = 0.f, O = 0.f;
#pragma unroll
            for (int x = 0; x < CW; x++) {
                // a warp without positions has m = -inf and l = 0; NaN scores leave m and make l NaN
                const float f = wm[x][col] == M ? 1.f : ex2(wm[x][col] - M);
                L += wl[x][col] * f;
                O += wo[((size_t)x * n_col + col) * KV8_HD + d] * (f * wscale[x]);
            }
            if (w.slot < 0) {
                const size_t row = (size_t)w.s * p.L + (col >> 1);
                // no position at all: zero
                p.out[row * p.ldo + (2 * w.kvh + (col & 1)) * KV8_HD + d] =
                    f32_to_bf16_rne(L == 0.f ? 0.f : O * (1.f / L));
            } else {
                float *part = p.part + (size_t)w.slot * n_col * (KV8_HD + 2);
                part[col * KV8_HD + d] = O;
                if (d == 0) {
                    part[n_col * KV8_HD + 2 * col] = M;
                    part[n_col * KV8_HD + 2 * col + 1] = L;
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&merge[1]);
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(&merge[1], merged & 1))) return;
        merged++;
        if (w.flags & R_END) return;
    }
}

// Merges the pair that begins in run c = blockIdx.x and ends behind it (at most
// one). A warp takes one column (128 dimensions, 4 per lane); with 2 or 4 columns
// the 8 warps share each column's pieces.
constexpr int CMB_WARPS = 8;
__global__ void __launch_bounds__(CMB_WARPS * 32) kv8_combine_kernel(const Kv8AttnArgs p, const Lay lay, int n_max) {
    __shared__ float red[CMB_WARPS][KV8_HD + 1];
    dep_wait();
    dep_launch();
    const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Cur cur{};
    long long u0 = 0, u1 = 0;
    int n = 0;
    long long tot = 0;
    locate(p, lay, [&](long long total) {
        const Cut cut(total, n_max);
        tot = total;
        u0 = u1 = total;
        n = cut.n;
        if (c < cut.n - 1) {
            u0 = cut.start(c);
            u1 = cut.start(c + 1);
        }
        return u1;
    }, &cur);
    if (c >= n - 1) return;
    const int kvh = (int)(cur.x / cur.upp), j = (int)(cur.x % cur.upp);
    const long long first = u1 - j;                            // the pair's first unit
    if (j == 0 || first < u0) return;                          // no pair crosses, or it began earlier
    const int pieces = Cut(tot, n_max).run_of(first + cur.upp - 1) - c + 1;
    const int n_col = 2 * p.L, wpc = max(1, CMB_WARPS / n_col), sub = warp % wpc;
    const size_t stride = (size_t)n_col * (KV8_HD + 2);
    const float *own = p.part + 2 * (size_t)c * stride;        // piece k: slot 2 (c + k), the first 2 c or 2 c + 1
    const size_t own_off = first > u0 ? stride : 0;
    for (int col = warp / wpc; col < n_col; col += CMB_WARPS / wpc) {
        const size_t ml = (size_t)n_col * KV8_HD + 2 * col;
        float M = -INFINITY;
        for (int k = lane; k < pieces; k += 32) M = fmaxf(M, __ldcg(own + 2 * k * stride + (k ? 0 : own_off) + ml));
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, x));
        float L = 0.f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < pieces; k0 += 32 * wpc) {        // lane i of this batch: piece k0 + wpc i + sub
            const int k = k0 + wpc * lane + sub;
            float f = 0.f;
            if (k < pieces) {
                const float2 v = __ldcg((const float2 *)(own + 2 * k * stride + (k ? 0 : own_off) + ml));
                f = v.x == M ? 1.f : ex2(v.x - M);
                L += v.y * f;
            }
            const int take = min(32, (pieces - k0 - sub + wpc - 1) / wpc);
#pragma unroll 8
            for (int i = 0; i < take; i++) {
                const int ki = k0 + wpc * i + sub;
                const float w = __shfl_sync(0xFFFFFFFFu, f, i);
                const float4 v = __ldcg((const float4 *)(own + 2 * ki * stride + (ki ? 0 : own_off) + col * KV8_HD) + lane);
                O.x += v.x * w; O.y += v.y * w; O.z += v.z * w; O.w += v.w * w;
            }
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xFFFFFFFFu, L, x);
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
        const size_t row = (size_t)cur.s * p.L + (col >> 1);
        const float inv = L == 0.f ? 0.f : 1.f / L;
        uint2 *dst = (uint2 *)(p.out + row * p.ldo + (2 * kvh + (col & 1)) * KV8_HD) + lane;
        *dst = make_uint2(pack_bf16x2(O.x * inv, O.y * inv), pack_bf16x2(O.z * inv, O.w * inv));
    }
}

template <int NT>
constexpr int smem_bytes(int L) {
    return stages<NT>() * (2 * TILE + L * 512) + CW * 2 * L * KV8_HD * 4 + 1024;
}

constexpr int kSms = 148;
// CTAs that share an SM: shared memory (227 KB, 1 KB of it taken per CTA and about 1 KB static)
template <int NT>
int ctas(int L) {
    const int per_sm = 232448 / (smem_bytes<NT>(L) + 2560);
    return kSms * (per_sm < 1 ? 1 : per_sm > 3 ? 3 : per_sm);
}
int max_ctas(int L) { return L <= 4 ? ctas<1>(L) : ctas<2>(L); }

template <int NT>
int launch(cudaStream_t st, const CUtensorMap &tk, const CUtensorMap &tv, const Kv8AttnArgs &a) {
    static bool attr[64];
    int dev = 0;
    N550_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && !attr[dev]) {
        N550_CUDA_TRY(cudaFuncSetAttribute(kv8_attn_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           smem_bytes<NT>(4 * NT)));
        attr[dev] = true;
    }
    const size_t smem = smem_bytes<NT>(a.L);
    Lay lay{};
    const long long pairs = (long long)a.n_seqs * KV8_NKV;
    if (!a.part) {
        lay.kind = LAY_PAIR;
        N550_CUDA_TRY(launch_k(kv8_attn_kernel<NT>, dim3((unsigned)pairs), THREADS, smem, st, tk, tv, a, lay));
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
    const int n = (int)(most < ctas<NT>(a.L) ? most : ctas<NT>(a.L));
    N550_CUDA_TRY(launch_k(kv8_attn_kernel<NT>, dim3(n), THREADS, smem, st, tk, tv, a, lay));
    N550_LAUNCH_CHECK();
    if (n > 1) {
        N550_CUDA_TRY(launch_k(kv8_combine_kernel, dim3(n - 1), CMB_WARPS * 32, 0, st, a, lay, n));
        N550_LAUNCH_CHECK();
    }
    return N550_OK;
}

}  // namespace

size_t kv8_attn_workspace(int n_seqs, int L) {
    if (n_seqs <= 0 || L <= 0) return 0;
    return (size_t)max_ctas(L) * 2 * (2 * L) * (KV8_HD + 2) * sizeof(float);
}

int launch_kv8_attn(cudaStream_t st, const Kv8AttnArgs &a) {
    CUtensorMap tk, tv;
    // a row of 128 codes as 64 16-bit columns: one 128-byte swizzle row
    const uint64_t planes = (uint64_t)a.c.n_slots * a.c.n_layers * KV8_NKV;
    int rc = tmap_bf16_sw128_3d(&tk, a.c.k, a.c.max_len, 64, 64, KV8_BLOCK, planes, (uint64_t)a.c.max_len * 64);
    if (!rc) rc = tmap_bf16_sw128_3d(&tv, a.c.v, a.c.max_len, 64, 64, KV8_BLOCK, planes, (uint64_t)a.c.max_len * 64);
    if (rc) return rc;
    return a.L <= 4 ? launch<1>(st, tk, tv, a) : launch<2>(st, tk, tv, a);
}

}  // namespace n550
