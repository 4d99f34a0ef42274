// Attention of many queries per sequence over the 8-bit KV cache: the context's
// codes are written out once as BF16 (e4m3 times a power of two: exactly, for scales from
// 2^-124 to 2^119) in the plane order of the BF16 cache, packed for these sequences, and the
// tcgen05 prefill kernel runs over that.
//
// Bound: the tensor cores, from about 64 queries on. Writing out costs 768 bytes
// of traffic per position and KV head (256 read, 512 written) against 1024 flop
// per query of the attention; turning codes into BF16 inside the attention
// kernel instead would repeat it for every 128 queries.
#include "attention.h"
#include "kv8.h"
#include "launch.h"

namespace n550 {
namespace {

constexpr int WO_THREADS = 256;

// One CTA per (block, KV head, sequence): 64 positions of K and V, 8 codes per
// thread and step, so that a warp's store is 512 bytes in one piece (16 codes a
// step leave each 32-byte sector to two stores). A slot outside the cache gives
// zeros, so zero rows.
constexpr int WO_STEPS = KV8_BLOCK * KV8_HD / 8 / WO_THREADS;

__global__ void __launch_bounds__(WO_THREADS)
kv8_write_out_kernel(const Kv8View c, const int32_t *seq_ids, int len, uint16_t *kd, uint16_t *vd) {
    dep_wait();
    dep_launch();
    const int b = blockIdx.x, kvh = blockIdx.y, s = blockIdx.z;
    const int slot = seq_ids[s];
    const bool ok = slot >= 0 && slot < c.n_slots;
    const size_t plane = ok ? c.plane(slot, kvh) : 0;
    const size_t src = (plane * c.max_len + (size_t)b * KV8_BLOCK) * KV8_HD;
    const size_t dst = (((size_t)s * KV8_NKV + kvh) * len + (size_t)b * KV8_BLOCK) * KV8_HD;
    const int n = min(KV8_BLOCK, len - b * KV8_BLOCK) * (KV8_HD / 8);
    const float ks = ok ? c.ks[plane * c.nb + b] : 0.f, vs = ok ? c.vs[plane * c.nb + b] : 0.f;
    uint2 in[2][WO_STEPS];
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int k = 0; k < WO_STEPS; k++) {
            const int i = threadIdx.x + k * WO_THREADS;
            in[w][k] = ok && i < n ? __ldcs((const uint2 *)((w ? c.v : c.k) + src) + i) : make_uint2(0u, 0u);
        }
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int k = 0; k < WO_STEPS; k++) {
            const int i = threadIdx.x + k * WO_THREADS;
            if (i >= n) continue;
            const uint32_t x[2] = {in[w][k].x, in[w][k].y};
            const float sc = w ? vs : ks;
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float2 a = e4m3x2_to_f32x2(x[j] & 0xFFFFu), d = e4m3x2_to_f32x2(x[j] >> 16);
                // exact products: their BF16 form is their upper half (a scale below 2^-124 may
                // leave bits under 2^-133, which are cut off)
                o[2 * j] = __byte_perm(__float_as_uint(a.x * sc), __float_as_uint(a.y * sc), 0x7632);
                o[2 * j + 1] = __byte_perm(__float_as_uint(d.x * sc), __float_as_uint(d.y * sc), 0x7632);
            }
            ((uint4 *)((w ? vd : kd) + dst))[i] = make_uint4(o[0], o[1], o[2], o[3]);
        }
}

}  // namespace

namespace {

// Times in us, from B200 measurements. A pass of up to 8 queries streams the codes at
// 2.2 TB/s after 15 us; without a workspace a CTA of its own takes 1.7 us for each 128
// positions of a pair, 148 of them at a time. Writing out moves 768 bytes per position
// and head at 5 TB/s, and then a CTA takes 2 us for each 128 positions of 128 queries of
// a KV head, the longest context of a wave of 148 of them deciding. Measured
// (passes / whole, sequences x queries over positions): 8 x 5 over 2005 27 / 53, 8 x 16
// over 2016 60 / 54, 64 x 8 over 508 51 / 82, 2 x 8 over 30008 67 / 550 (16 CTAs);
// (passes without a workspace / whole in groups of 1, 2, 4 sequences): 16 x 64 over 8256
// 900 / 2402, 1264, 706; 8 x 512 over 33280 26307 / 4640, 2461, 1390.
double passes_us(int n_seqs, int L, int pos0, bool split) {
    const double len = (double)pos0 + L, passes = (L + KV8_FEW - 1) / KV8_FEW;
    if (split) return passes * (15.0 + n_seqs * len * KV8_NKV * 256 / 2.2e6);
    return passes * (4.0 + (n_seqs * KV8_NKV + 147) / 148 * (len / 128) * 1.7);
}
double whole_us(int n_seqs, int L, int pos0, int group) {
    const double len = (double)pos0 + L;
    const long long items = (long long)group * KV8_NKV * ((L + 127) / 128);
    return (n_seqs + group - 1) / group *
           (4.0 + group * len * KV8_NKV * 768 / 5e6 + (double)((items + 147) / 148) * (len / 128) * 2.0);
}

}  // namespace

bool kv8_in_passes(int n_seqs, int L, int pos0) {
    return L <= KV8_FEW || passes_us(n_seqs, L, pos0, true) < whole_us(n_seqs, L, pos0, n_seqs);
}

int kv8_prefill_group(int n_seqs, int L, int pos0, size_t ws_bytes) {
    if (L <= KV8_FEW) return 0;
    const size_t fit = ws_bytes / kv8_prefill_workspace(1, L, pos0);
    if (fit >= (size_t)n_seqs) return kv8_in_passes(n_seqs, L, pos0) ? 0 : n_seqs;
    if (!fit) return 0;
    const int groups = (int)(((size_t)n_seqs + fit - 1) / fit), group = (n_seqs + groups - 1) / groups;   // of even sizes
    const bool split = ws_bytes >= kv8_attn_workspace(n_seqs, KV8_FEW);
    return passes_us(n_seqs, L, pos0, split) < whole_us(n_seqs, L, pos0, group) ? 0 : group;
}

int launch_kv8_passes(cudaStream_t st, const Kv8AttnArgs &a) {
    Kv8AttnArgs p = a;
    for (int j = 0; j < a.L; j += KV8_FEW) {
        p.row0 = j;
        p.pos0 = a.pos0 + j;
        p.L = a.L - j < KV8_FEW ? a.L - j : KV8_FEW;
        if (int rc = launch_kv8_attn(st, p)) return rc;
    }
    return N550_OK;
}

size_t kv8_prefill_workspace(int n_seqs, int L, int pos0) {
    return 2 * sizeof(uint16_t) * (size_t)n_seqs * KV8_NKV * ((size_t)pos0 + L) * KV8_HD;
}

namespace {

// n_seqs sequences from `s0` on, whose contexts fit `ws`.
int launch_group(cudaStream_t st, const Kv8AttnArgs &a, int s0, int n_seqs, void *ws) {
    const int len = a.pos0 + a.L;
    const int32_t *seq_ids = a.seq_ids + s0;
    const size_t row = (size_t)s0 * a.L;
    uint16_t *kd = (uint16_t *)ws, *vd = kd + (size_t)n_seqs * KV8_NKV * len * KV8_HD;
    const dim3 grid((len + KV8_BLOCK - 1) / KV8_BLOCK, KV8_NKV, n_seqs);
    N550_CUDA_TRY(launch_k(kv8_write_out_kernel, grid, WO_THREADS, 0, st, a.c, seq_ids, len, kd, vd));
    N550_LAUNCH_CHECK();
    AttnPrefillArgs p{};
    p.q = a.q + row * a.ldq; p.kc = kd; p.vc = vd; p.out = a.out + row * a.ldo;
    p.ldq = a.ldq; p.ldo = a.ldo; p.L = a.L; p.pos0 = a.pos0;
    p.max_len = len;
    p.kv_planes = n_seqs * KV8_NKV;
    p.packed = true;
    return launch_attn_prefill(st, p, n_seqs);
}

}  // namespace

int launch_kv8_prefill(cudaStream_t st, const Kv8AttnArgs &a, void *ws, int group) {
    for (int s0 = 0; s0 < a.n_seqs; s0 += group)
        if (int rc = launch_group(st, a, s0, a.n_seqs - s0 < group ? a.n_seqs - s0 : group, ws)) return rc;
    return N550_OK;
}

}  // namespace n550
