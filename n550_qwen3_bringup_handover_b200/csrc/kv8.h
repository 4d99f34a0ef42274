// Internal interface of the 8-bit KV cache kernels (not part of the C ABI).
//
// The cache (n550_kv8_cache) holds, for each (slot, layer, KV head) plane, the
// positions' K and V as e4m3 codes [max_len][128], one FP32 power-of-two scale
// per block of 64 positions for each of K and V, and per block and K channel the
// smallest and the largest code (bounds [n_blocks][2][128]).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace n550 {

constexpr int KV8_HD = 128;
constexpr int KV8_NKV = 8;
constexpr int KV8_NH = 16;
constexpr int KV8_BLOCK = N550_KV8_BLOCK;
constexpr float kKv8ScaleLog2 = 0.08838834764831845f * 1.4426950408889634f;   // qwen3.c:296, log2 domain

struct Kv8View {
    uint8_t *k, *v;
    float *ks, *vs;
    uint8_t *kb;               // NULL: no bounds kept
    int n_slots, n_layers, max_len, nb, layer;
    // plane of (slot, KV head) in this layer
    __host__ __device__ __forceinline__ size_t plane(int slot, int kvh) const {
        return ((size_t)slot * n_layers + layer) * KV8_NKV + kvh;
    }
};

// Checks the cache and the layer and fills the view; N550_OK or N550_ERR_ARG.
int kv8_view(const n550_kv8_cache *c, int layer, Kv8View *v);

// Two e4m3 codes (low byte first) -> FP16 pair; exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f32x2(uint32_t two) {
    const uint32_t h = e4m3x2_to_f16x2(two);
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}
// (lo, hi) -> two e4m3 codes, round to nearest even; beyond +-448 (infinities
// too) the largest finite code, NaN the NaN code.
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Positions 0..pos that a query at `pos` attends to: none for a negative
// position or a slot outside the cache, at most the cache's max_len.
__device__ __forceinline__ int kv8_ctx(const Kv8View &c, int slot, int pos) {
    return slot < 0 || slot >= c.n_slots || pos < 0 ? 0 : min(pos, c.max_len - 1) + 1;
}

// FP16 pair -> two e4m3 codes, as above.
__device__ __forceinline__ uint32_t f16x2_to_e4m3x2(uint32_t h) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(h));
    return r;
}

struct Kv8AppendArgs {
    Kv8View c;
    const void *k, *v;         // rows [n_seqs * L][ld], KV head h at columns 128 h ..
    int ld, L;
    const int32_t *seq_ids;
    const int32_t *pos;        // first position per sequence, or NULL: pos0 for all
    int pos0;
};

struct Kv8AttnArgs {
    Kv8View c;
    const uint16_t *q;         // BF16 rows [n_seqs * L][ldq]
    uint16_t *out;             // BF16 rows [n_seqs * L][ldo]
    const int32_t *seq_ids;
    const int32_t *pos;        // first query position per sequence, or NULL: pos0 for all
    const int32_t *blocks;     // [n_seqs][8][n_select]
    int n_select;              // < 0: no list, the whole context
    int ldq, ldo, L, pos0, n_seqs;
    int rows, row0;            // a sequence's rows in q and out, and the first of these L among them
    float *part;               // split partials, or NULL
};

int launch_kv8_append(cudaStream_t st, const Kv8AppendArgs &a, bool f32, int n_seqs);
constexpr int KV8_FEW = 8;     // most queries per sequence of launch_kv8_attn
// Whether L queries per sequence at positions pos0 .. take the streaming kernel, in
// passes of KV8_FEW, rather than launch_kv8_prefill; and those passes.
bool kv8_in_passes(int n_seqs, int L, int pos0);
int launch_kv8_passes(cudaStream_t st, const Kv8AttnArgs &a);
// Many queries: codes written out as BF16 to `ws`, then the BF16 prefill kernel, in
// groups of `group` sequences (of which ws holds kv8_prefill_workspace bytes).
int launch_kv8_prefill(cudaStream_t st, const Kv8AttnArgs &a, void *ws, int group);
// Sequences per group with a workspace of that many bytes; 0: passes.
int kv8_prefill_group(int n_seqs, int L, int pos0, size_t ws_bytes);
size_t kv8_prefill_workspace(int n_seqs, int L, int pos0);
int launch_kv8_attn(cudaStream_t st, const Kv8AttnArgs &a);
// The merge of launch_kv8_attn alone, of all the runs that a call can have.
int launch_kv8_merge(cudaStream_t st, const Kv8AttnArgs &a);
size_t kv8_attn_workspace(int n_seqs, int L);

struct Kv8SelectArgs {
    Kv8View c;
    const uint16_t *q;
    const int32_t *seq_ids, *pos;
    int32_t *blocks;           // [n_seqs][8][n_select]
    int ldq, n_seqs, n_select, n_sink, n_recent;
};
int launch_kv8_select(cudaStream_t st, const Kv8SelectArgs &a);

}  // namespace n550
