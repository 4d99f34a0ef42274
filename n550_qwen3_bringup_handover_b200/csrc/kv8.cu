// Exported entry points of the 8-bit KV cache (include/n550_qwen3.h): argument
// checks and routing.
#include "kv8.h"

namespace n550 {

int kv8_view(const n550_kv8_cache *c, int layer, Kv8View *v) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || c->n_slots <= 0 || c->n_layers <= 0 ||
        c->max_len <= 0 || c->max_len > 1 << 30 || layer < 0 || layer >= c->n_layers ||
        (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_bounds) & 15) ||
        (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3) ||
        (long long)c->n_slots * c->n_layers * KV8_NKV > (1LL << 31) - 1)
        return N550_ERR_ARG;
    v->k = c->k; v->v = c->v; v->ks = c->k_scale; v->vs = c->v_scale; v->kb = c->k_bounds;
    v->n_slots = c->n_slots; v->n_layers = c->n_layers; v->max_len = c->max_len;
    v->nb = (int)(((long long)c->max_len + KV8_BLOCK - 1) / KV8_BLOCK);
    v->layer = layer;
    return N550_OK;
}

namespace {

// Split partials go to a workspace that is large enough, 16-byte aligned.
float *split_ws(void *ws, size_t bytes, size_t need) {
    return ws && bytes >= need && ((uintptr_t)ws & 15) == 0 ? (float *)ws : nullptr;
}

// gridDim.y and .z end at 65535
constexpr int kMaxSeqs = 65535;

// a pair's list and its eight heads are counted in 32 bits
constexpr int kMaxSelect = 1 << 24;

bool rows_ok(const void *p, int ld, int esz) {
    return p && ((uintptr_t)p & 15) == 0 && ld >= KV8_NH * KV8_HD && (long long)ld * esz % 16 == 0;
}

}  // namespace
}  // namespace n550

using namespace n550;

extern "C" {

int n550_kv8_append(void *stream, const n550_kv8_cache *c, int layer, const void *k, const void *v,
                    int type, int ld, const int32_t *seq_ids, const int32_t *pos, int n_seqs, int L) {
    Kv8AppendArgs a{};
    if (int rc = kv8_view(c, layer, &a.c)) return rc;
    if (n_seqs < 0 || L < 0 || (type != N550_F32 && type != N550_BF16)) return N550_ERR_ARG;
    if (n_seqs == 0 || L == 0) return N550_OK;
    const int esz = type == N550_F32 ? 4 : 2;
    if (!k || !v || !seq_ids || !pos || L > c->max_len || ld < KV8_NKV * KV8_HD || n_seqs > kMaxSeqs ||
        (long long)ld * esz % 16 || (((uintptr_t)k | (uintptr_t)v) & 15))
        return N550_ERR_ARG;
    a.k = k; a.v = v; a.ld = ld; a.L = L; a.seq_ids = seq_ids; a.pos = pos;
    return launch_kv8_append((cudaStream_t)stream, a, type == N550_F32, n_seqs);
}

size_t n550_attention_kv8_workspace(int n_seqs) { return kv8_attn_workspace(n_seqs, 1); }

int n550_attention_decode_kv8(void *stream, const uint16_t *q, int ldq, const n550_kv8_cache *c,
                              int layer, const int32_t *seq_ids, const int32_t *pos, int n_seqs,
                              uint16_t *out, int ldo, void *workspace, size_t workspace_bytes) {
    Kv8AttnArgs a{};
    if (int rc = kv8_view(c, layer, &a.c)) return rc;
    if (n_seqs < 0) return N550_ERR_ARG;
    if (n_seqs == 0) return N550_OK;
    if (!rows_ok(q, ldq, 2) || !rows_ok(out, ldo, 2) || !seq_ids || !pos || n_seqs > kMaxSeqs)
        return N550_ERR_ARG;
    a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo; a.seq_ids = seq_ids; a.pos = pos;
    a.L = a.rows = 1; a.n_seqs = n_seqs; a.n_select = -1;
    a.part = split_ws(workspace, workspace_bytes, kv8_attn_workspace(n_seqs, 1));
    return launch_kv8_attn((cudaStream_t)stream, a);
}

int n550_attention_sparse_kv8(void *stream, const uint16_t *q, int ldq, const n550_kv8_cache *c,
                              int layer, const int32_t *seq_ids, const int32_t *pos,
                              const int32_t *blocks, int n_select, int n_seqs, uint16_t *out, int ldo,
                              void *workspace, size_t workspace_bytes) {
    Kv8AttnArgs a{};
    if (int rc = kv8_view(c, layer, &a.c)) return rc;
    if (n_seqs < 0 || n_select < 0) return N550_ERR_ARG;
    if (n_seqs == 0) return N550_OK;
    if (!rows_ok(q, ldq, 2) || !rows_ok(out, ldo, 2) || !seq_ids || !pos ||
        (!blocks && n_select) || n_select > kMaxSelect || n_seqs > kMaxSeqs)
        return N550_ERR_ARG;
    a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo; a.seq_ids = seq_ids; a.pos = pos;
    a.blocks = blocks; a.n_select = n_select;
    a.L = a.rows = 1; a.n_seqs = n_seqs;
    a.part = split_ws(workspace, workspace_bytes, kv8_attn_workspace(n_seqs, 1));
    return launch_kv8_attn((cudaStream_t)stream, a);
}

int n550_check_kv8_merge(void *stream, int n_seqs, void *workspace, size_t workspace_bytes, uint16_t *out,
                         int ldo) {
    if (n_seqs < 1 || n_seqs > kMaxSeqs || !rows_ok(out, ldo, 2)) return N550_ERR_ARG;
    Kv8AttnArgs a{};
    a.out = out; a.ldo = ldo; a.L = a.rows = 1; a.n_seqs = n_seqs;
    a.part = split_ws(workspace, workspace_bytes, kv8_attn_workspace(n_seqs, 1));
    return a.part ? launch_kv8_merge((cudaStream_t)stream, a) : N550_ERR_ARG;
}

size_t n550_attention_prefill_kv8_workspace(int n_seqs, int L, int pos0) {
    if (n_seqs <= 0 || L <= 0 || pos0 < 0) return 0;
    return kv8_in_passes(n_seqs, L, pos0) ? kv8_attn_workspace(n_seqs, L < KV8_FEW ? L : KV8_FEW)
                                          : kv8_prefill_workspace(n_seqs, L, pos0);
}

int n550_attention_prefill_kv8(void *stream, const uint16_t *q, int ldq, const n550_kv8_cache *c,
                               int layer, const int32_t *seq_ids, int n_seqs, int L, int pos0,
                               uint16_t *out, int ldo, void *workspace, size_t workspace_bytes) {
    Kv8AttnArgs a{};
    if (int rc = kv8_view(c, layer, &a.c)) return rc;
    if (n_seqs < 0 || L < 0 || pos0 < 0) return N550_ERR_ARG;
    if (n_seqs == 0 || L == 0) return N550_OK;
    if (!rows_ok(q, ldq, 2) || !rows_ok(out, ldo, 2) || !seq_ids || n_seqs > kMaxSeqs ||
        (long long)pos0 + L > c->max_len)
        return N550_ERR_ARG;
    a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo; a.seq_ids = seq_ids;
    a.L = L; a.pos0 = pos0; a.n_seqs = n_seqs; a.n_select = -1;
    a.rows = L;
    if (!split_ws(workspace, workspace_bytes, 0)) workspace_bytes = 0;
    if (const int group = kv8_prefill_group(n_seqs, L, pos0, workspace_bytes))
        return launch_kv8_prefill((cudaStream_t)stream, a, workspace, group);
    // (a workspace too small for the splits' partials: passes without splits)
    a.part = split_ws(workspace, workspace_bytes, kv8_attn_workspace(n_seqs, L < KV8_FEW ? L : KV8_FEW));
    return launch_kv8_passes((cudaStream_t)stream, a);
}

int n550_kv8_select_blocks(void *stream, const uint16_t *q, int ldq, const n550_kv8_cache *c, int layer,
                           const int32_t *seq_ids, const int32_t *pos, int n_seqs, int n_select,
                           int n_sink, int n_recent, int32_t *blocks) {
    Kv8SelectArgs a{};
    if (int rc = kv8_view(c, layer, &a.c)) return rc;
    if (!c->k_bounds || n_seqs < 0 || n_select < 1 || n_sink < 0 || n_recent < 0 ||
        (long long)n_sink + n_recent > n_select)
        return N550_ERR_ARG;
    if (a.c.nb > N550_KV8_SELECT_MAX_BLOCKS) return N550_ERR_UNSUPPORTED;
    if (n_seqs == 0) return N550_OK;
    if (!rows_ok(q, ldq, 2) || !seq_ids || !pos || !blocks || n_seqs > kMaxSeqs) return N550_ERR_ARG;
    a.q = q; a.ldq = ldq; a.seq_ids = seq_ids; a.pos = pos; a.blocks = blocks;
    a.n_seqs = n_seqs; a.n_select = n_select; a.n_sink = n_sink; a.n_recent = n_recent;
    return launch_kv8_select((cudaStream_t)stream, a);
}

}  // extern "C"
