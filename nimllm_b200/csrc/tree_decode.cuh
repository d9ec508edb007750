// tree_decode.cuh -- what the kernels of tree and scored decode share.
#pragma once
#include "cache_rows.cuh"

namespace nimllm {

// One query row is (token i, query head g of its KV head), numbered i * G + g inside the (sequence, KV head); a token of
// sequence b attends rows 0 .. len-1 and, by its mask, the draft rows len .. len + drafts - 1.  Decode that keeps score
// is the same with one token and no draft rows.
struct TreeParams {
    const void *q;
    const void *k, *v;
    CacheRows rows;
    const int32_t *seq_len, *n_new;
    const uint64_t *mask;        // [B, n, words]; null: draft j sees drafts 0 .. j
    void *out;
    float *partials_out;
    int q_dtype, out_dtype;
    int max_len, drafts;         // drafts: 0 for a scored decode
    int B, n, Hq, Hkv, G, words;
    float scale_log2e;
    // scored decode
    float *score;                // [B][Hkv][score_rows]
    int64_t score_rows;
    float decay;
    // workspace
    float *recs;                 // pieces of split rows: {o[D], m, l, 0, 0}
    float *raw;                  // scored: scaled scores in log2 units, [B][Hq][raw_ld]
    float *stats;                // scored: {m in log2 units, l} per [B][Hq], l = -1: the row was cut
    int64_t raw_ld;
    int chunk_rows, max_chunks;
};

__device__ __forceinline__ int tree_committed(const TreeParams &p, int b) {
    const int hi = min(p.max_len, p.rows.cap);
    return clamp_len(p.seq_len ? p.seq_len[b] : p.max_len, hi);
}
// draft rows of the sequence in the cache
__device__ __forceinline__ int tree_drafts(const TreeParams &p, int b, int len) {
    const int live = p.n_new ? clamp_len(p.n_new[b], p.n) : p.n;
    return min(min(live, p.drafts), p.rows.cap - len);
}
// tokens that have a result
__device__ __forceinline__ int tree_tokens(const TreeParams &p, int b) { return p.n_new ? clamp_len(p.n_new[b], p.n) : p.n; }
__device__ __forceinline__ bool tree_sees(const TreeParams &p, int b, int i, int j) {
    if (!p.mask) return j <= i;
    return (p.mask[((int64_t)b * p.n + i) * p.words + (j >> 6)] >> (j & 63)) & 1;
}
// row of out / partials_out of query row qr of (b, kvh)
__device__ __forceinline__ int64_t tree_out_row(const TreeParams &p, int b, int kvh, int qr) {
    const int i = qr / p.G;
    return ((int64_t)b * p.n + i) * p.Hq + kvh * p.G + (qr - i * p.G);
}

// 1 / l for the sum l of a softmax, 0 for a row that attends nothing.  NaN stays NaN, and an infinite sum times the 0 that it gives.
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.f ? 1.f / l : l; }

// the kernels for bf16 caches (tree_wide_tc.cu, tree_narrow_tc.cu) and for fp32 caches (tree_f32.cu)
size_t tree_tc_workspace_bytes(int batch, int n, int n_head, int n_kv_head, int head_dim);
size_t tree_f32_workspace_bytes(int batch, int n, int n_head, int n_kv_head, int head_dim, int max_total);
int launch_tree_f32(const char *who, TreeParams &p, int head_dim, int max_total, void *workspace, cudaStream_t st);
int launch_tree_tc(const char *who, TreeParams &p, int head_dim, void *workspace, cudaStream_t st);

}  // namespace nimllm
