// tree_decode.cu -- attention of drafted tokens over a KV cache, and decode that keeps score of the cached rows.
//
//   out[b, i, h] = sum_r w_r v_r,  w = softmax over the rows r that token i attends of  scale q . k_r
//   score[b, kvh, r] = decay * score[b, kvh, r] + sum over the query heads of kvh of w_r          (scored decode)
//
// This file holds the entry points and the choice of the kernel: tree_narrow_tc.cu and tree_wide_tc.cu (bf16 caches), tree_f32.cu (fp32
// caches), each followed by the launch of tree_finish.cuh.  The G query heads of a KV head and the n tokens of a sequence are rows of
// one tile, so that a cached row is read once for all of them.
#include "tree_decode.cuh"

namespace nimllm {

namespace {

constexpr int kScoredMaxGroup = 6144;      // query heads of a KV head: a score block keeps 8 bytes of each in 48 KB of shared memory

size_t round256(size_t x) { return (x + 255) / 256 * 256; }
size_t record_bytes(int batch, int n, int n_head, int n_kv_head, int head_dim, int max_total, int cache_dtype) {
    return round256(cache_dtype == NIMLLM_BF16 ? tree_tc_workspace_bytes(batch, n, n_head, n_kv_head, head_dim)
                                               : tree_f32_workspace_bytes(batch, n, n_head, n_kv_head, head_dim, max_total));
}
// whole tiles of the tensor-core kernels are written
int64_t raw_rows(int max_len) { return ((int64_t)max_len + 127) / 128 * 128; }

// what the launches' grids and 32-bit row numbers hold
bool fits(int batch, int n, int n_head, int n_kv_head, int max_len) {
    return batch <= 65535 && (int64_t)n_kv_head * (((int64_t)n * (n_head / n_kv_head) + 31) / 32) <= 65535 && max_len <= (1 << 30);
}

// q, shapes and the workspace of both entry points
int tree_launch(const char *who, TreeParams &p, const void *workspace, size_t workspace_bytes, size_t need, int cache_dtype, int head_dim,
                cudaStream_t st) {
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(NIMLLM_ERR_WORKSPACE, "%s: workspace %zu bytes, need %zu", who, workspace_bytes, need);
    if (need > 0 && ((uintptr_t)workspace & 255)) return fail(NIMLLM_ERR_ARG, "%s: workspace must be 256-byte aligned", who);
    const int max_total = p.max_len + p.drafts;
    unsigned char *ws = (unsigned char *)workspace;
    p.recs = (float *)ws;
    p.raw = nullptr; p.stats = nullptr; p.raw_ld = 0;
    if (p.score) {
        p.raw_ld = raw_rows(p.max_len);
        p.stats = (float *)(ws + record_bytes(p.B, p.n, p.Hq, p.Hkv, head_dim, max_total, cache_dtype));
        p.raw = (float *)((unsigned char *)p.stats + round256((size_t)p.B * p.Hq * 2 * sizeof(float)));
    }
    return cache_dtype == NIMLLM_BF16 ? launch_tree_tc(who, p, head_dim, ws, st) : launch_tree_f32(who, p, head_dim, max_total, ws, st);
}

int check_shape(const char *who, const void *q, int q_dtype, const void *out, int out_dtype, const float *partials_out, int max_len,
                int batch, int n, int n_head, int n_kv_head, int head_dim) {
    if (!q || (!out && !partials_out)) return fail(NIMLLM_ERR_ARG, "%s: null q / output pointer", who);
    if (batch <= 0 || n <= 0 || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || max_len < 0)
        return fail(NIMLLM_ERR_ARG, "%s: bad shape B=%d n=%d Hq=%d Hkv=%d max_len=%d", who, batch, n, n_head, n_kv_head, max_len);
    if (!dtype_ok(q_dtype) || !dtype_ok(out_dtype)) return fail(NIMLLM_ERR_ARG, "%s: unknown dtype", who);
    if (head_dim != 64 && head_dim != 128) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: head_dim %d (64 and 128 are built)", who, head_dim);
    if (n > kTreeMaxTokens) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: n %d > %d", who, n, kTreeMaxTokens);
    if (!fits(batch, n, n_head, n_kv_head, max_len))
        return fail(NIMLLM_ERR_UNSUPPORTED, "%s: batch %d, n %d, Hq %d or max_len %d is too large", who, batch, n, n_head, max_len);
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)partials_out) & 15) return fail(NIMLLM_ERR_ARG, "%s: q and the outputs must be 16-byte aligned", who);
    return NIMLLM_OK;
}

int decode_tree(const char *who, const CacheRows &rows, const void *q, int q_dtype, const void *k, const void *v, int cache_dtype,
                const int32_t *seq_len, int max_len, const int32_t *n_new, const uint64_t *tree_mask, void *out, int out_dtype,
                float *partials_out, int batch, int n, int n_head, int n_kv_head, int head_dim, float scale, void *workspace,
                size_t workspace_bytes, void *stream) {
    if (int rc = check_shape(who, q, q_dtype, out, out_dtype, partials_out, max_len, batch, n, n_head, n_kv_head, head_dim)) return rc;
    if ((uintptr_t)tree_mask & 7) return fail(NIMLLM_ERR_ARG, "%s: tree_mask must be 8-byte aligned", who);
    TreeParams p = {};
    p.q = q; p.k = k; p.v = v; p.rows = rows; p.seq_len = seq_len; p.n_new = n_new; p.mask = tree_mask;
    p.out = out; p.partials_out = partials_out; p.q_dtype = q_dtype; p.out_dtype = out_dtype; p.max_len = max_len; p.drafts = n;
    p.B = batch; p.n = n; p.Hq = n_head; p.Hkv = n_kv_head; p.G = n_head / n_kv_head; p.words = (n + 63) / 64;
    p.scale_log2e = scale * kLog2e;
    const size_t need = nimllm_attn_decode_tree_workspace_bytes(batch, n, n_head, n_kv_head, head_dim, max_len, cache_dtype);
    return tree_launch(who, p, workspace, workspace_bytes, need, cache_dtype, head_dim, (cudaStream_t)stream);
}

int decode_scored(const char *who, const CacheRows &rows, const void *q, int q_dtype, const void *k, const void *v, int cache_dtype,
                  const int32_t *seq_len, int max_len, void *out, int out_dtype, float *score, int64_t score_rows, float decay,
                  int batch, int n_head, int n_kv_head, int head_dim, float scale, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_shape(who, q, q_dtype, out, out_dtype, nullptr, max_len, batch, 1, n_head, n_kv_head, head_dim)) return rc;
    if (!score) return fail(NIMLLM_ERR_ARG, "%s: null score", who);
    if (max_len <= 0) return fail(NIMLLM_ERR_ARG, "%s: max_len %d", who, max_len);
    if (score_rows < max_len) return fail(NIMLLM_ERR_ARG, "%s: %lld scores per KV head, max_len %d", who, (long long)score_rows, max_len);
    if (n_kv_head > 65535) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: Hkv %d", who, n_kv_head);
    if (n_head / n_kv_head > kScoredMaxGroup)
        return fail(NIMLLM_ERR_UNSUPPORTED, "%s: %d query heads per KV head (at most %d)", who, n_head / n_kv_head, kScoredMaxGroup);
    TreeParams p = {};
    p.q = q; p.k = k; p.v = v; p.rows = rows; p.seq_len = seq_len;
    p.out = out; p.q_dtype = q_dtype; p.out_dtype = out_dtype; p.max_len = max_len; p.drafts = 0;
    p.B = batch; p.n = 1; p.Hq = n_head; p.Hkv = n_kv_head; p.G = n_head / n_kv_head; p.words = 1;
    p.scale_log2e = scale * kLog2e; p.score = score; p.score_rows = score_rows; p.decay = decay;
    const size_t need = nimllm_attn_decode_scored_workspace_bytes(batch, n_head, n_kv_head, head_dim, max_len, cache_dtype);
    return tree_launch(who, p, workspace, workspace_bytes, need, cache_dtype, head_dim, (cudaStream_t)stream);
}

}  // namespace

}  // namespace nimllm

using namespace nimllm;

extern "C" {

size_t nimllm_attn_decode_tree_workspace_bytes(int batch, int n, int n_head, int n_kv_head, int head_dim, int max_len, int cache_dtype) {
    if (batch <= 0 || n <= 0 || n > kTreeMaxTokens || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || head_dim <= 0 || max_len < 0 ||
        !fits(batch, n, n_head, n_kv_head, max_len))
        return 0;                                          // the call refuses the same shapes
    return record_bytes(batch, n, n_head, n_kv_head, head_dim, max_len + n, cache_dtype);
}

int nimllm_attn_decode_tree(const void *q, int q_dtype, const void *k_cache, const void *v_cache, int cache_dtype, const int64_t *kv_off,
                            int64_t seq_stride, int64_t head_stride, int max_seq, const int32_t *seq_len, int max_len,
                            const int32_t *n_new, const uint64_t *tree_mask, void *out, int out_dtype, float *partials_out, int batch,
                            int n, int n_head, int n_kv_head, int head_dim, float scale, void *workspace, size_t workspace_bytes,
                            void *stream) {
    const char *who = "attn_decode_tree";
    CacheRows rows;
    if (int rc = contiguous_rows(rows, who, k_cache, v_cache, cache_dtype, kv_off, seq_stride, head_stride, max_seq, head_dim)) return rc;
    return decode_tree(who, rows, q, q_dtype, k_cache, v_cache, cache_dtype, seq_len, max_len, n_new, tree_mask, out, out_dtype, partials_out,
                       batch, n, n_head, n_kv_head, head_dim, scale, workspace, workspace_bytes, stream);
}

int nimllm_attn_decode_tree_paged(const void *q, int q_dtype, const void *k_pages, const void *v_pages, int cache_dtype,
                                  const int32_t *page_table, int max_pages, int page_rows, int n_pages, const int32_t *seq_len,
                                  int max_len, const int32_t *n_new, const uint64_t *tree_mask, void *out, int out_dtype,
                                  float *partials_out, int batch, int n, int n_head, int n_kv_head, int head_dim, float scale,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "attn_decode_tree_paged";
    CacheRows rows;
    if (int rc = paged_rows(rows, who, k_pages, v_pages, cache_dtype, page_table, max_pages, page_rows, n_pages, n_kv_head, head_dim)) return rc;
    return decode_tree(who, rows, q, q_dtype, k_pages, v_pages, cache_dtype, seq_len, max_len, n_new, tree_mask, out, out_dtype, partials_out,
                       batch, n, n_head, n_kv_head, head_dim, scale, workspace, workspace_bytes, stream);
}

size_t nimllm_attn_decode_scored_workspace_bytes(int batch, int n_head, int n_kv_head, int head_dim, int max_len, int cache_dtype) {
    if (batch <= 0 || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || head_dim <= 0 || max_len <= 0 || !fits(batch, 1, n_head, n_kv_head, max_len))
        return 0;
    return record_bytes(batch, 1, n_head, n_kv_head, head_dim, max_len, cache_dtype) + round256((size_t)batch * n_head * 2 * sizeof(float)) +
           (size_t)batch * n_head * raw_rows(max_len) * sizeof(float);
}

int nimllm_attn_decode_scored(const void *q, int q_dtype, const void *k_cache, const void *v_cache, int cache_dtype, const int64_t *kv_off,
                              int64_t seq_stride, int64_t head_stride, int max_seq, const int32_t *seq_len, int max_len, void *out,
                              int out_dtype, float *score, int64_t score_rows, float decay, int batch, int n_head, int n_kv_head,
                              int head_dim, float scale, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "attn_decode_scored";
    CacheRows rows;
    if (int rc = contiguous_rows(rows, who, k_cache, v_cache, cache_dtype, kv_off, seq_stride, head_stride, max_seq, head_dim)) return rc;
    return decode_scored(who, rows, q, q_dtype, k_cache, v_cache, cache_dtype, seq_len, max_len, out, out_dtype, score, score_rows, decay, batch,
                         n_head, n_kv_head, head_dim, scale, workspace, workspace_bytes, stream);
}

int nimllm_attn_decode_scored_paged(const void *q, int q_dtype, const void *k_pages, const void *v_pages, int cache_dtype,
                                    const int32_t *page_table, int max_pages, int page_rows, int n_pages, const int32_t *seq_len,
                                    int max_len, void *out, int out_dtype, float *score, int64_t score_rows, float decay, int batch,
                                    int n_head, int n_kv_head, int head_dim, float scale, void *workspace, size_t workspace_bytes,
                                    void *stream) {
    const char *who = "attn_decode_scored_paged";
    CacheRows rows;
    if (int rc = paged_rows(rows, who, k_pages, v_pages, cache_dtype, page_table, max_pages, page_rows, n_pages, n_kv_head, head_dim)) return rc;
    return decode_scored(who, rows, q, q_dtype, k_pages, v_pages, cache_dtype, seq_len, max_len, out, out_dtype, score, score_rows, decay, batch,
                         n_head, n_kv_head, head_dim, scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
