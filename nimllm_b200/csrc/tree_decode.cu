// tree_decode.cu -- attention of drafted tokens over a KV cache, and decode that keeps score of the cached rows.
//
//   out[b, i, h] = sum_r w_r v_r,  w = softmax over the rows r that token i attends of  scale q . k_r
//   score[b, kvh, r] = decay * score[b, kvh, r] + sum over the query heads of kvh of w_r          (scored decode)
//
// This file holds the entry points, the CUDA-core kernel and the launches that finish a call.  The G query heads of a KV head
// and the n tokens of a sequence are rows of one tile, so that a cached row is read once for all of them.
#include "tree_finish.cuh"

namespace nimllm {

namespace {

constexpr int kBM = 32, kBN = 32;    // query rows and cached rows of a tile

template <int D> constexpr size_t fma_smem() { return (size_t)(kBM + 2 * kBN) * (D + 4) * sizeof(float) + (size_t)kBM * (kBN + 1) * sizeof(float); }

// One CTA: 32 query rows of one (sequence, KV head) over one chunk of cached rows.  fp32 throughout; a thread owns a 2 x 2
// piece of the score tile, then one query row's D/8 output columns.
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_fma_kernel(TreeParams p) {
    extern __shared__ float sm[];
    constexpr int LD = D + 4;
    float *sq = sm, *sk = sq + kBM * LD, *sv = sk + kBN * LD, *ss = sv + kBN * LD;
    launch_dependents();
    grid_dependency_wait();
    const int chunk = blockIdx.x, b = blockIdx.z;
    const int q_tiles = (p.n * p.G + kBM - 1) / kBM;
    const int kvh = blockIdx.y / q_tiles, q0 = (blockIdx.y % q_tiles) * kBM;
    const int len = tree_committed(p, b), drafts = tree_drafts(p, b, len);
    const int R = tree_tokens(p, b) * p.G;                 // live query rows
    if (q0 >= R) return;
    const int total = len + drafts;
    const int n_chunks = total <= p.chunk_rows ? 1 : (total + p.chunk_rows - 1) / p.chunk_rows;
    if (chunk >= n_chunks) return;
    const int r_begin = chunk * p.chunk_rows, r_end = min(total, r_begin + p.chunk_rows);
    const int tid = threadIdx.x;

    for (int x = tid; x < kBM * D; x += 256) {
        const int qr = x / D, d = x % D;
        float v = 0.f;
        if (q0 + qr < R) v = load_as_f32(p.q, p.q_dtype, tree_out_row(p, b, kvh, q0 + qr) * D + d) * p.scale_log2e;
        sq[qr * LD + d] = v;
    }
    const int row = tid >> 3, c8 = tid & 7;                // softmax and output: 8 threads per query row
    const int token = (q0 + row) / p.G;
    float m = -INFINITY, l = 0.f;
    float acc[D / 8];
#pragma unroll
    for (int i = 0; i < D / 8; i++) acc[i] = 0.f;

    constexpr int VEC = Elem<T>::kVec;
    const T *kg = reinterpret_cast<const T *>(p.k), *vg = reinterpret_cast<const T *>(p.v);
    for (int r0 = r_begin; r0 < r_end; r0 += kBN) {
        __syncthreads();
        for (int x = tid; x < kBN * (D / VEC); x += 256) {
            const int r = x / (D / VEC), c = (x % (D / VEC)) * VEC;
            float fk[VEC], fv[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) fk[i] = fv[i] = 0.f;
            if (r0 + r < r_end) {
                const int64_t at = cache_row(p.rows, b, kvh, r0 + r);
                if (at >= 0) {
                    Elem<T>::unpack(ldg_stream(kg + at + c), fk);
                    Elem<T>::unpack(ldg_stream(vg + at + c), fv);
                }
            }
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                *reinterpret_cast<float4 *>(sk + r * LD + c + i) = make_float4(fk[i], fk[i + 1], fk[i + 2], fk[i + 3]);
                *reinterpret_cast<float4 *>(sv + r * LD + c + i) = make_float4(fv[i], fv[i + 1], fv[i + 2], fv[i + 3]);
            }
        }
        __syncthreads();
        {
            const int ty = tid >> 4, tx = tid & 15;
            float s[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll 8
            for (int d = 0; d < D; d += 4) {
                float4 a[2], k[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    a[i] = *reinterpret_cast<const float4 *>(sq + (ty + 16 * i) * LD + d);
                    k[i] = *reinterpret_cast<const float4 *>(sk + (tx + 16 * i) * LD + d);
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        s[i][j] = fmaf(a[i].x, k[j].x, fmaf(a[i].y, k[j].y, fmaf(a[i].z, k[j].z, fmaf(a[i].w, k[j].w, s[i][j]))));
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) ss[(ty + 16 * i) * (kBN + 1) + tx + 16 * j] = s[i][j];
        }
        __syncthreads();
        const bool tail = r0 + kBN > len;                  // rows that not every token attends, or no rows
        float x[4], mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = c8 + 8 * j, r = r0 + c;
            x[j] = ss[row * (kBN + 1) + c];
            bool see = r < r_end && q0 + row < R;
            if (see && tail && r >= len) see = tree_sees(p, b, token, r - len);
            if (see && p.rows.table) see = cache_row(p.rows, b, kvh, r) >= 0;
            if (!see) x[j] = -INFINITY;
            if (see && p.raw) p.raw[((int64_t)b * p.Hq + kvh * p.G + q0 + row) * p.raw_ld + r] = x[j];
            mx = fmaxf(mx, x[j]);
        }
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float m_new = fmaxf(m, mx), safe = m_new == -INFINITY ? 0.f : m_new;
        const float corr = ex2(m - safe);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[j] = ex2(x[j] - safe);
            sum += x[j];
            ss[row * (kBN + 1) + c8 + 8 * j] = x[j];
        }
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        l = l * corr + sum;
        m = m_new;
#pragma unroll
        for (int i = 0; i < D / 8; i++) acc[i] *= corr;
        __syncwarp();                                      // a query row's eight threads are in one warp
        for (int r = 0; r < kBN; r++) {
            const float w = ss[row * (kBN + 1) + r];
            if (tail && w == 0.f) continue;                // a row that is not attended may hold anything
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                const float4 v = *reinterpret_cast<const float4 *>(sv + r * LD + i * 32 + c8 * 4);
                acc[4 * i] = fmaf(w, v.x, acc[4 * i]);
                acc[4 * i + 1] = fmaf(w, v.y, acc[4 * i + 1]);
                acc[4 * i + 2] = fmaf(w, v.z, acc[4 * i + 2]);
                acc[4 * i + 3] = fmaf(w, v.w, acc[4 * i + 3]);
            }
        }
    }
    if (q0 + row >= R) return;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int64_t orow = tree_out_row(p, b, kvh, q0 + row);
    constexpr int W = D + 4;
    float *rec = n_chunks > 1 ? p.recs + ((int64_t)chunk * p.B * p.n * p.Hq + orow) * W : (p.partials_out ? p.partials_out + orow * W : nullptr);
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = i * 32 + c8 * 4 + j;
            const float val = acc[4 * i + j] * inv;
            if (rec) rec[d] = val;
            if (n_chunks == 1 && p.out) store_from_f32(p.out, p.out_dtype, orow * D + d, val);
        }
    if (c8 == 0) {
        if (rec) *reinterpret_cast<float4 *>(rec + D) = make_float4(m * kLn2, l, 0.f, 0.f);
        if (p.stats) *reinterpret_cast<float2 *>(p.stats + 2 * orow) = make_float2(m, n_chunks == 1 ? inv : -1.f);   // -1: cut
    }
}

// rows of a chunk: enough CTAs for four on every SM, at least 128 rows each
int tree_chunk_rows(int batch, int n, int n_head, int n_kv_head, int max_total) {
    const int64_t tiles = (int64_t)batch * n_kv_head * (((int64_t)n * (n_head / n_kv_head) + kBM - 1) / kBM);
    int64_t c = (tiles * max_total + 4 * sm_count() - 1) / (4 * sm_count());
    const int64_t least = ((int64_t)max_total + treetc::kMaxPieces - 1) / treetc::kMaxPieces;
    c = c < least ? least : c;
    c = (c + kBN - 1) / kBN * kBN;
    return (int)(c < 128 ? 128 : (c > (1 << 30) ? 1 << 30 : c));
}
size_t fma_record_bytes(int batch, int n, int n_head, int n_kv_head, int head_dim, int max_total) {
    const int chunk = tree_chunk_rows(batch, n, n_head, n_kv_head, max_total);
    const int64_t chunks = ((int64_t)max_total + chunk - 1) / chunk;
    return chunks <= 1 ? 0 : (size_t)chunks * batch * n * n_head * rec_stride(head_dim) * sizeof(float);
}
size_t round256(size_t x) { return (x + 255) / 256 * 256; }
bool use_tensor_cores(int cache_dtype) { return cache_dtype == NIMLLM_BF16; }
size_t record_bytes(int batch, int n, int n_head, int n_kv_head, int head_dim, int max_total, int cache_dtype) {
    return round256(use_tensor_cores(cache_dtype) ? tree_tc_workspace_bytes(batch, n, n_head, n_kv_head, head_dim)
                                                    : fma_record_bytes(batch, n, n_head, n_kv_head, head_dim, max_total));
}
// whole tiles of the tensor-core kernels are written
int64_t raw_rows(int max_len) { return ((int64_t)max_len + 127) / 128 * 128; }

template <typename T, int D>
cudaError_t launch_fma(const TreeParams &p, dim3 grid, cudaStream_t st) {
    static bool ready[64] = {};                            // the attribute is per device; setting it twice does no harm
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(tree_fma_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)fma_smem<D>());
        if (e != cudaSuccess) return e;
        if (dev < 64) ready[dev] = true;
    }
    e = launch_dependent(tree_fma_kernel<T, D>, grid, 256, fma_smem<D>(), st, p);
    treetc::FinishArgs f = {};
    return e == cudaSuccess ? treetc::launch_finish<D>(p, f, st) : e;
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
    cudaError_t e = cudaSuccess;
    if (use_tensor_cores(cache_dtype)) {
        if (int rc = launch_tree_tc(who, p, head_dim, ws, st)) return rc;
    } else {
        p.chunk_rows = tree_chunk_rows(p.B, p.n, p.Hq, p.Hkv, max_total);
        p.max_chunks = (int)(((int64_t)max_total + p.chunk_rows - 1) / p.chunk_rows);
        const int q_tiles = (p.n * p.G + kBM - 1) / kBM;
        const dim3 grid(p.max_chunks, p.Hkv * q_tiles, p.B);
        e = head_dim == 64 ? launch_fma<float, 64>(p, grid, st) : launch_fma<float, 128>(p, grid, st);
    }
    if (e != cudaSuccess) return fail(NIMLLM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return NIMLLM_OK;
}

int check_shape(const char *who, const void *q, int q_dtype, const void *out, int out_dtype, const float *partials_out, int max_len,
                int batch, int n, int n_head, int n_kv_head, int head_dim) {
    if (!q || (!out && !partials_out)) return fail(NIMLLM_ERR_ARG, "%s: null q / output pointer", who);
    if (batch <= 0 || n <= 0 || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || max_len < 0)
        return fail(NIMLLM_ERR_ARG, "%s: bad shape B=%d n=%d Hq=%d Hkv=%d max_len=%d", who, batch, n, n_head, n_kv_head, max_len);
    if (!dtype_ok(q_dtype) || !dtype_ok(out_dtype)) return fail(NIMLLM_ERR_ARG, "%s: unknown dtype", who);
    if (head_dim != 64 && head_dim != 128) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: head_dim %d (64 and 128 are built)", who, head_dim);
    if (n > kTreeMaxTokens) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: n %d > %d", who, n, kTreeMaxTokens);
    if (batch > 65535 || (int64_t)n_kv_head * (((int64_t)n * (n_head / n_kv_head) + kBM - 1) / kBM) > 65535 || max_len > (1 << 30))
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
    if (batch <= 0 || n <= 0 || n > kTreeMaxTokens || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || head_dim <= 0 || max_len < 0) return 0;
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
    if (batch <= 0 || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || head_dim <= 0 || max_len <= 0) return 0;
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
