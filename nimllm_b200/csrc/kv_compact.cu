// kv_compact.cu -- rows of the KV cache moved down: the accepted path of a drafted tree, and the rows that an eviction keeps.
//
// Both are a gather with increasing sources, row i <- row src[i] with src[i] >= i, done in place.  A block owns whole columns
// (16-byte pieces of the rows) of one (sequence, KV head) and walks the destinations upwards in batches: it loads a batch's
// rows, waits for all of its threads, stores them.  A later batch reads rows src[j] >= j behind everything stored so far, so
// one barrier per batch is all the order that is needed.
#include "cache_rows.cuh"

namespace nimllm {

namespace {

// ------------------------------------------------------------------------------------------------ accepted path
struct AcceptParams {
    unsigned char *k, *v;
    CacheRows rows;
    int64_t layer_bytes;
    const int32_t *path, *n_path, *seq_len;
    int32_t *new_len;         // null: written by lens_kernel afterwards
    int max_path, n, L, B, Hkv;
    int elem, row16;          // bytes per element, 16-byte pieces per row
};

// The usable length of a path: it ends before the first entry that is not a draft of this tree or does not lie behind its
// predecessor.  Every thread of the block gets it; s_path holds the entries.
__device__ __forceinline__ int path_length(const AcceptParams &p, int b, int len, int *s_path, int *s_m) {
    const int m0 = clamp_len(p.n_path[b], p.max_path);
    if (threadIdx.x == 0) *s_m = m0;
    for (int i = threadIdx.x; i < m0; i += blockDim.x) s_path[i] = p.path[(int64_t)b * p.max_path + i];
    __syncthreads();
    for (int i = threadIdx.x; i < m0; i += blockDim.x) {
        const int x = s_path[i], before = i ? s_path[i - 1] : -1;
        if (x <= before || x >= p.n || x >= p.rows.cap - len) atomicMin(s_m, i);
    }
    __syncthreads();
    return *s_m;
}

__global__ void __launch_bounds__(256) accept_kernel(AcceptParams p) {
    __shared__ int s_path[kTreeMaxTokens];
    __shared__ int s_m;
    launch_dependents();
    grid_dependency_wait();
    const int kvh = blockIdx.x % p.Hkv, b = (blockIdx.x / p.Hkv) % p.B, layer = blockIdx.x / (p.Hkv * p.B);
    const int len = clamp_len(p.seq_len[b], p.rows.cap);
    const int m = path_length(p, b, len, s_path, &s_m);
    if (p.new_len && layer == 0 && kvh == 0 && threadIdx.x == 0) p.new_len[b] = len + m;
    unsigned char *kb = p.k + (int64_t)layer * p.layer_bytes, *vb = p.v + (int64_t)layer * p.layer_bytes;
    const int units = m * p.row16;
    for (int u0 = 0; u0 < units; u0 += blockDim.x) {
        const int u = u0 + threadIdx.x;
        int64_t to = -1, fro = -1;
        uint4 x, y;
        if (u < units) {
            const int i = u / p.row16, c = u - i * p.row16;
            if (s_path[i] != i) {
                to = cache_row(p.rows, b, kvh, len + i);
                fro = cache_row(p.rows, b, kvh, len + s_path[i]);
                if (fro < 0) to = -1;
                if (to >= 0) {
                    to = to * p.elem + c * 16;
                    fro = fro * p.elem + c * 16;
                    x = *reinterpret_cast<const uint4 *>(kb + fro);
                    y = *reinterpret_cast<const uint4 *>(vb + fro);
                }
            }
        }
        __syncthreads();
        if (to >= 0) {
            *reinterpret_cast<uint4 *>(kb + to) = x;
            *reinterpret_cast<uint4 *>(vb + to) = y;
        }
    }
}

// new_len is the array that accept_kernel reads: its blocks are all done when this one writes it
__global__ void __launch_bounds__(256) accept_lens_kernel(AcceptParams p, int32_t *new_len) {
    __shared__ int s_path[kTreeMaxTokens];
    __shared__ int s_m;
    launch_dependents();
    grid_dependency_wait();
    const int b = blockIdx.x;
    const int len = clamp_len(p.seq_len[b], p.rows.cap);
    const int m = path_length(p, b, len, s_path, &s_m);
    if (threadIdx.x == 0) new_len[b] = len + m;
}

int kv_accept(const char *who, const CacheRows &rows, void *k, void *v, int cache_dtype, int n_layer, int64_t layer_stride, const int32_t *path,
              int max_path, const int32_t *n_path, const int32_t *seq_len, int32_t *new_len, int n, int batch, int n_kv_head, int head_dim,
              void *stream) {
    if (!path || !n_path || !seq_len || !new_len) return fail(NIMLLM_ERR_ARG, "%s: null path / n_path / seq_len / new_len", who);
    if (batch <= 0 || n_kv_head <= 0 || n_layer <= 0 || n <= 0 || max_path <= 0)
        return fail(NIMLLM_ERR_ARG, "%s: bad shape B=%d Hkv=%d layers=%d n=%d max_path=%d", who, batch, n_kv_head, n_layer, n, max_path);
    if (n > kTreeMaxTokens || max_path > n)
        return fail(NIMLLM_ERR_UNSUPPORTED, "%s: n %d (at most %d), max_path %d (at most n)", who, n, kTreeMaxTokens, max_path);
    if ((int64_t)n_layer * batch * n_kv_head > 0x7fffffff) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: too many (layer, sequence, KV head) blocks", who);
    const int elem = (int)dtype_size(cache_dtype);
    if (head_dim <= 0 || head_dim * elem % 16 != 0) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: head_dim %d: rows must be a multiple of 16 bytes", who, head_dim);
    if (layer_stride * elem % 16 != 0) return fail(NIMLLM_ERR_ARG, "%s: layer_stride must be a multiple of 16 bytes", who);
    AcceptParams p;
    p.k = (unsigned char *)k; p.v = (unsigned char *)v; p.rows = rows; p.layer_bytes = layer_stride * elem;
    p.path = path; p.n_path = n_path; p.seq_len = seq_len; p.new_len = new_len == seq_len ? nullptr : new_len;
    p.max_path = max_path; p.n = n; p.L = n_layer; p.B = batch; p.Hkv = n_kv_head; p.elem = elem; p.row16 = head_dim * elem / 16;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = launch_dependent(accept_kernel, dim3(n_layer * batch * n_kv_head), 256, 0, st, p);
    if (e == cudaSuccess && !p.new_len) e = launch_dependent(accept_lens_kernel, dim3(batch), 256, 0, st, p, new_len);
    if (e != cudaSuccess) return fail(NIMLLM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return NIMLLM_OK;
}

// ------------------------------------------------------------------------------------------------ eviction
struct EvictParams {
    unsigned char *k, *v;
    CacheRows rows;
    float *score;             // [B][Hkv][score_rows]
    int64_t score_rows;
    const int32_t *seq_len;
    int32_t *new_len;         // null: written by evict_lens_kernel afterwards
    int32_t *kept;            // [B][Hkv][keep]
    int max_len, keep, n_sink, n_recent, B, Hkv;
    int elem, row16, split16; // 16-byte pieces per row and per block
};

__device__ __forceinline__ int evict_len(const EvictParams &p, int b) { return clamp_len(p.seq_len ? p.seq_len[b] : p.max_len, p.max_len); }

// order of the scores as unsigned numbers: -0 = +0, NaN below everything
__device__ __forceinline__ uint32_t score_key(float s) {
    if (s != s) return 0u;
    const uint32_t x = __float_as_uint(s + 0.f);      // -0 + 0 = +0
    return (x & 0x80000000u) ? ~x : (x | 0x80000000u);
}

constexpr int kSelThreads = 1024;

// One block per (sequence, KV head): the key of the last row that is kept by its score (radix select, 8 bits a pass), then
// the kept rows in order.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictParams p) {
    __shared__ int s_hist[256];
    __shared__ int s_digit, s_left;
    __shared__ int s_eq[kSelThreads / 32], s_keep[kSelThreads / 32];
    launch_dependents();
    grid_dependency_wait();
    const int pair = blockIdx.x, b = pair / p.Hkv;
    const int len = evict_len(p, b), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int32_t *kept = p.kept + (int64_t)pair * p.keep;
    if (p.new_len && pair % p.Hkv == 0 && tid == 0) p.new_len[b] = min(len, p.keep);
    if (len <= p.keep) {
        for (int i = tid; i < p.keep; i += kSelThreads) kept[i] = i < len ? i : -1;
        return;
    }
    const float *score = p.score + (int64_t)pair * p.score_rows;
    const int mid0 = p.n_sink, mid1 = len - p.n_recent;        // len > keep >= n_sink + n_recent
    int left = p.keep - p.n_sink - p.n_recent;                 // rows still to be chosen among those at or below the prefix
    uint32_t prefix = 0;
    if (left > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) s_hist[tid] = 0;
            __syncthreads();
            for (int r = mid0 + tid; r < mid1; r += kSelThreads) {
                const uint32_t key = score_key(score[r]);
                if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(key >> shift) & 255], 1);
            }
            __syncthreads();
            if (warp == 0) {
                // digits from the top: lane l holds 255 - 8l .. 248 - 8l
                int c[8], sum = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) { c[j] = s_hist[255 - 8 * lane - j]; sum += c[j]; }
                int incl = sum;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, incl, off);
                    if (lane >= off) incl += x;
                }
                int above = incl - sum;
                if (above < left && incl >= left) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        if (above < left && above + c[j] >= left) { s_digit = 255 - 8 * lane - j; s_left = left - above; }
                        above += c[j];
                    }
                }
            }
            __syncthreads();
            prefix |= (uint32_t)s_digit << shift;
            left = s_left;
            __syncthreads();
        }
    }
    // rows in order: 0.. n_sink, the middle rows above the last key or equal to it while any are left, the last n_recent
    int eq_before = 0, kept_before = 0;
    const bool none = p.keep == p.n_sink + p.n_recent;
    for (int r0 = 0; r0 < len; r0 += kSelThreads) {
        const int r = r0 + tid;
        const bool mid = r >= mid0 && r < mid1;
        const uint32_t key = mid ? score_key(score[r]) : 0u;
        const bool eq = mid && !none && key == prefix;
        const uint32_t eq_mask = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) s_eq[warp] = __popc(eq_mask);
        __syncthreads();
        int eq_rank = eq_before + __popc(eq_mask & ((1u << lane) - 1)), eq_all = 0;
        for (int w = 0; w < kSelThreads / 32; w++) {
            if (w < warp) eq_rank += s_eq[w];
            eq_all += s_eq[w];
        }
        const bool take = r < len && (!mid || (!none && (key > prefix || (eq && eq_rank < left))));
        const uint32_t mask = __ballot_sync(0xffffffffu, take);
        if (lane == 0) s_keep[warp] = __popc(mask);
        __syncthreads();
        int at = kept_before + __popc(mask & ((1u << lane) - 1)), all = 0;
        for (int w = 0; w < kSelThreads / 32; w++) {
            if (w < warp) at += s_keep[w];
            all += s_keep[w];
        }
        if (take) kept[at] = r;
        eq_before += eq_all;
        kept_before += all;
    }
}

constexpr int kMoveRows = 8;   // rows in flight per thread

__global__ void __launch_bounds__(256) evict_move_kernel(EvictParams p) {
    launch_dependents();
    grid_dependency_wait();
    const int pair = blockIdx.x, b = pair / p.Hkv, kvh = pair - b * p.Hkv;
    const int len = evict_len(p, b);
    if (len <= p.keep) return;
    const int32_t *kept = p.kept + (int64_t)pair * p.keep;
    const int splits = p.row16 / p.split16;
    if ((int)blockIdx.y == 2 * splits) {
        // the scores move with their rows; the rows to come start from nothing
        float *score = p.score + (int64_t)pair * p.score_rows;
        for (int j0 = 0; j0 < p.keep; j0 += 256 * kMoveRows) {
            float x[kMoveRows];
#pragma unroll
            for (int u = 0; u < kMoveRows; u++) {
                const int j = j0 + u * 256 + threadIdx.x;
                if (j < p.keep) x[u] = score[kept[j]];
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kMoveRows; u++) {
                const int j = j0 + u * 256 + threadIdx.x;
                if (j < p.keep) score[j] = x[u];
            }
        }
        __syncthreads();
        for (int r = p.keep + threadIdx.x; r < len; r += 256) score[r] = 0.f;
        return;
    }
    unsigned char *base = (int)blockIdx.y < splits ? p.k : p.v;
    const int c = ((int)blockIdx.y % splits) * p.split16 + (int)threadIdx.x % p.split16;
    const int rows_per_step = 256 / p.split16, row_in = (int)threadIdx.x / p.split16;
    for (int j0 = 0; j0 < p.keep; j0 += rows_per_step * kMoveRows) {
        uint4 x[kMoveRows];
        int64_t to[kMoveRows];
#pragma unroll
        for (int u = 0; u < kMoveRows; u++) {
            const int j = j0 + u * rows_per_step + row_in;
            to[u] = -1;
            if (j < p.keep) {
                const int r = kept[j];
                if (r != j) {
                    const int64_t fro = cache_row(p.rows, b, kvh, r);
                    to[u] = cache_row(p.rows, b, kvh, j);
                    if (fro < 0) to[u] = -1;
                    if (to[u] >= 0) {
                        to[u] = to[u] * p.elem + c * 16;
                        x[u] = *reinterpret_cast<const uint4 *>(base + fro * p.elem + c * 16);
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveRows; u++)
            if (to[u] >= 0) *reinterpret_cast<uint4 *>(base + to[u]) = x[u];
    }
}

__global__ void __launch_bounds__(256) evict_lens_kernel(EvictParams p, int32_t *new_len) {
    launch_dependents();
    grid_dependency_wait();
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < p.B) new_len[b] = min(evict_len(p, b), p.keep);
}

int kv_evict(const char *who, const CacheRows &rows, void *k, void *v, int cache_dtype, float *score, int64_t score_rows, const int32_t *seq_len,
             int max_len, int keep, int n_sink, int n_recent, int32_t *kept, int32_t *new_len, int batch, int n_kv_head, int head_dim,
             void *stream) {
    if (!score || !kept || !new_len) return fail(NIMLLM_ERR_ARG, "%s: null score / kept / new_len", who);
    if (batch <= 0 || n_kv_head <= 0 || max_len <= 0) return fail(NIMLLM_ERR_ARG, "%s: bad shape B=%d Hkv=%d max_len=%d", who, batch, n_kv_head, max_len);
    if (keep <= 0 || n_sink < 0 || n_recent < 0 || n_sink > keep || n_recent > keep - n_sink)
        return fail(NIMLLM_ERR_ARG, "%s: keep %d must be positive and hold n_sink %d + n_recent %d", who, keep, n_sink, n_recent);
    if (max_len > rows.cap) return fail(NIMLLM_ERR_ARG, "%s: max_len %d, a sequence holds %d rows", who, max_len, rows.cap);
    if (score_rows < max_len) return fail(NIMLLM_ERR_ARG, "%s: %lld scores per KV head, max_len %d", who, (long long)score_rows, max_len);
    if ((int64_t)batch * n_kv_head > 0x7fffffff) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: too many (sequence, KV head) pairs", who);
    const int elem = (int)dtype_size(cache_dtype);
    if (head_dim <= 0 || head_dim * elem % 16 != 0) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: head_dim %d: rows must be a multiple of 16 bytes", who, head_dim);
    EvictParams p;
    p.k = (unsigned char *)k; p.v = (unsigned char *)v; p.rows = rows; p.score = score; p.score_rows = score_rows; p.seq_len = seq_len;
    p.new_len = new_len == seq_len ? nullptr : new_len; p.kept = kept; p.max_len = max_len; p.keep = keep; p.n_sink = n_sink;
    p.n_recent = n_recent; p.B = batch; p.Hkv = n_kv_head; p.elem = elem; p.row16 = head_dim * elem / 16;
    // 64-byte column pieces where the row divides into them: more blocks than (sequence, KV head) pairs
    p.split16 = p.row16 % 4 == 0 ? 4 : (p.row16 % 2 == 0 ? 2 : 1);
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = launch_dependent(evict_select_kernel, dim3(batch * n_kv_head), kSelThreads, 0, st, p);
    if (e == cudaSuccess)
        e = launch_dependent(evict_move_kernel, dim3(batch * n_kv_head, 2 * (p.row16 / p.split16) + 1), 256, 0, st, p);
    if (e == cudaSuccess && !p.new_len) e = launch_dependent(evict_lens_kernel, dim3((batch + 255) / 256), 256, 0, st, p, new_len);
    if (e != cudaSuccess) return fail(NIMLLM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return NIMLLM_OK;
}

}  // namespace

}  // namespace nimllm

using namespace nimllm;

extern "C" {

int nimllm_kv_accept(void *k_cache, void *v_cache, int cache_dtype, int n_layer, int64_t layer_stride, const int64_t *kv_off,
                     int64_t seq_stride, int64_t head_stride, int max_seq, const int32_t *path, int max_path, const int32_t *n_path,
                     const int32_t *seq_len, int32_t *new_len, int n, int batch, int n_kv_head, int head_dim, void *stream) {
    CacheRows rows;
    if (int rc = contiguous_rows(rows, "kv_accept", k_cache, v_cache, cache_dtype, kv_off, seq_stride, head_stride, max_seq, head_dim)) return rc;
    return kv_accept("kv_accept", rows, k_cache, v_cache, cache_dtype, n_layer, layer_stride, path, max_path, n_path, seq_len, new_len, n, batch,
                     n_kv_head, head_dim, stream);
}

int nimllm_kv_accept_paged(void *k_pages, void *v_pages, int cache_dtype, int n_layer, int64_t layer_stride, const int32_t *page_table,
                           int max_pages, int page_rows, int n_pages, const int32_t *path, int max_path, const int32_t *n_path,
                           const int32_t *seq_len, int32_t *new_len, int n, int batch, int n_kv_head, int head_dim, void *stream) {
    CacheRows rows;
    if (int rc = paged_rows(rows, "kv_accept_paged", k_pages, v_pages, cache_dtype, page_table, max_pages, page_rows, n_pages, n_kv_head, head_dim)) return rc;
    return kv_accept("kv_accept_paged", rows, k_pages, v_pages, cache_dtype, n_layer, layer_stride, path, max_path, n_path, seq_len, new_len, n,
                     batch, n_kv_head, head_dim, stream);
}

int nimllm_kv_evict(void *k_cache, void *v_cache, int cache_dtype, const int64_t *kv_off, int64_t seq_stride, int64_t head_stride,
                    int max_seq, float *score, int64_t score_rows, const int32_t *seq_len, int max_len, int keep, int n_sink, int n_recent,
                    int32_t *kept, int32_t *new_len, int batch, int n_kv_head, int head_dim, void *stream) {
    CacheRows rows;
    if (int rc = contiguous_rows(rows, "kv_evict", k_cache, v_cache, cache_dtype, kv_off, seq_stride, head_stride, max_seq, head_dim)) return rc;
    return kv_evict("kv_evict", rows, k_cache, v_cache, cache_dtype, score, score_rows, seq_len, max_len, keep, n_sink, n_recent, kept, new_len,
                    batch, n_kv_head, head_dim, stream);
}

int nimllm_kv_evict_paged(void *k_pages, void *v_pages, int cache_dtype, const int32_t *page_table, int max_pages, int page_rows,
                          int n_pages, float *score, int64_t score_rows, const int32_t *seq_len, int max_len, int keep, int n_sink,
                          int n_recent, int32_t *kept, int32_t *new_len, int batch, int n_kv_head, int head_dim, void *stream) {
    CacheRows rows;
    if (int rc = paged_rows(rows, "kv_evict_paged", k_pages, v_pages, cache_dtype, page_table, max_pages, page_rows, n_pages, n_kv_head, head_dim)) return rc;
    return kv_evict("kv_evict_paged", rows, k_pages, v_pages, cache_dtype, score, score_rows, seq_len, max_len, keep, n_sink, n_recent, kept,
                    new_len, batch, n_kv_head, head_dim, stream);
}

}  // extern "C"
