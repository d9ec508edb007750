// kv_compact.cu -- rows of the KV cache moved down: the accepted path of a drafted tree, and the rows that an eviction keeps.
//
// Both are a gather with increasing sources, row i <- row src[i] with src[i] >= i, done in place.  A block owns whole columns
// (16-byte pieces of the rows) of one (sequence, KV head) and walks the destinations upwards in batches: it loads a batch's
// rows, waits for all of its threads, stores them.  A later batch reads rows src[j] >= j behind everything stored so far, so
// one barrier per batch is all the order that is needed.
//
// Both are bound by HBM once they are large.  Measured (graph replay): accepting along trees of 64 tokens, 48 sequences x 30 layers of
// 8 heads of 128 bf16, 31.6 us = 6.0 TB/s; one sequence 4.2 us.  Evicting 8 sequences of 20 - 32 K rows to 8 K, 129 us: 24 for the
// selection, 103 for the rows, whose sources are scattered rows of 256 bytes (5.2 TB/s counted as read and written); one sequence of
// 512 rows 14.4 us, two launches.
#include <cooperative_groups.h>

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

// Both operators move rows within their blocks, a block at a time: blocks that overlap are refused.  With kv_off the host does not know
// how far the sequences lie apart.
int check_apart(const char *who, const CacheRows &rows, int n_layer, int64_t layer_stride, int batch, int n_kv_head) {
    if (rows.table) {
        if (n_layer > 1 && (layer_stride < 0 ? -layer_stride : layer_stride) < rows.n_pages * rows.page_stride)
            return fail(NIMLLM_ERR_ARG, "%s: layer_stride %lld: the pages of two layers overlap", who, (long long)layer_stride);
        return NIMLLM_OK;
    }
    if (blocks_apart((int64_t)rows.cap * rows.D, {n_layer, rows.kv_off ? 1 : batch, n_kv_head}, {layer_stride, rows.seq_stride, rows.head_stride})) return NIMLLM_OK;
    return fail(NIMLLM_ERR_ARG, "%s: layer_stride %lld, seq_stride %lld, head_stride %lld: blocks of max_seq rows overlap", who, (long long)layer_stride,
                (long long)rows.seq_stride, (long long)rows.head_stride);
}

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
    if (int rc = check_apart(who, rows, n_layer, layer_stride, batch, n_kv_head)) return rc;
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

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kSelBins = 2048;
constexpr int kSelKeys = 40960;        // keys that a block keeps in shared memory; a longer part is read again in every pass

// A cluster of blocks per (sequence, KV head), each with a consecutive part of the rows: the key of the last row that is kept by its
// score (radix select, digits of 11, 11 and 10 bits, histograms summed over the cluster's shared memory), then the kept rows in
// order.  A warp has consecutive rows too, so that their places follow from one prefix over the warps.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t s_key[];
    __shared__ int s_hist[3][kSelBins];
    __shared__ int s_warp[kSelWarps], s_digit, s_left;
    __shared__ int2 s_cnt[kSelWarps];
    __shared__ int2 s_total;
    launch_dependents();
    grid_dependency_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int pair = blockIdx.x / parts, b = pair / p.Hkv;
    const int len = evict_len(p, b), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int32_t *kept = p.kept + (int64_t)pair * p.keep;
    if (p.new_len && part == 0 && pair % p.Hkv == 0 && tid == 0) p.new_len[b] = min(len, p.keep);
    if (len <= p.keep) {                                   // the same in every block of the cluster
        for (int i = part * kSelThreads + tid; i < p.keep; i += parts * kSelThreads) kept[i] = i < len ? i : -1;
        return;
    }
    const float *score = p.score + (int64_t)pair * p.score_rows;
    const int mid0 = p.n_sink, mid1 = len - p.n_recent;    // len > keep >= n_sink + n_recent
    // this block's rows: whole groups of 32 for every warp
    const int per_warp = ((len + parts * kSelWarps - 1) / (parts * kSelWarps) + 31) / 32 * 32;
    const int begin = part * kSelWarps * per_warp, rows = max(0, min(len - begin, kSelWarps * per_warp));
    const bool in_smem = kSelWarps * per_warp <= kSelKeys;
    if (in_smem)
        for (int i = tid; i < rows; i += kSelThreads) s_key[i] = score_key(score[begin + i]);
    for (int i = tid; i < 3 * kSelBins; i += kSelThreads) (&s_hist[0][0])[i] = 0;
    __syncthreads();
    auto key_of = [&](int i) { return in_smem ? s_key[i] : score_key(score[begin + i]); };
    auto is_mid = [&](int i) { return begin + i >= mid0 && begin + i < mid1; };

    const int wanted = p.keep - p.n_sink - p.n_recent;
    int left = wanted;                                     // rows still to be chosen among those with the prefix
    uint32_t prefix = 0;
    if (wanted > 0) {
#pragma unroll 1
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11, above = shift + bits;
            for (int i = tid; i < rows; i += kSelThreads) {
                const uint32_t key = key_of(i);
                if (is_mid(i) && (pass == 0 || (key >> above) == (prefix >> above))) atomicAdd(&s_hist[pass][(key >> shift) & ((1 << bits) - 1)], 1);
            }
            cluster.sync();
            // thread t has the digits 2047 - 2t and 2046 - 2t, highest first
            int c0 = 0, c1 = 0;
            for (int q = 0; q < parts; q++) {
                const int *h = cluster.map_shared_rank(&s_hist[pass][0], q);
                c0 += h[kSelBins - 1 - 2 * tid];
                c1 += h[kSelBins - 2 - 2 * tid];
            }
            int incl = c0 + c1;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += x;
            }
            if (lane == 31) s_warp[warp] = incl;
            __syncthreads();
            int before = incl - c0 - c1 + __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[lane] : 0);
            if (before < left && before + c0 >= left) { s_digit = kSelBins - 1 - 2 * tid; s_left = left - before; }
            else if (before + c0 < left && before + c0 + c1 >= left) { s_digit = kSelBins - 2 - 2 * tid; s_left = left - before - c0; }
            __syncthreads();
            prefix |= (uint32_t)s_digit << shift;
            left = s_left;
        }
    }
    // kept: the rows in front and behind, the middle ones above the last key, and of those equal to it the first `left`
    const int w0 = warp * per_warp, w1 = min(rows, w0 + per_warp);
    int above = 0, equal = 0;
    for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t key = key_of(i);
        const bool mid = is_mid(i);
        above += !mid || (wanted > 0 && key > prefix);
        equal += mid && wanted > 0 && key == prefix;
    }
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) s_cnt[warp] = make_int2(above, equal);
    __syncthreads();
    const int2 mine = s_cnt[lane];
    if (warp == 0) {
        const int x = __reduce_add_sync(0xffffffffu, mine.x), y = __reduce_add_sync(0xffffffffu, mine.y);
        if (lane == 0) s_total = make_int2(x, y);
    }
    cluster.sync();
    int above_before = 0, equal_before = 0;
    for (int q = 0; q < part; q++) {
        const int2 t = *cluster.map_shared_rank(&s_total, q);
        above_before += t.x;
        equal_before += t.y;
    }
    above_before += __reduce_add_sync(0xffffffffu, lane < warp ? mine.x : 0);
    equal_before += __reduce_add_sync(0xffffffffu, lane < warp ? mine.y : 0);
    for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t key = i < w1 ? key_of(i) : 0u;
        const bool mid = is_mid(i);
        const bool up = i < w1 && (!mid || (wanted > 0 && key > prefix)), eq = i < w1 && mid && wanted > 0 && key == prefix;
        const uint32_t up_mask = __ballot_sync(0xffffffffu, up), eq_mask = __ballot_sync(0xffffffffu, eq), lower = (1u << lane) - 1;
        const int eq_rank = equal_before + __popc(eq_mask & lower);
        // in front of row i: all that are above, and the equal ones as far as they are kept
        if (up || (eq && eq_rank < left)) kept[above_before + __popc(up_mask & lower) + min(eq_rank, left)] = begin + i;
        above_before += __popc(up_mask);
        equal_before += __popc(eq_mask);
    }
    cluster.sync();                                        // nobody leaves while its shared memory may still be read
}

constexpr int kMoveThreads = 512, kMoveRows = 4, kMoveStages = 3;      // rows of a thread in a batch, batches under way
constexpr int kMoveSmem = kMoveStages * kMoveRows * kMoveThreads * 16;

// A block owns whole columns of one (sequence, KV head).  Batches are fetched with cp.async into shared memory that only the fetching
// thread reads again, two batches ahead of the one that is stored.
__global__ void __launch_bounds__(kMoveThreads, 2) evict_move_kernel(EvictParams p) {
    extern __shared__ uint4 s_move[];
    launch_dependents();
    grid_dependency_wait();
    const int pair = blockIdx.x, b = pair / p.Hkv, kvh = pair - b * p.Hkv, tid = threadIdx.x;
    const int len = evict_len(p, b);
    if (len <= p.keep) return;
    const int32_t *kept = p.kept + (int64_t)pair * p.keep;
    const int splits = p.row16 / p.split16;
    if ((int)blockIdx.y == 2 * splits) {
        // the scores move with their rows; the rows to come start from nothing
        float *score = p.score + (int64_t)pair * p.score_rows;
        constexpr int kBatch = 8;
        for (int j0 = 0; j0 < p.keep; j0 += kMoveThreads * kBatch) {
            float x[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                const int j = j0 + u * kMoveThreads + tid;
                if (j < p.keep) x[u] = score[kept[j]];
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                const int j = j0 + u * kMoveThreads + tid;
                if (j < p.keep) score[j] = x[u];
            }
        }
        __syncthreads();
        for (int r = p.keep + tid; r < len; r += kMoveThreads) score[r] = 0.f;
        return;
    }
    const int step = kMoveThreads / p.split16, row_in = tid / p.split16, batch = step * kMoveRows;
    const bool idle = row_in >= step;                      // threads that a piece of a row does not divide into
    unsigned char *base = ((int)blockIdx.y < splits ? p.k : p.v) + (((int)blockIdx.y % splits) * p.split16 + tid % p.split16) * 16;
    const bool paged = p.rows.table != nullptr;
    const int row_bytes = p.row16 * 16;
    if (!paged) base += cache_row(p.rows, b, kvh, 0) * p.elem;
    auto row_at = [&](int r) -> int64_t {                  // bytes from base; < 0: no page
        if (!paged) return (int64_t)r * row_bytes;
        const int64_t at = cache_row(p.rows, b, kvh, r);
        return at < 0 ? -1 : at * p.elem;
    };
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(s_move) + tid * 16;
    int next[kMoveRows];                                   // the sources of the batch that is fetched next
    auto fetch_index = [&](int j0) {
#pragma unroll
        for (int u = 0; u < kMoveRows; u++) {
            const int j = j0 + u * step + row_in;
            next[u] = j < p.keep && !idle ? kept[j] : -1;
        }
    };
    uint32_t moves[kMoveStages];                           // per stage: the rows that move, one bit each
    auto fetch = [&](int stage, int j0) {
        uint32_t m = 0;
#pragma unroll
        for (int u = 0; u < kMoveRows; u++) {
            const int j = j0 + u * step + row_in;
            if (next[u] >= 0 && next[u] != j) {
                const int64_t fro = row_at(next[u]);
                if (fro >= 0 && (!paged || row_at(j) >= 0)) {
                    m |= 1u << u;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + (stage * kMoveRows + u) * (kMoveThreads * 16)), "l"(base + fro) : "memory");
                }
            }
        }
        moves[stage] = m;
        asm volatile("cp.async.commit_group;" ::: "memory");
        fetch_index(j0 + batch);
    };
    // A batch stores rows j .. j + batch - 1 only, behind the barrier that says that everybody has fetched it; the batches behind it have
    // their sources at or behind j + batch and may be fetched before or after.
    fetch_index(0);
#pragma unroll
    for (int t = 0; t < kMoveStages - 1; t++) fetch(t, t * batch);
    for (int j0 = 0; j0 < p.keep; j0 += kMoveStages * batch) {
#pragma unroll
        for (int t = 0; t < kMoveStages; t++) {
            fetch((t + kMoveStages - 1) % kMoveStages, j0 + (t + kMoveStages - 1) * batch);
            asm volatile("cp.async.wait_group %0;" ::"n"(kMoveStages - 1) : "memory");
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kMoveRows; u++)
                if ((moves[t] >> u) & 1)
                    __stcs(reinterpret_cast<uint4 *>(base + row_at(j0 + t * batch + u * step + row_in)), s_move[(t * kMoveRows + u) * kMoveThreads + tid]);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
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
    if (int rc = check_apart(who, rows, 1, 0, batch, n_kv_head)) return rc;
    EvictParams p;
    p.k = (unsigned char *)k; p.v = (unsigned char *)v; p.rows = rows; p.score = score; p.score_rows = score_rows; p.seq_len = seq_len;
    p.new_len = new_len == seq_len ? nullptr : new_len; p.kept = kept; p.max_len = max_len; p.keep = keep; p.n_sink = n_sink;
    p.n_recent = n_recent; p.B = batch; p.Hkv = n_kv_head; p.elem = elem; p.row16 = head_dim * elem / 16;
    // whole rows to a block while the (sequence, KV head) pairs fill the GPU, else column pieces of 64 bytes at least: 64 pairs of
    // 8 K rows of 256 bytes take 129 us in pieces and 143 in whole rows, 8 pairs of 20 K rows 81 and 185
    const int64_t pairs = (int64_t)batch * n_kv_head;
    p.split16 = p.row16;
    while (p.split16 > 4 && p.split16 % 2 == 0 && 2 * pairs * (p.row16 / p.split16) < sm_count()) p.split16 /= 2;
    if (p.split16 > kMoveThreads) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: head_dim %d", who, head_dim);
    // blocks of a cluster that select for a pair: as many as the SMs hold at once, 2048 rows each at least.  One block a pair instead:
    // 140 us for 129 (64 pairs of 32 K rows), 88 for 81 (8 pairs)
    int parts = 1;
    while (parts < 8 && 2 * pairs * parts <= sm_count() && max_len >= parts * 4096) parts *= 2;
    const size_t part_rows = (((size_t)max_len + parts * kSelWarps - 1) / (parts * kSelWarps) + 31) / 32 * 32 * kSelWarps;
    const size_t smem = (part_rows <= kSelKeys ? part_rows : kSelKeys) * sizeof(uint32_t);
    if (pairs * parts > 0x7fffffff) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: too many (sequence, KV head) pairs", who);
    cudaStream_t st = (cudaStream_t)stream;
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !ready[dev])) {
        e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelKeys * (int)sizeof(uint32_t));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(evict_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMoveSmem);
        if (e == cudaSuccess && dev < 64) ready[dev] = true;
    }
    if (e == cudaSuccess) {
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = parts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(pairs * parts)); cfg.blockDim = dim3(kSelThreads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
        cfg.attrs = attr; cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, evict_select_kernel, p);
    }
    if (e == cudaSuccess)
        e = launch_dependent(evict_move_kernel, dim3((unsigned)pairs, 2 * (p.row16 / p.split16) + 1), kMoveThreads, kMoveSmem, st, p);
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
