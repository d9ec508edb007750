// cache_rows.cuh -- where a row of the KV cache lives, for the kernels that take both layouts.
#pragma once
#include "common.cuh"

namespace nimllm {

constexpr int kTreeMaxTokens = 256;   // drafted tokens of one sequence

// contiguous (table == null): sequence b at kv_off[b] or b * seq_stride, KV head h at h * head_stride, row r at r * D;
// paged: row r in page table[b][r >> page_shift], a page is [Hkv][page_rows][D].  All in elements.
struct CacheRows {
    const int64_t *kv_off;
    int64_t seq_stride, head_stride;
    const int32_t *table;
    int max_pages, page_shift, n_pages;
    int64_t page_stride;
    int cap;                          // rows that a (sequence, KV head) block can hold
    int D;
};

// element offset of a row of K (and of V), -1 when the row has no page.  0 <= r < cap.
__device__ __forceinline__ int64_t cache_row(const CacheRows &c, int b, int kvh, int r) {
    if (c.table) {
        const int pg = c.table[(int64_t)b * c.max_pages + (r >> c.page_shift)];
        if (pg < 0 || pg >= c.n_pages) return -1;
        return (int64_t)pg * c.page_stride + (((int64_t)kvh << c.page_shift) + (r & ((1 << c.page_shift) - 1))) * c.D;
    }
    return (c.kv_off ? c.kv_off[b] : (int64_t)b * c.seq_stride) + (int64_t)kvh * c.head_stride + (int64_t)r * c.D;
}

__device__ __forceinline__ int clamp_len(int v, int hi) { return v < 0 ? 0 : (v > hi ? hi : v); }

// The host's checks of the two layouts (NIMLLM_OK or the status with its message set).
inline int contiguous_rows(CacheRows &c, const char *who, const void *k, const void *v, int dtype, const int64_t *kv_off,
                           int64_t seq_stride, int64_t head_stride, int max_seq, int head_dim) {
    if (!k || !v) return fail(NIMLLM_ERR_ARG, "%s: null cache", who);
    if (!dtype_ok(dtype)) return fail(NIMLLM_ERR_ARG, "%s: unknown dtype", who);
    if (max_seq <= 0) return fail(NIMLLM_ERR_ARG, "%s: max_seq %d", who, max_seq);
    if (((uintptr_t)k | (uintptr_t)v) & 15) return fail(NIMLLM_ERR_ARG, "%s: cache pointers must be 16-byte aligned", who);
    const int64_t per16 = 16 / (int64_t)dtype_size(dtype);
    if (head_stride % per16 != 0 || (!kv_off && seq_stride % per16 != 0))
        return fail(NIMLLM_ERR_ARG, "%s: seq_stride and head_stride must be multiples of 16 bytes", who);
    c = CacheRows{kv_off, seq_stride, head_stride, nullptr, 0, 0, 0, 0, max_seq, head_dim};
    return NIMLLM_OK;
}
inline int paged_rows(CacheRows &c, const char *who, const void *k, const void *v, int dtype, const int32_t *page_table,
                      int max_pages, int page_rows, int n_pages, int n_kv_head, int head_dim) {
    if (!k || !v || !page_table) return fail(NIMLLM_ERR_ARG, "%s: null pages / page table", who);
    if (!dtype_ok(dtype)) return fail(NIMLLM_ERR_ARG, "%s: unknown dtype", who);
    int shift = 0;
    while (shift < 30 && (1 << shift) < page_rows) shift++;
    if (page_rows < 32 || (1 << shift) != page_rows)
        return fail(NIMLLM_ERR_ARG, "%s: page_rows %d must be a power of two >= 32", who, page_rows);
    if (max_pages <= 0 || n_pages <= 0 || (int64_t)max_pages * page_rows > 0x7fffffff)
        return fail(NIMLLM_ERR_ARG, "%s: bad max_pages %d / n_pages %d", who, max_pages, n_pages);
    if (((uintptr_t)k | (uintptr_t)v) & 15) return fail(NIMLLM_ERR_ARG, "%s: pages must be 16-byte aligned", who);
    c = CacheRows{nullptr, 0, 0, page_table, max_pages, shift, n_pages, (int64_t)n_kv_head * page_rows * head_dim, max_pages * page_rows, head_dim};
    return NIMLLM_OK;
}

// True when no two blocks of `block` elements overlap that lie stride[i] apart in each of three directions, count[i] of them (moves in
// place by a thread block per cache block race with one another otherwise).  Strides that nest, each one clear of all that the
// smaller ones reach over, are apart; for others every difference of two blocks is looked at.
inline bool blocks_apart(int64_t block, const int64_t (&count_in)[3], const int64_t (&stride_in)[3]) {
    __int128 n[3] = {1, 1, 1}, s[3] = {0, 0, 0};
    int m = 0;
    for (int i = 0; i < 3; i++) {
        if (count_in[i] <= 1) continue;
        __int128 x = stride_in[i];
        x = x < 0 ? -x : x;
        if (x < block) return false;
        int at = m++;
        for (; at > 0 && s[at - 1] > x; at--) { s[at] = s[at - 1]; n[at] = n[at - 1]; }
        s[at] = x; n[at] = count_in[i];
    }
    __int128 reach = block;
    bool nested = true;
    for (int i = 0; i < m; i++) {
        nested &= s[i] >= reach;
        reach += s[i] * (n[i] - 1);
    }
    if (nested) return true;
    for (__int128 k = 0; k < n[2]; k++)
        for (__int128 j = k ? 1 - n[1] : 0; j < n[1]; j++) {
            if (j == 0 && k == 0) continue;                // one direction alone: its stride clears a block
            const __int128 d = j * s[1] + k * s[2];
            for (__int128 i = -d / s[0] - 1; i <= -d / s[0] + 1; i++) {
                if (i <= -n[0] || i >= n[0]) continue;
                const __int128 gap = d + i * s[0];
                if (gap < block && gap > -(__int128)block) return false;
            }
        }
    return true;
}

// The programmatic-dependent launch that the decode kernels use: the kernel waits on the device (grid_dependency_wait)
// before it touches memory.
template <typename... P, typename... A>
inline cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace nimllm
