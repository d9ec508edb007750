// tree_finish.cuh -- the one launch behind the attention kernels of tree and scored decode: pieces of cut rows are joined, rows
// without anything to attend become zeros, and the scores of a scored decode are brought up to date.
//
// The three jobs are independent (a score block joins the maxima and sums that it needs by itself), so they share a launch: block
// numbers first count the joins, then groups of 32 sequences, then the score blocks.
#pragma once
#include "tree_tc.cuh"

namespace nimllm {
namespace treetc {

constexpr int kFinishThreads = 256, kScoreRows = 4 * kFinishThreads;

// The pieces of a query row.  Tensor-core kernels: records of consecutive CTAs (tree_tc.cuh); CUDA-core kernel: one record per chunk of
// rows.  n = 1: the kernel stored the row itself; n = 0: there was nothing to attend.
struct Pieces {
    int n;
    const float *first, *second;       // record of piece 0, of piece 1; the others follow at `step`
    int64_t step;
    __device__ const float *rec(int x) const { return x == 0 ? first : second + (x - 1) * step; }
};
struct FinishArgs {
    TcArgs tc;
    int rpt, tile, workers;            // tensor-core kernels; workers = 0: the chunks of the CUDA-core kernel
    int join_rows, n_join, n_zero, n_score;   // query rows of a join block; blocks of the three kinds
};

template <int D> __device__ __forceinline__ Pieces tc_pieces(const TreeParams &p, const FinishArgs &f, int b, int kvh, int qr, int total, int R) {
    constexpr int W = D + 4;
    Pieces x{0, nullptr, nullptr, 0};
    if (total == 0) return x;
    const int64_t T = f.tc.cum[p.B];
    const int wa = (int)(T < f.workers ? T : f.workers);
    const int q_tiles = (R + f.rpt - 1) / f.rpt, tiles = (total + f.tile - 1) / f.tile;
    const int qt = qr / f.rpt, r = qr - qt * f.rpt;
    const int64_t s = f.tc.cum[b] + ((int64_t)kvh * q_tiles + qt) * tiles;
    const int w0 = owner_of(s, T, wa);
    x.n = owner_of(s + tiles - 1, T, wa) - w0 + 1;
    x.step = (int64_t)2 * f.tc.rec_rows * W;
    x.first = p.recs + ((int64_t)w0 * 2 + (first_unit(w0, T, wa) < s ? 1 : 0)) * f.tc.rec_rows * W + r * W;
    x.second = p.recs + ((int64_t)(w0 + 1) * 2) * f.tc.rec_rows * W + r * W;
    return x;
}
template <int D> __device__ __forceinline__ Pieces chunk_pieces(const TreeParams &p, int64_t orow, int total) {
    constexpr int W = D + 4;
    Pieces x;
    x.n = total <= p.chunk_rows ? 1 : (total + p.chunk_rows - 1) / p.chunk_rows;      // an empty row is stored by chunk 0
    x.step = (int64_t)p.B * p.n * p.Hq * W;
    x.first = p.recs + orow * W;
    x.second = x.first + x.step;
    return x;
}

// maximum (natural units) and, relative to it, the sum of a row's pieces, in every lane
template <int D> __device__ __forceinline__ void pieces_stats(const Pieces &x, int lane, float &M, float &L) {
    M = -INFINITY;
    for (int i = lane; i < x.n; i += 32) {
        const float2 ml = *reinterpret_cast<const float2 *>(x.rec(i) + D);
        if (ml.y > 0.f) M = fmaxf(M, ml.x);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    const float safe = M == -INFINITY ? 0.f : M;
    L = 0.f;
    for (int i = lane; i < x.n; i += 32) {
        const float2 ml = *reinterpret_cast<const float2 *>(x.rec(i) + D);
        if (ml.y > 0.f) L += ml.y * ex2((ml.x - safe) * kLog2e);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
}

// one warp: the row that its pieces make
template <int D> __device__ __forceinline__ void join_row(const TreeParams &p, const Pieces &x, int64_t orow, int lane) {
    float M, L;
    pieces_stats<D>(x, lane, M, L);
    const float safe = M == -INFINITY ? 0.f : M, inv = L > 0.f ? 1.f / L : 0.f;
    constexpr int V = D / 32;                              // columns of a lane, side by side
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = 0.f;
#pragma unroll 8
    for (int i = 0; i < x.n; i++) {
        const float *rec = x.rec(i);
        const float2 ml = *reinterpret_cast<const float2 *>(rec + D);
        const float w = ml.y > 0.f ? ml.y * ex2((ml.x - safe) * kLog2e) * inv : 0.f;
        if constexpr (V == 4) {
            const float4 o = *reinterpret_cast<const float4 *>(rec + lane * 4);
            acc[0] = fmaf(w, o.x, acc[0]); acc[1] = fmaf(w, o.y, acc[1]); acc[2] = fmaf(w, o.z, acc[2]); acc[3] = fmaf(w, o.w, acc[3]);
        } else {
            const float2 o = *reinterpret_cast<const float2 *>(rec + lane * 2);
            acc[0] = fmaf(w, o.x, acc[0]); acc[1] = fmaf(w, o.y, acc[1]);
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int d = lane * V + j;
        if (p.out) store_from_f32(p.out, p.out_dtype, orow * D + d, acc[j]);
        if (p.partials_out) p.partials_out[orow * (D + 4) + d] = acc[j];
    }
    if (lane == 0 && p.partials_out) *reinterpret_cast<float4 *>(p.partials_out + orow * (D + 4) + D) = make_float4(M, L, 0.f, 0.f);
}

template <int D>
__global__ void __launch_bounds__(kFinishThreads, 5) tree_finish_kernel(TreeParams p, FinishArgs f) {
    __shared__ float2 s_stat[256];
    launch_dependents();
    grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int x = blockIdx.x;
    if (x < f.n_join) {
        if (f.workers == 0) {
            // rows of out, eight a block
            const int64_t orow = (int64_t)x * 8 + warp;
            if (orow >= (int64_t)p.B * p.n * p.Hq) return;
            const int b = (int)(orow / ((int64_t)p.n * p.Hq)), i = (int)(orow / p.Hq % p.n);
            if (i >= tree_tokens(p, b)) return;
            const int len = tree_committed(p, b);
            const Pieces pc = chunk_pieces<D>(p, orow, len + tree_drafts(p, b, len));
            if (pc.n > 1) join_row<D>(p, pc, orow, lane);
            return;
        }
        // the pair whose first cut is where CTA w begins; `per` blocks share its rows
        const int per = f.rpt / f.join_rows, w = x / per + 1, r_first = (x % per) * f.join_rows;
        const int64_t T = f.tc.cum[p.B];
        const int wa = (int)(T < f.workers ? T : f.workers);
        if (w >= wa) return;
        const int4 at = f.tc.starts[w];                    // sequence, KV head and q tile, tile
        if (at.z == 0 || owner_of(first_unit(w, T, wa) - at.z, T, wa) != w - 1) return;
        const int len = tree_committed(p, at.x), total = len + tree_drafts(p, at.x, len), R = tree_tokens(p, at.x) * p.G;
        const int q_tiles = (R + f.rpt - 1) / f.rpt, kvh = at.y / q_tiles, qt = at.y - kvh * q_tiles;
        for (int r = r_first + warp; r < r_first + f.join_rows && qt * f.rpt + r < R; r += 8) {
            const int qr = qt * f.rpt + r;
            join_row<D>(p, tc_pieces<D>(p, f, at.x, kvh, qr, total, R), tree_out_row(p, at.x, kvh, qr), lane);
        }
        return;
    }
    x -= f.n_join;
    if (x < f.n_zero) {
        // 32 sequences: the tokens of an empty one attend nothing
        const int b = x * 32 + lane;
        bool empty = false;
        if (b < p.B) {
            const int len = tree_committed(p, b);
            empty = len + tree_drafts(p, b, len) == 0 && tree_tokens(p, b) > 0;
        }
        for (uint32_t todo = __ballot_sync(0xffffffffu, empty); todo; todo &= todo - 1) {
            const int e = x * 32 + __ffs(todo) - 1;
            for (int r = warp; r < tree_tokens(p, e) * p.Hq; r += 8) {
                const int64_t orow = (int64_t)e * p.n * p.Hq + r;
                for (int d = lane * 4; d < D; d += 128) store_row4<D>(p, orow, d, make_float4(0.f, 0.f, 0.f, 0.f));
                if (lane == 0) store_row_stats<D>(p, orow, -INFINITY, 0.f);
            }
        }
        return;
    }
    x -= f.n_zero;
    // score[r] = decay * score[r] + sum over the G heads of exp2(raw - m) / l, four rows a thread.  What a block reads first -- length,
    // statistics, raw scores, old scores -- has addresses that depend on nothing, so that its loads wait for memory together.
    const int blocks = (p.max_len + kScoreRows - 1) / kScoreRows;
    const int pair = x / blocks, b = pair / p.Hkv, kvh = pair - b * p.Hkv;
    const int r0 = (x - pair * blocks) * kScoreRows, row = r0 + threadIdx.x * 4;
    const int64_t h0 = (int64_t)b * p.Hq + kvh * p.G;
    const float *raw = p.raw + h0 * p.raw_ld + row;
    constexpr int kAhead = 4;
    float4 ahead[kAhead];
    const bool in_raw = row < p.max_len;                   // the workspace holds whole rows of scores, whatever the length
#pragma unroll
    for (int g = 0; g < kAhead; g++) ahead[g] = in_raw && g < p.G ? __ldcs(reinterpret_cast<const float4 *>(raw + g * p.raw_ld)) : make_float4(0.f, 0.f, 0.f, 0.f);
    float *s = p.score + ((int64_t)b * p.Hkv + kvh) * p.score_rows + row;
    float old[4];
#pragma unroll
    for (int j = 0; j < 4; j++) old[j] = p.decay != 0.f && row + j < p.max_len ? s[j] : 0.f;
    float2 st = make_float2(0.f, 0.f);
    if ((int)threadIdx.x < min(256, p.G)) st = *reinterpret_cast<const float2 *>(p.stats + 2 * (h0 + threadIdx.x));
    const int len = tree_committed(p, b);
    if (r0 >= len) return;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int g0 = 0; g0 < p.G; g0 += 256) {
        const int n = min(256, p.G - g0);
        if (g0) {
            __syncthreads();
            if ((int)threadIdx.x < n) st = *reinterpret_cast<const float2 *>(p.stats + 2 * (h0 + g0 + threadIdx.x));
        }
        if ((int)threadIdx.x < n) s_stat[threadIdx.x] = st;
        // a negative sum marks a row that was cut: its pieces are joined here
        if (__syncthreads_or((int)threadIdx.x < n && st.y < 0.f)) {
            for (int g = warp; g < n; g += 8) {
                const Pieces pc = f.workers ? tc_pieces<D>(p, f, b, kvh, g0 + g, len, p.G) : chunk_pieces<D>(p, h0 + g0 + g, len);
                float M, L;
                pieces_stats<D>(pc, lane, M, L);
                if (lane == 0) s_stat[g] = make_float2(M * kLog2e, L > 0.f ? 1.f / L : 0.f);
            }
            __syncthreads();
        }
        if (row < len) {
#pragma unroll 4
            for (int g = 0; g < n; g++) {
                const float4 v = g0 == 0 && g < kAhead ? ahead[g & (kAhead - 1)] : *reinterpret_cast<const float4 *>(raw + (g0 + g) * p.raw_ld);
                const float2 t = s_stat[g];
                sum[0] += ex2(v.x - t.x) * t.y; sum[1] += ex2(v.y - t.x) * t.y;
                sum[2] += ex2(v.z - t.x) * t.y; sum[3] += ex2(v.w - t.x) * t.y;
            }
        }
    }
    // the four rows lie in one page (page_rows >= 32); without a page they have no raw score
    if (row >= len || (p.rows.table && cache_row(p.rows, b, kvh, row) < 0)) return;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (row + j < len) s[j] = (p.decay == 0.f ? 0.f : p.decay * old[j]) + sum[j];
}

template <int D> inline cudaError_t launch_finish(const TreeParams &p, FinishArgs &f, cudaStream_t st) {
    if (f.workers) {
        f.join_rows = f.rpt < 8 ? f.rpt : 8;
        f.n_join = (f.workers - 1) * (f.rpt / f.join_rows);
        f.n_zero = (p.B + 31) / 32;
    } else {
        f.n_join = p.max_chunks > 1 ? (int)(((int64_t)p.B * p.n * p.Hq + 7) / 8) : 0;
        f.n_zero = 0;
    }
    f.n_score = p.score ? p.B * p.Hkv * ((p.max_len + kScoreRows - 1) / kScoreRows) : 0;
    const int64_t blocks = (int64_t)f.n_join + f.n_zero + (p.score ? (int64_t)p.B * p.Hkv * ((p.max_len + kScoreRows - 1) / kScoreRows) : 0);
    if (blocks == 0) return cudaSuccess;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return launch_dependent(tree_finish_kernel<D>, dim3((unsigned)blocks), kFinishThreads, 0, st, p, f);
}

}  // namespace treetc
}  // namespace nimllm
