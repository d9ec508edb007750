// tree_finish.cuh -- the one launch behind the attention kernels of tree and scored decode: pieces of cut rows are joined, rows
// without anything to attend become zeros, and the scores of a scored decode are brought up to date.
//
// The three jobs are independent (a score block joins the maxima and sums that it needs by itself), so they share a launch: block
// numbers first count the joins, then groups of 32 sequences, then the score blocks.
#pragma once
#include "tree_tc.cuh"

namespace nimllm {
namespace treetc {

constexpr int kFinishThreads = 256, kScoreRows = 4096;
constexpr int kMaxPieces = 180;        // 32 rows of them in 48 KB

// The pieces of a query row.  Tensor-core kernels: records of consecutive CTAs (tree_tc.cuh); CUDA-core kernel: one record per chunk of
// rows.  n = 1: the kernel stored the row itself; n = 0: there was nothing to attend.
// Column d of row r is at rec(i) + r * row + d / 4 * col + d % 4, its maximum and sum where column D would be.
struct Pieces {
    int n;
    const float *first, *second;       // record of piece 0, of piece 1; the others follow at `step`
    int64_t step;
    int row, col;
    __device__ const float *rec(int x) const { return x == 0 ? first : second + (x - 1) * step; }
};
struct FinishArgs {
    TcArgs tc;
    int rpt, tile, workers;            // tensor-core kernels; workers = 0: the chunks of the CUDA-core kernel
    bool by_col;                       // the records are [D / 4 + 1][row][4], as a thread per row stores them best
    int n_join, n_zero;                // blocks of the first two kinds
};

template <int D> __device__ __forceinline__ Pieces tc_pieces(const TreeParams &p, const FinishArgs &f, int b, int kvh, int qr, int total, int R) {
    constexpr int W = D + 4;
    Pieces x{0, nullptr, nullptr, 0, f.by_col ? 4 : W, f.by_col ? 4 * f.tc.rec_rows : 4};
    if (total == 0) return x;
    const int64_t T = f.tc.cum[p.B];
    const int wa = (int)(T < f.workers ? T : f.workers);
    const int q_tiles = (R + f.rpt - 1) / f.rpt, tiles = (total + f.tile - 1) / f.tile;
    const int qt = qr / f.rpt, r = qr - qt * f.rpt;
    const int64_t s = f.tc.cum[b] + ((int64_t)kvh * q_tiles + qt) * tiles;
    const int w0 = owner_of(s, T, wa);
    x.n = owner_of(s + tiles - 1, T, wa) - w0 + 1;
    x.step = (int64_t)2 * f.tc.rec_rows * W;
    x.first = p.recs + ((int64_t)w0 * 2 + (first_unit(w0, T, wa) < s ? 1 : 0)) * f.tc.rec_rows * W + r * x.row;
    x.second = p.recs + ((int64_t)(w0 + 1) * 2) * f.tc.rec_rows * W + r * x.row;
    return x;
}
template <int D> __device__ __forceinline__ Pieces chunk_pieces(const TreeParams &p, int64_t orow, int total) {
    constexpr int W = D + 4;
    Pieces x;
    x.row = W; x.col = 4;
    x.n = total <= p.chunk_rows ? 1 : (total + p.chunk_rows - 1) / p.chunk_rows;      // an empty row is stored by chunk 0
    x.step = (int64_t)p.B * p.n * p.Hq * W;
    x.first = p.recs + orow * W;
    x.second = x.first + x.step;
    return x;
}

// maximum (natural units) and, relative to it, the sum of a row's pieces, in every lane.  A piece is empty when its sum is zero; one whose
// sum is NaN counts, so that the row has no number either.
template <int D> __device__ __forceinline__ void pieces_stats(const Pieces &x, int lane, float &M, float &L) {
    M = -INFINITY;
    for (int i = lane; i < x.n; i += 32) {
        const float2 ml = *reinterpret_cast<const float2 *>(x.rec(i) + D / 4 * x.col);
        if (ml.y != 0.f) M = fmaxf(M, ml.x);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    const float safe = M == -INFINITY ? 0.f : M;
    L = 0.f;
    for (int i = lane; i < x.n; i += 32) {
        const float2 ml = *reinterpret_cast<const float2 *>(x.rec(i) + D / 4 * x.col);
        if (ml.y != 0.f) L += ml.y * ex2((ml.x - safe) * kLog2e);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
}

// What the scores of a row are worked out from, exp2(raw - m) / l.  l - l: without a finite sum there is no reference either, so that they are
// all NaN; without any weight the reference is above them all.
__device__ __forceinline__ float2 score_stats(float m, float l) { return make_float2(l != 0.f ? m + (l - l) : INFINITY, inverse_sum(l)); }

// One block joins up to 32 rows that are cut alike.  `out_row(r)` is row r's row of out.
// First every (row, piece) statistic is fetched at once and turned into the piece's weight, then every 16 bytes of the rows is a sum
// over the pieces whose loads wait for nothing else.
constexpr int kJoinRows = 32;
template <int D, typename OutRow>
__device__ __forceinline__ void join_rows(const TreeParams &p, const Pieces &x, int rows, OutRow out_row, float2 *s_ml) {
    constexpr int W = D + 4, kLanes = kFinishThreads / kJoinRows;
    for (int e = threadIdx.x; e < rows * x.n; e += kFinishThreads) {
        const int i = e / rows, r = e - i * rows;
        s_ml[r * x.n + i] = *reinterpret_cast<const float2 *>(x.rec(i) + r * x.row + D / 4 * x.col);
    }
    __syncthreads();
    const int r = threadIdx.x / kLanes, sub = threadIdx.x % kLanes;
    if (r < rows) {                                        // eight threads of one warp per row
        float2 *ml = s_ml + r * x.n;
        const unsigned mask = 0xffu << (threadIdx.x & 24);
        float M = -INFINITY, L = 0.f;
        for (int i = sub; i < x.n; i += kLanes)
            if (ml[i].y != 0.f) M = fmaxf(M, ml[i].x);
#pragma unroll
        for (int off = kLanes / 2; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(mask, M, off));
        const float safe = M == -INFINITY ? 0.f : M;
        for (int i = sub; i < x.n; i += kLanes) {
            const float w = ml[i].y != 0.f ? ml[i].y * ex2((ml[i].x - safe) * kLog2e) : 0.f;
            ml[i].x = w;
            L += w;
        }
#pragma unroll
        for (int off = kLanes / 2; off > 0; off >>= 1) L += __shfl_xor_sync(mask, L, off);
        const float inv = inverse_sum(L);
        for (int i = sub; i < x.n; i += kLanes) ml[i].x *= inv;
        if (sub == 0 && p.partials_out) *reinterpret_cast<float4 *>(p.partials_out + out_row(r) * W + D) = make_float4(M, L, 0.f, 0.f);
    }
    __syncthreads();
    // a warp has four rows by eight 16-byte columns: whole sectors of records in either layout, and of out
    for (int e = threadIdx.x; e < (rows + 3) / 4 * D; e += kFinishThreads) {
        const int rr = e / D * 4 + (e & 3), d = e % D / 4 * 4;
        if (rr >= rows) continue;
        const float2 *w = s_ml + rr * x.n;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < x.n; i++) {
            const float4 o = *reinterpret_cast<const float4 *>(x.rec(i) + rr * x.row + d / 4 * x.col);
            const float f = w[i].x;
            acc.x = fmaf(f, o.x, acc.x); acc.y = fmaf(f, o.y, acc.y); acc.z = fmaf(f, o.z, acc.z); acc.w = fmaf(f, o.w, acc.w);
        }
        store_row4<D>(p, out_row(rr), d, acc);
    }
}

template <int D>
__global__ void __launch_bounds__(kFinishThreads, 4) tree_finish_kernel(TreeParams p, FinishArgs f) {
    extern __shared__ float2 s_dyn[];                      // join: kJoinRows x pieces; score: the G heads
    float2 *s_stat = s_dyn;
    launch_dependents();
    grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int x = blockIdx.x;
    if (x < f.n_join) {
        if (f.workers == 0) {
            // 32 rows of a sequence's results
            const int per = (p.n * p.Hq + kJoinRows - 1) / kJoinRows, b = x / per, first = (x - b * per) * kJoinRows;
            const int rows = min(kJoinRows, tree_tokens(p, b) * p.Hq - first);
            const int len = tree_committed(p, b);
            const int64_t orow = (int64_t)b * p.n * p.Hq + first;
            const Pieces pc = chunk_pieces<D>(p, orow, len + tree_drafts(p, b, len));
            if (rows > 0 && pc.n > 1) join_rows<D>(p, pc, rows, [&](int r) { return orow + r; }, s_dyn);
            return;
        }
        // the pair whose first cut is where CTA w begins; `per` blocks share its rows
        const int per = f.rpt > kJoinRows ? f.rpt / kJoinRows : 1, w = x / per + 1, first = (x % per) * kJoinRows;
        const int64_t T = f.tc.cum[p.B];
        const int4 at = f.tc.starts[w];                    // sequence, KV head and q tile, tile (not written past the last worker)
        const int wa = (int)(T < f.workers ? T : f.workers);
        if (w >= wa || at.z == 0 || owner_of(first_unit(w, T, wa) - at.z, T, wa) != w - 1) return;
        const int len = tree_committed(p, at.x), total = len + tree_drafts(p, at.x, len), R = tree_tokens(p, at.x) * p.G;
        const int q_tiles = (R + f.rpt - 1) / f.rpt, kvh = at.y / q_tiles, q0 = (at.y - kvh * q_tiles) * f.rpt + first;
        const int rows = min(min(kJoinRows, f.rpt), R - q0);
        if (rows > 0)
            join_rows<D>(p, tc_pieces<D>(p, f, at.x, kvh, q0, total, R), rows, [&](int r) { return tree_out_row(p, at.x, kvh, q0 + r); }, s_dyn);
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
    // score[r] = decay * score[r] + sum over the G heads of exp2(raw - m) / l: a block has up to 4096 rows of a pair, four a thread at a
    // time.  What it reads first -- length, statistics, raw scores, old scores -- has addresses that depend on nothing, so that its
    // loads wait for memory together, and the next rows' are under way while these are worked on.
    const int blocks = (p.max_len + kScoreRows - 1) / kScoreRows;
    const int pair = x / blocks, b = pair / p.Hkv, kvh = pair - b * p.Hkv;
    const int r0 = (x - pair * blocks) * kScoreRows;
    const int64_t h0 = (int64_t)b * p.Hq + kvh * p.G;
    const float *raw = p.raw + h0 * p.raw_ld;
    float *score = p.score + (int64_t)pair * p.score_rows;
    const bool vec = !((uintptr_t)score & 15);
    constexpr int kAhead = 4;                              // heads whose raw scores are fetched ahead
    struct Ahead { float4 raw[kAhead], old; };
    auto fetch = [&](Ahead &a, int row) {                  // the workspace holds whole rows of raw scores, whatever the length
#pragma unroll
        for (int g = 0; g < kAhead; g++) a.raw[g] = row < p.max_len && g < p.G ? __ldcs(reinterpret_cast<const float4 *>(raw + g * p.raw_ld + row)) : make_float4(0.f, 0.f, 0.f, 0.f);
        a.old = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p.decay != 0.f) {
            if (vec && row + 4 <= p.max_len) {
                a.old = *reinterpret_cast<const float4 *>(score + row);
            } else {
                if (row < p.max_len) a.old.x = score[row];
                if (row + 1 < p.max_len) a.old.y = score[row + 1];
                if (row + 2 < p.max_len) a.old.z = score[row + 2];
                if (row + 3 < p.max_len) a.old.w = score[row + 3];
            }
        }
    };
    int row = r0 + threadIdx.x * 4;
    Ahead now;
    fetch(now, row);
    for (int g = threadIdx.x; g < p.G; g += kFinishThreads) {
        const float2 t = *reinterpret_cast<const float2 *>(p.stats + 2 * (h0 + g));
        s_stat[g] = t.y < 0.f ? t : score_stats(t.x, t.y);
    }
    const int len = tree_committed(p, b);
    if (r0 >= len) return;
    __syncthreads();
    // A negative sum marks a row that was cut: its pieces are joined here.  Every head is asked by itself: heads in different query tiles
    // (128 or 256 of them) are cut apart from one another.  A head's entry is read and written by one warp, once all warps have looked.
    bool cut = false;
    for (int g = lane; g < p.G; g += 32) cut |= s_stat[g].y < 0.f;
    if (__any_sync(0xffffffffu, cut)) {
        __syncthreads();
        for (int g = warp; g < p.G; g += kFinishThreads / 32) {
            const bool cut_g = s_stat[g].y < 0.f;
            __syncwarp();
            if (!cut_g) continue;
            const Pieces pc = f.workers ? tc_pieces<D>(p, f, b, kvh, g, len, p.G) : chunk_pieces<D>(p, h0 + g, len);
            float M, L;
            pieces_stats<D>(pc, lane, M, L);
            if (lane == 0) s_stat[g] = score_stats(M * kLog2e, L);
        }
        __syncthreads();
    }
    for (; row < min(len, r0 + kScoreRows); row += 4 * kFinishThreads) {
        Ahead next;
        if (row + 4 * kFinishThreads < min(len, r0 + kScoreRows)) fetch(next, row + 4 * kFinishThreads);
        float sum[4] = {p.decay * now.old.x, p.decay * now.old.y, p.decay * now.old.z, p.decay * now.old.w};
        auto head = [&](const float4 &v, int g) {
            const float2 t = s_stat[g];
            sum[0] += ex2(v.x - t.x) * t.y; sum[1] += ex2(v.y - t.x) * t.y;
            sum[2] += ex2(v.z - t.x) * t.y; sum[3] += ex2(v.w - t.x) * t.y;
        };
#pragma unroll
        for (int g = 0; g < kAhead; g++)
            if (g < p.G) head(now.raw[g], g);
#pragma unroll 4
        for (int g = kAhead; g < p.G; g++) head(*reinterpret_cast<const float4 *>(raw + g * p.raw_ld + row), g);
        // the four rows lie in one page (page_rows >= 32); without a page they have no raw score
        if (!p.rows.table || cache_row(p.rows, b, kvh, row) >= 0) {
            if (vec && row + 4 <= len) {
                *reinterpret_cast<float4 *>(score + row) = make_float4(sum[0], sum[1], sum[2], sum[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (row + j < len) score[row + j] = sum[j];
            }
        }
        now = next;
    }
}

template <int D> inline cudaError_t launch_finish(const TreeParams &p, FinishArgs &f, cudaStream_t st) {
    size_t pieces;
    if (f.workers) {
        f.n_join = (f.workers - 1) * (f.rpt > kJoinRows ? f.rpt / kJoinRows : 1);
        f.n_zero = (p.B + 31) / 32;
        pieces = f.workers;
    } else {
        f.n_join = p.max_chunks > 1 ? p.B * ((p.n * p.Hq + kJoinRows - 1) / kJoinRows) : 0;
        f.n_zero = 0;
        pieces = p.max_chunks;
    }
    const int64_t blocks = (int64_t)f.n_join + f.n_zero + (p.score ? (int64_t)p.B * p.Hkv * ((p.max_len + kScoreRows - 1) / kScoreRows) : 0);
    if (blocks == 0) return cudaSuccess;
    if (blocks > 0x7fffffff || pieces > kMaxPieces) return cudaErrorInvalidConfiguration;
    size_t smem = f.n_join ? kJoinRows * pieces * sizeof(float2) : 0;
    if (p.score && smem < p.G * sizeof(float2)) smem = p.G * sizeof(float2);
    return launch_dependent(tree_finish_kernel<D>, dim3((unsigned)blocks), kFinishThreads, smem, st, p, f);
}

}  // namespace treetc
}  // namespace nimllm
