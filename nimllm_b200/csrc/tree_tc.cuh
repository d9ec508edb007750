// tree_tc.cuh -- what the two tensor-core kernels of tree and scored decode share: the work list and the row stores.
//
// All tiles of a batch are one list ordered by (sequence, KV head, query tile, row), cut into equal spans, one per CTA (one CTA
// per SM).  A CTA cuts at most two (sequence, KV head, query tile) triples; their pieces go to its two record slots of `recs` and
// tree_finish_kernel (tree_finish.cuh) finds them by the same arithmetic.
#pragma once
#include "tcgen05.cuh"
#include "tree_decode.cuh"

namespace nimllm {
namespace treetc {

struct TcArgs {
    int64_t *cum;              // [B + 1] units before each sequence, written by CTA 0 for the finishing launch
    int4 *starts;              // per CTA: sequence, (KV head, q tile), tile of its first unit
    int q_terms, p_terms, stages;
    int rec_rows;              // query rows of a record slot
};

__host__ __device__ inline int64_t first_unit(int w, int64_t T, int wa) { return (int64_t)w * T / wa; }
__host__ __device__ inline int owner_of(int64_t u, int64_t T, int wa) { return (int)(((u + 1) * wa - 1) / T); }

// what a sequence contributes: q tiles of RPT rows per KV head and tiles of TILE cached rows per q tile
struct SeqWork {
    int len, drafts, total, R, q_tiles, tiles;
};
template <int RPT, int TILE> __device__ __forceinline__ SeqWork seq_work(const TreeParams &p, int b) {
    SeqWork s;
    s.len = tree_committed(p, b);
    s.drafts = tree_drafts(p, b, s.len);
    s.total = s.len + s.drafts;
    s.R = tree_tokens(p, b) * p.G;
    s.q_tiles = (s.R + RPT - 1) / RPT;
    s.tiles = s.R ? (s.total + TILE - 1) / TILE : 0;
    return s;
}
template <int RPT, int TILE> __device__ __forceinline__ int64_t seq_units(const TreeParams &p, int b) {
    const SeqWork s = seq_work<RPT, TILE>(p, b);
    return (int64_t)p.Hkv * s.q_tiles * s.tiles;
}

// A CTA's span, segment by segment: tiles [i0, i1) of q tile qt of KV head kvh of sequence b
struct Segment {
    int b, kvh, qt, i0, i1;
    SeqWork w;
    bool whole;
    int slot;
};
template <int RPT, int TILE> struct SpanWalk {
    const TreeParams &p;
    int b, h, i0, remaining;
    bool first;
    SeqWork w;
    __device__ SpanWalk(const TreeParams &p_, int b_, int h_, int i_, int n) : p(p_), b(b_), h(h_), i0(i_), remaining(n), first(true) {
        if (n > 0) w = seq_work<RPT, TILE>(p, b);
    }
    __device__ bool next(Segment &s) {
        if (remaining <= 0) return false;
        while (w.tiles == 0 || h >= p.Hkv * w.q_tiles) {
            b++; h = 0; i0 = 0;
            w = seq_work<RPT, TILE>(p, b);
        }
        s.b = b; s.kvh = h / w.q_tiles; s.qt = h - s.kvh * w.q_tiles; s.w = w;
        s.i0 = i0;
        s.i1 = min(w.tiles, i0 + remaining);
        s.whole = i0 == 0 && s.i1 == w.tiles;
        s.slot = first ? 0 : 1;
        remaining -= s.i1 - s.i0;
        first = false;
        i0 = s.i1;
        if (i0 == w.tiles) { i0 = 0; h++; }
        return true;
    }
};

// The span of this CTA, found by all of its threads: a prefix of the sequences' units over the block.  Contains barriers; returns the
// number of units (0: nothing to do) and leaves the first one in `start`.
struct SpanStart {
    int b, h, i;
    int64_t warp_sum[32];
};
template <int RPT, int TILE, int THREADS>
__device__ __forceinline__ int span_begin(const TreeParams &p, const TcArgs &a, SpanStart &start) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = (p.B + THREADS - 1) / THREADS;
    const int b_beg = min(p.B, (int)threadIdx.x * per), b_end = min(p.B, b_beg + per);
    int64_t sum = 0;
    for (int b = b_beg; b < b_end; b++) sum += seq_units<RPT, TILE>(p, b);
    int64_t incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += x;
    }
    if (lane == 31) start.warp_sum[warp] = incl;
    __syncthreads();
    int64_t excl = incl - sum, T = 0;
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) excl += start.warp_sum[w];
        T += start.warp_sum[w];
    }
    if (blockIdx.x == 0) {
        int64_t c = excl;
        for (int b = b_beg; b < b_end; b++) { a.cum[b] = c; c += seq_units<RPT, TILE>(p, b); }
        if (threadIdx.x == 0) a.cum[p.B] = T;
    }
    const int wa = (int)(T < (int64_t)gridDim.x ? T : (int64_t)gridDim.x);
    if ((int)blockIdx.x >= wa) return 0;
    const int64_t u0 = first_unit(blockIdx.x, T, wa);
    if (u0 >= excl && u0 < excl + sum) {
        int64_t c = excl;
        for (int b = b_beg; b < b_end; b++) {
            const SeqWork w = seq_work<RPT, TILE>(p, b);
            const int64_t n = (int64_t)p.Hkv * w.q_tiles * w.tiles;
            if (u0 < c + n) {
                start.b = b;
                start.h = (int)((u0 - c) / w.tiles);
                start.i = (int)((u0 - c) % w.tiles);
                break;
            }
            c += n;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) a.starts[blockIdx.x] = make_int4(start.b, start.h, start.i, 0);
    return (int)(first_unit(blockIdx.x + 1, T, wa) - u0);
}

// 16 bytes from global to shared memory, or zeros (bytes = 0: the source is not read)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// the same for rows that nobody reads again in this launch: they leave L2 first, so that records, scores and code stay
__device__ __forceinline__ uint64_t evict_first_policy() {
    uint64_t pol;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
    return pol;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(policy) : "memory");
}
// arrives on the barrier when this thread's copies so far have landed.  The reader of the data is the tensor core: the warp that
// issues the MMAs orders the copies before them with a proxy fence behind its wait.
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int D>
__device__ __forceinline__ void store_row4(const TreeParams &p, int64_t orow, int d, float4 x) {
    if (p.out) {
        if (p.out_dtype == NIMLLM_F32) *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.out) + orow * D + d) = x;
        else *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(p.out) + orow * D + d) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
    }
    if (p.partials_out) *reinterpret_cast<float4 *>(p.partials_out + orow * (D + 4) + d) = x;
}
// eight columns: 16 bytes of a bf16 row
template <int D>
__device__ __forceinline__ void store_row8(const TreeParams &p, int64_t orow, int d, const float *x) {
    if (p.out && p.out_dtype == NIMLLM_BF16 && !p.partials_out) {
        *reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(p.out) + orow * D + d) =
            make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
    } else {
        store_row4<D>(p, orow, d, make_float4(x[0], x[1], x[2], x[3]));
        store_row4<D>(p, orow, d + 4, make_float4(x[4], x[5], x[6], x[7]));
    }
}
template <int D>
__device__ __forceinline__ void store_row_stats(const TreeParams &p, int64_t orow, float m, float l) {
    if (p.partials_out) *reinterpret_cast<float4 *>(p.partials_out + orow * (D + 4) + D) = make_float4(m * kLn2, l, 0.f, 0.f);
    if (p.stats) *reinterpret_cast<float2 *>(p.stats + 2 * orow) = make_float2(m, l);
}

// a row that was cut has no statistics yet: the score blocks join its pieces themselves
__device__ __forceinline__ void mark_cut(const TreeParams &p, int64_t orow) {
    if (p.stats) p.stats[2 * orow + 1] = -1.f;
}

// tree_narrow_tc.cu: few query rows
bool tree_narrow_takes(int R, int q_terms, int p_terms, int head_dim);
cudaError_t launch_tree_narrow(const TreeParams &p, TcArgs &a, int head_dim, cudaStream_t st);
int tree_narrow_status(int reset, int *status_out);
constexpr int kNarrowRows = 32, kNarrowTile = 128;

}  // namespace treetc
}  // namespace nimllm
