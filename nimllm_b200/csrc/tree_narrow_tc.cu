// tree_narrow_tc.cu -- tree and scored decode over bf16 caches with at most 32 query rows per KV head, on the tensor cores.
//
// Few query rows would leave most of an M = 128 tile of queries empty, so the products are turned round: cached rows are M.
//     S^T = K Q^T     (128 cached rows x N, one thread per cached row)
//     O^T += V^T P^T  (head_dim x N, A = V as it lies in the cache, B = P^T written to shared memory by the softmax)
// and N is the query rows, 16 or 32, times the bf16 terms of an fp32 q (S) or of P (O): the terms are further columns of the
// same MMA, so that 32-bit precision costs little tensor time.  An fp32 q and the P of fp32 results have three terms (2^-26 left), the P
// of bf16 results two (2^-17 left).
//
// Measured (graph replay): scored decode of 32 sequences of 2 - 8 K rows in pages, 32 q / 8 kv heads of 128, bf16: 122 us, 104 at the
// measured peak of HBM (5.6 TB/s).  256 sequences of 512 - 4096 rows, 5 tokens, 9 q / 3 kv heads of 64, fp32 q and results: 118 us, of which
// the rows' bytes are 70: tiles of head size 64 have half the bytes and are bound by what a tile costs, whatever its segment.  A CTA has
// about 94 tiles in five segments, 1.15 us or 2200 cycles each (64 sequences with segments of 24 tiles: 1.19 us): a softmax group
// writes its next P only behind its own P V, and 128 threads vote once a tile.  The tensor pipe is active for 12 % of that launch, DRAM 43 %.
//
//   warps 0-3, 4-7   two softmax groups, taking the tiles of 128 rows in turn: the waits of one hide behind the other
//   warps 8-11       K rows (8, 9) and V rows (10, 11) into a ring of slots with cp.async, swizzled, exact to the row
//                    (tree_wide_tc.cu says why no TMA)
//   warp 12          walks the CTA's span and hands its segments to the others; Q of the segments to come (two buffers), and which
//                    query rows see each of their drafts
//   warps 13, 14     issue K Q^T and V^T P^T, each in order and waiting for its own operands alone
//   warp 15          joins the two groups' sums at the end of a segment and stores them, beside the next one's tiles
//
// Softmax across threads: with one thread per cached row a query row's maximum lies across 128 threads.  It is not needed: a
// reference per query row that some score has and none passes by more than 2^32 serves as well, because P is rounded relative to
// its own size and fp32 has the range.  The first row of a segment gives it; later tiles only vote (one barrier) whether a score
// has grown past it.  Sums of P stay in the thread until the segment ends.
//
// O^T is accumulated in TMEM over four tiles of a group at most (32 steps of the tensor core's adder), then added to registers.
#include "tree_tc.cuh"

namespace nimllm {
namespace treetc {

namespace {

using namespace tc;

__device__ int g_narrow_status = 0;    // sticky, nimllm_attn_decode_tree_status

constexpr int kTile = kNarrowTile;
constexpr int kMaxSlots = 12;
constexpr int kThreads = 512;
constexpr int kWindow = 4;             // tiles of a group between two readings of O^T
constexpr float kGrow = 32.f;          // log2 units by which a score may pass the reference
constexpr float kUnset = -1e30f;       // reference of a query row that has attended nothing yet: any score passes it
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColO = 192;    // per group: S^T 96 columns, O^T 64 columns
constexpr int kKvBox = kTile * 128;    // bytes of a 64-column box of K or V rows
constexpr int kPBytes = kTile * 128;   // P^T of a group: 128 rows x 64 columns
constexpr int kSegs = 8;

struct SegEntry {
    int b, kvh, i0, i1, len, total, R, flags;      // b < 0: the end; flags: 1 whole, 2 the second record slot
};

struct Bars {
    uint64_t full[kMaxSlots], empty[kMaxSlots];
    uint64_t seg_full[kSegs], seg_empty[kSegs];
    uint64_t q_full[2], q_empty[2], q_asked;
    uint64_t s_full[2], s_free[2], p_ready[2], pv_done[2];
    uint64_t x_ready, x_free, drain[2];
    uint32_t tmem_base;
    volatile int abort_flag;
    SpanStart start;
    SegEntry segs[kSegs];
    int valid[8];                      // by tile: bit h, the page of rows 32h .. exists
    uint32_t sees[8][32];              // by segment: the query rows that attend draft j, one bit each (8: a group reads a
                                       // segment's until it takes scores of the next but one, up to five segments on)
    alignas(16) float ref[2][32];      // the groups' references
    float xref[2][32];                 // and what they were at the end of a segment
    float wmax[2][4][32], wsum[2][4][32];
    float2 join[32];                   // what the two groups' O count, and the row of out
    int64_t orow[32];
};

// true in all 128 threads of the group when it is in any; orders the group's shared memory like a barrier
__device__ __forceinline__ bool group_any(int group, bool x) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(r) : "r"((uint32_t)x), "r"(group + 1) : "memory");
    return r != 0;
}

template <int N> __device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t *r) {
    if constexpr (N == 32) tmem_ld32(at, r);
    else if constexpr (N == 16) tmem_ld16(at, r);
    else if constexpr (N == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(at) : "memory");
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <int N> __device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t *r) {
    if constexpr (N == 32) tmem_st32(at, r);
    else if constexpr (N == 16) tmem_st16(at, r);
    else if constexpr (N == 8) tmem_st8(at, r);
    else asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// x = (ADD: x +) the sum of the TERMS' columns of an accumulator, all loads in flight together where registers allow
template <int N, int RP, int TERMS, bool ADD> __device__ __forceinline__ void tmem_terms(uint32_t at, float *x) {
    constexpr int kBatch = N <= 16 ? TERMS : 1;
#pragma unroll
    for (int t0 = 0; t0 < TERMS; t0 += kBatch) {
        uint32_t y[kBatch][N];
#pragma unroll
        for (int t = 0; t < kBatch; t++) tmem_ld<N>(at + (t0 + t) * RP, y[t]);
        tc_wait_ld();
#pragma unroll
        for (int r = 0; r < N; r++)
#pragma unroll
            for (int t = 0; t < kBatch; t++) x[r] = ADD || t0 + t > 0 ? x[r] + __uint_as_float(y[t][r]) : __uint_as_float(y[t][r]);
    }
}

// Column sums over the warp: lane r (and its copies at r + N, ...) gets the sum of v[r].  Halving exchange: N - 1 shuffles for the
// first log2(N) steps, one for each of the others.
template <int N> __device__ __forceinline__ float column_sum(float *v, int lane) {
#pragma unroll
    for (int h = N / 2; h > 0; h >>= 1) {
        const bool up = lane & h;
#pragma unroll
        for (int r = 0; r < h; r++) {
            const float give = up ? v[r] : v[r + h], keep = up ? v[r + h] : v[r];
            v[r] = keep + __shfl_xor_sync(0xffffffffu, give, h);
        }
    }
    float s = v[0];
#pragma unroll
    for (int off = 16; off >= N; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    return s;
}

// segment s of the queue, in every lane; false at the end and when a wait gave up (ok says which)
__device__ __forceinline__ bool next_segment(Bars &sb, int s, SegEntry &e, bool &ok, int lane) {
    ok = __all_sync(0xffffffffu, mbar_wait(&sb.seg_full[s % kSegs], (s / kSegs) & 1, &sb.abort_flag));
    if (!ok) return false;
    e = sb.segs[s % kSegs];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sb.seg_empty[s % kSegs]);
    return e.b >= 0;
}

// RC: query rows that are computed (the rest of the 16 or 32 columns stays zero); NQ, NP: terms of q and of P
template <int D, int RC, int NQ, int NP>
__global__ void __launch_bounds__(kThreads, 1) tree_narrow_kernel(TreeParams p, TcArgs a) {
    constexpr int RP = RC <= 16 ? 16 : 32;     // columns of a term
    constexpr int kSlot = kTile * D * 2;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Bars sb;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    constexpr int n_s = RP * NQ, n_o = RP * NP;
    constexpr int q_box = n_s * 128, q_bytes = n_s * D * 2;
    uint8_t *s_kv = smem, *s_p = s_kv + a.stages * kSlot, *s_q = s_p + 2 * kPBytes;
    float *s_x = reinterpret_cast<float *>(s_q + 2 * q_bytes);       // the groups' O at the end of a segment: [2][RC][D]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    launch_dependents();
    grid_dependency_wait();
    const int n_units = span_begin<kNarrowRows, kTile, kThreads>(p, a, sb.start);
    if (n_units == 0) return;
    if (threadIdx.x == 0) {
        sb.abort_flag = 0;
        for (int s = 0; s < a.stages; s++) { mbar_init(&sb.full[s], 65); mbar_init(&sb.empty[s], 1); }
        for (int s = 0; s < kSegs; s++) { mbar_init(&sb.seg_full[s], 1); mbar_init(&sb.seg_empty[s], 15); }
        for (int g = 0; g < 2; g++) {
            mbar_init(&sb.q_full[g], 32); mbar_init(&sb.q_empty[g], 1);
            mbar_init(&sb.s_full[g], 1); mbar_init(&sb.s_free[g], 4);
            mbar_init(&sb.p_ready[g], 4); mbar_init(&sb.pv_done[g], 1);
        }
        mbar_init(&sb.q_asked, 32); mbar_init(&sb.x_ready, 8); mbar_init(&sb.x_free, 1); mbar_init(&sb.drain[0], 1); mbar_init(&sb.drain[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // columns that no query row fills stay zero, in Q and in P
    for (int x = threadIdx.x; x < (2 * kPBytes + 2 * q_bytes) / 16; x += kThreads) reinterpret_cast<uint4 *>(s_p)[x] = make_uint4(0, 0, 0, 0);
    fence_async();
    if (warp == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sb.tmem_base)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sb.tmem_base;
    volatile int *abort_flag = &sb.abort_flag;
    SegEntry sg;
    bool ok = true;

    // 128 registers a thread at launch; the eight warps that only issue give (128 - 72), the softmax warps take (184 - 128)
    if (warp >= 8 && warp < 12) {
        // ---------------------------------------------------------------- slot 2k of the stream is K_k, slot 2k + 1 is V_k
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        constexpr int kChunks = D / 8, kStep = 64 / kChunks;
        const int which = (warp - 8) >> 1, t = (int)threadIdx.x - 256 - which * 64, c = t % kChunks, r_in = t / kChunks;
        const uint32_t kv = smem_u32(s_kv);
        const __nv_bfloat16 *src = reinterpret_cast<const __nv_bfloat16 *>(which ? p.v : p.k) + c * 8;
        const uint64_t once = evict_first_policy();
        int k = 0, slot = which, phase = 1;
        for (int seg = 0; next_segment(sb, seg, sg, ok, lane); seg++) {
            // the loads of the first Q go out before a ring full of rows queues up in front of them
            if (seg == 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(&sb.q_asked, 0, abort_flag)))) break;
            for (int i = sg.i0; i < sg.i1; i++, k++) {
                const int t0 = i * kTile, n = min(kTile, sg.total - t0);
                int64_t h[4];
                int valid = 0;
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    h[y] = y * 32 < n ? cache_row(p.rows, sg.b, sg.kvh, t0 + y * 32) : 0;
                    valid |= (h[y] >= 0 ? 1 : 0) << y;
                }
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.empty[slot], phase, abort_flag)))) break;
                if (t == 0) {                              // the 65th arrival publishes the tile's word
                    if (which == 0) sb.valid[k & 7] = valid;
                    mbar_arrive(&sb.full[slot]);
                }
                const uint32_t dst = kv + slot * kSlot + (c >> 3) * kKvBox;
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const int r_end = h[y] >= 0 ? n - y * 32 : 0;
                    const __nv_bfloat16 *g = src + (h[y] >= 0 ? h[y] : 0) + r_in * D;
#pragma unroll
                    for (int r0 = 0; r0 < 32; r0 += kStep) {
                        const int rr = y * 32 + r0 + r_in;
                        const bool have = r0 + r_in < r_end;
                        cp_async16(dst + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), have ? g + r0 * D : src, have ? 16 : 0, once);
                    }
                }
                cp_async_arrive(&sb.full[slot]);
                slot += 2;
                if (slot >= a.stages) { slot = which; phase ^= 1; }
            }
            if (!ok) break;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 12) {
        // ---------------------------------------------------------------- Q: row r of term t is row t * RP + r of the B operand
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        SpanWalk<kNarrowRows, kTile> walk(p, sb.start.b, sb.start.h, sb.start.i, n_units);
        for (int seg = 0;; seg++) {
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.seg_empty[seg % kSegs], ((seg / kSegs) & 1) ^ 1, abort_flag)))) break;
            Segment s;
            const bool more = walk.next(s);
            sg = more ? SegEntry{s.b, s.kvh, s.i0, s.i1, s.w.len, s.w.total, s.w.R, (s.whole ? 1 : 0) | (s.slot ? 2 : 0)} : SegEntry{-1, 0, 0, 0, 0, 0, 0, 0};
            if (lane == 0) {
                sb.segs[seg % kSegs] = sg;
                mbar_arrive(&sb.seg_full[seg % kSegs]);
            }
            if (!more) break;
            const int buf = seg & 1;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.q_empty[buf], ((seg >> 1) & 1) ^ 1, abort_flag)))) break;
            const uint32_t qs = smem_u32(s_q) + buf * q_bytes;
            const int rows = sg.R;                         // <= RC: one q tile
            uint64_t bits = 0;
            if (sg.total > sg.len && lane < rows) {
                // lane r: the drafts that query row r attends; transposed below, for the thread that has a draft's row
                const int token = lane / p.G;
                bits = p.mask ? p.mask[((int64_t)sg.b * p.n + token) * p.words] : (2ull << token) - 1;
            }
            constexpr bool f32 = NQ == 3;
            constexpr int chunks = f32 ? D / 4 : D / 8, step = 32 / chunks;      // 16-byte pieces of a row of q
            const int c = lane % chunks;
            const char *qg = reinterpret_cast<const char *>(p.q) + c * 16;
            for (int r0 = 0; r0 < rows; r0 += 8 * step) {
                uint4 x[8];
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const int r = r0 + u * step + lane / chunks;
                    if (r < rows) x[u] = *reinterpret_cast<const uint4 *>(qg + tree_out_row(p, sg.b, sg.kvh, r) * (chunks * 16));
                }
                if (seg == 0 && r0 == 0) mbar_arrive(&sb.q_asked);
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const int r = r0 + u * step + lane / chunks;
                    if (r < rows) {
                        if (!f32) {
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(qs + (c >> 3) * q_box + r * 128 + (((c & 7) ^ (r & 7)) << 4)),
                                         "r"(x[u].x), "r"(x[u].y), "r"(x[u].z), "r"(x[u].w) : "memory");
                        } else {
                            float v[4] = {__uint_as_float(x[u].x), __uint_as_float(x[u].y), __uint_as_float(x[u].z), __uint_as_float(x[u].w)};
#pragma unroll
                            for (int term = 0; term < 3; term++) {
                                const uint32_t lo = pack_bf16(v[0], v[1]), hi = pack_bf16(v[2], v[3]);
                                v[0] -= bf16lo(lo); v[1] -= bf16hi(lo); v[2] -= bf16lo(hi); v[3] -= bf16hi(hi);
                                const int rr = term * RP + r;
                                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(qs + (c >> 4) * q_box + rr * 128 + ((((c & 15) >> 1) ^ (rr & 7)) << 4) + (c & 1) * 8),
                                             "r"(lo), "r"(hi) : "memory");
                            }
                        }
                    }
                }
            }
            if (sg.total > sg.len) {
#pragma unroll 4
                for (int j = 0; j < 32; j++) {
                    const uint32_t col = __ballot_sync(0xffffffffu, (bits >> j) & 1);
                    if (lane == j) sb.sees[seg & 7][j] = col;
                }
            }
            fence_async();
            mbar_arrive(&sb.q_full[buf]);
        }
    } else if (warp == 13) {
        // ---------------------------------------------------------------- S^T (the warp stays converged, one elected lane executes)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const uint32_t leader = elect_one();
        const uint32_t idesc = instr_desc(kTile, n_s, 0, 0);
        constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29), kLbo = 1u << 16;
        const uint32_t kv_base = smem_u32(s_kv), q_base = smem_u32(s_q);
        int k = 0, slot = 0, phase = 0;
        for (int seg = 0; next_segment(sb, seg, sg, ok, lane); seg++) {
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.q_full[seg & 1], (seg >> 1) & 1, abort_flag)))) break;
            const uint32_t q_lo = (((q_base + (seg & 1) * q_bytes) >> 4) & 0x3FFFu) | kLbo;
            for (int i = sg.i0; i < sg.i1; i++, k++) {
                const int g = k & 1, cg = k >> 1;
                ok = mbar_wait(&sb.full[slot], phase, abort_flag);
                if (ok && cg > 0) ok = mbar_wait(&sb.s_free[g], (cg - 1) & 1, abort_flag);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                fence_async();
                tc_fence_after();
                const uint32_t k_lo = (((kv_base + (uint32_t)slot * kSlot) >> 4) & 0x3FFFu) | kLbo;
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++)
                    mma_ss_if(leader, tmem + kColS + g * 96, make_desc(k_lo + (ks >> 2) * (kKvBox >> 4) + (ks & 3) * 2, kDescHi),
                              make_desc(q_lo + (ks >> 2) * (q_box >> 4) + (ks & 3) * 2, kDescHi), idesc, ks > 0);
                tc_commit_if(leader, &sb.s_full[g]);
                tc_commit_if(leader, &sb.empty[slot]);
                slot += 2;
                if (slot >= a.stages) { slot = 0; phase ^= 1; }
            }
            if (!ok) break;
            tc_commit_if(leader, &sb.q_empty[seg & 1]);
        }
        tc_commit_if(leader, &sb.drain[0]);
        mbar_wait(&sb.drain[0], 0, abort_flag);
    } else if (warp == 14) {
        // ---------------------------------------------------------------- O^T
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const uint32_t leader = elect_one();
        const uint32_t idesc = instr_desc(D, n_o, 1, 1);
        constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29), kLbo = (uint32_t)(kKvBox >> 4) << 16;
        const uint32_t kv_base = smem_u32(s_kv), p_base = smem_u32(s_p);
        int k = 0, slot = 1, phase = 0;
        for (int seg = 0; next_segment(sb, seg, sg, ok, lane); seg++) {
            const int n = sg.i1 - sg.i0;
            for (int j = 0; j < n; j++, k++) {
                const int g = k & 1, cg = k >> 1;
                ok = mbar_wait(&sb.full[slot], phase, abort_flag) && mbar_wait(&sb.p_ready[g], cg & 1, abort_flag);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                fence_async();
                tc_fence_after();
                const uint32_t v_lo = (((kv_base + (uint32_t)slot * kSlot) >> 4) & 0x3FFFu) | kLbo;
                const uint32_t p_lo = (((p_base + g * kPBytes) >> 4) & 0x3FFFu) | kLbo;
                const uint32_t add = (j >> 1) % kWindow != 0 ? 1u : 0u;     // tile j >> 1 of its group in this segment
#pragma unroll
                for (int ks = 0; ks < kTile / 16; ks++)
                    mma_ss_if(leader, tmem + kColO + g * 64, make_desc(v_lo + ks * 128, kDescHi), make_desc(p_lo + ks * 128, kDescHi), idesc, ks > 0 ? 1u : add);
                tc_commit_if(leader, &sb.pv_done[g]);
                tc_commit_if(leader, &sb.empty[slot]);
                slot += 2;
                if (slot >= a.stages) { slot = 1; phase ^= 1; }
            }
            if (!ok) break;
        }
        tc_commit_if(leader, &sb.drain[1]);
        mbar_wait(&sb.drain[1], 0, abort_flag);
    } else if (warp == 15) {
        // ---------------------------------------------------------------- results
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        constexpr int W = D + 4;
        for (int seg = 0; next_segment(sb, seg, sg, ok, lane); seg++) {
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.x_ready, seg & 1, abort_flag)))) break;
            float *rec = sg.flags & 1 ? nullptr : p.recs + ((int64_t)blockIdx.x * 2 + (sg.flags >> 1)) * a.rec_rows * W;
            if (lane < sg.R) {                             // lane r: how much of each group's O counts
                const int r = lane;
                const float r0 = sb.xref[0][r], r1 = sb.xref[1][r];
                const float s0 = (sb.wsum[0][0][r] + sb.wsum[0][1][r]) + (sb.wsum[0][2][r] + sb.wsum[0][3][r]);
                const float s1 = (sb.wsum[1][0][r] + sb.wsum[1][1][r]) + (sb.wsum[1][2][r] + sb.wsum[1][3][r]);
                const float M = fmaxf(r0, r1), m = M == kUnset ? -INFINITY : M;
                const float f0 = ex2(r0 - M), f1 = ex2(r1 - M);
                const float L = s0 * f0 + s1 * f1, inv = inverse_sum(L);
                const int64_t orow = tree_out_row(p, sg.b, sg.kvh, r);
                sb.join[r] = make_float2(f0 * inv, f1 * inv);
                sb.orow[r] = orow;
                if (rec) {
                    *reinterpret_cast<float4 *>(rec + r * W + D) = make_float4(m * kLn2, L, 0.f, 0.f);
                    mark_cut(p, orow);
                } else {
                    store_row_stats<D>(p, orow, m, L);
                }
            }
            __syncwarp();
#pragma unroll 2
            for (int e = lane; e < sg.R * (D / 4); e += 32) {
                const int r = e / (D / 4), col = e % (D / 4) * 4;
                const float2 f = sb.join[r];
                const float4 o0 = *reinterpret_cast<const float4 *>(s_x + r * D + col), o1 = *reinterpret_cast<const float4 *>(s_x + (RC + r) * D + col);
                const float4 v = make_float4(o0.x * f.x + o1.x * f.y, o0.y * f.x + o1.y * f.y, o0.z * f.x + o1.z * f.y, o0.w * f.x + o1.w * f.y);
                if (rec) *reinterpret_cast<float4 *>(rec + r * W + col) = v;
                else store_row4<D>(p, sb.orow[r], col, v);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sb.x_free);
        }
    } else {
        // ---------------------------------------------------------------- softmax groups
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        const int g = warp >> 2, w = warp & 3, row = w * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(w * 32) << 16);
        const uint32_t s_at = lanes + kColS + g * 96, o_at = lanes + kColO + g * 64;
        const uint32_t p_row = smem_u32(s_p) + g * kPBytes + row * 128;
        const float c = p.scale_log2e;
        // the output column of this thread: head_dim 64 is an M = 64 tile, whose rows sit in 16 lanes of every warp
        const bool has_d = D == 128 || lane < 16;
        const int d = D == 128 ? row : w * 16 + (lane & 15);
        int k = 0, cg = 0;
        float acc[RC], l[RC];
        // every exit of the group is decided by a vote, so that its barriers always meet
        for (int seg = 0;; seg++) {
            const bool more = next_segment(sb, seg, sg, ok, lane);
            if (group_any(g, !ok) || !more) break;
#pragma unroll
            for (int r = 0; r < RC; r++) { acc[r] = 0.f; l[r] = 0.f; }
            int jg = 0;                                                        // this group's tiles of the segment
            bool quit = false;
            const int k_seg = k - sg.i0;
            for (int i = sg.i0 + ((k & 1) != g ? 1 : 0); i < sg.i1; i += 2) {
                const int t0 = i * kTile, kk = k_seg + i;
                ok = mbar_wait(&sb.s_full[g], cg & 1, abort_flag);
                if (ok && cg > 0) ok = mbar_wait(&sb.pv_done[g], (cg - 1) & 1, abort_flag);   // P may be written, O^T read
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after();
                float x[RC];
                bool grown = !ok;
                if (ok) {
                    tmem_terms<RC, RP, NQ, false>(s_at, x);
                    const int valid = sb.valid[kk & 7];
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sb.s_free[g]);
                    if (jg > 0 && jg % kWindow == 0) tmem_terms<RC, RP, NP, true>(o_at, acc);
#pragma unroll
                    for (int r = 0; r < RC; r++) x[r] *= c;
                    const int at = t0 + row;
                    if (p.raw) {
                        float *raw = p.raw + ((int64_t)sg.b * p.Hq + sg.kvh * p.G) * p.raw_ld + at;
#pragma unroll
                        for (int r = 0; r < RC; r++)
                            if (r < sg.R) raw[(int64_t)r * p.raw_ld] = x[r];
                    }
                    if (t0 + kTile > sg.len || valid != 15) {
                        const int j = at - sg.len;                             // >= 0: a draft row
                        uint32_t see = 0;
                        if (at < sg.total && ((valid >> w) & 1)) see = j < 0 ? 0xffffffffu : sb.sees[seg & 7][j];
#pragma unroll
                        for (int r = 0; r < RC; r++)
                            if (!((see >> r) & 1)) x[r] = -INFINITY;
                    }
                }
                if (jg == 0) {
                    // the references: the scores of the tile's first row, where there is one
                    if (row == 0) {
#pragma unroll
                        for (int r = 0; r < RC; r++) sb.ref[g][r] = ok && x[r] > -INFINITY && x[r] < INFINITY ? x[r] : kUnset;
                    }
                    group_any(g, false);
                }
                float ref[RC];
#pragma unroll
                for (int r = 0; r < RC; r++) ref[r] = sb.ref[g][r];
                if (ok) {
                    float top = -INFINITY;
#pragma unroll
                    for (int r = 0; r < RC; r++) top = fmaxf(top, x[r] - ref[r]);
                    grown = top > kGrow;
                }
                if (group_any(g, grown)) {
                    if ((quit = group_any(g, !ok || *abort_flag))) break;
                    // a query row whose reference was passed takes the tile's maximum for one; what has been added up so far follows
#pragma unroll
                    for (int r = 0; r < RC; r++) {
                        float m = x[r];
#pragma unroll
                        for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
                        if (lane == 0) sb.wmax[g][w][r] = m;
                    }
                    group_any(g, false);
                    float f[RC];
#pragma unroll
                    for (int r = 0; r < RC; r++) {
                        const float m = fmaxf(fmaxf(sb.wmax[g][0][r], sb.wmax[g][1][r]), fmaxf(sb.wmax[g][2][r], sb.wmax[g][3][r]));
                        f[r] = 1.f;
                        if (m > ref[r] + kGrow && m < INFINITY) {
                            f[r] = ex2(ref[r] - m);
                            ref[r] = m;
                        }
                        if (row == 0) sb.ref[g][r] = ref[r];
                        l[r] *= f[r];
                        acc[r] *= f[r];
                    }
                    if (jg % kWindow != 0) {
#pragma unroll
                        for (int t = 0; t < NP; t++) {
                            uint32_t o[RC];
                            tmem_ld<RC>(o_at + t * RP, o);
                            tc_wait_ld();
#pragma unroll
                            for (int r = 0; r < RC; r++) o[r] = __float_as_uint(__uint_as_float(o[r]) * f[r]);
                            tmem_st<RC>(o_at + t * RP, o);
                        }
                        tc_wait_st();
                    }
                    group_any(g, false);                                       // wmax is read, ref written
                }
                // P^T in two or three bf16 terms, up to 16 columns at a time (of 32: 8, and the references fetched again)
                constexpr int kGroup = RC <= 16 ? RC : 8;
#pragma unroll
                for (int y = 0; y < RC; y += kGroup) {
                    uint32_t pk[NP][kGroup / 2];
                    if constexpr (RC > 16) {
#pragma unroll
                        for (int r = 0; r < kGroup; r++) ref[y + r] = sb.ref[g][y + r];
                    }
#pragma unroll
                    for (int r = 0; r < kGroup; r += 2) {
                        float e0 = ex2(x[y + r] - ref[y + r]), e1 = ex2(x[y + r + 1] - ref[y + r + 1]);
                        l[y + r] += e0;
                        l[y + r + 1] += e1;
                        uint32_t h = pack_bf16(e0, e1);
                        pk[0][r / 2] = h;
#pragma unroll
                        for (int t = 1; t < NP; t++) {
                            e0 -= bf16lo(h); e1 -= bf16hi(h);
                            h = pack_bf16(e0, e1);
                            pk[t][r / 2] = h;
                        }
                    }
#pragma unroll
                    for (int t = 0; t < NP; t++) {
                        if constexpr (RC == 4) {
                            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(p_row + (((t * (RP / 8)) ^ (row & 7)) << 4)), "r"(pk[t][0]), "r"(pk[t][1]) : "memory");
                        } else {
#pragma unroll
                            for (int z = 0; z < kGroup; z += 8)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p_row + (((t * (RP / 8) + (y + z) / 8) ^ (row & 7)) << 4)),
                                             "r"(pk[t][z / 2]), "r"(pk[t][z / 2 + 1]), "r"(pk[t][z / 2 + 2]), "r"(pk[t][z / 2 + 3]) : "memory");
                        }
                    }
                }
                fence_async();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sb.p_ready[g]);
                jg++;
                cg++;
            }
            if (quit) break;
            k += sg.i1 - sg.i0;

            // ---- end of the segment: the group leaves its sums in shared memory
            ok = jg == 0 || mbar_wait(&sb.pv_done[g], (cg - 1) & 1, abort_flag);
            if (ok && seg > 0) ok = mbar_wait(&sb.x_free, (seg - 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (group_any(g, !ok)) break;
            tc_fence_after();
            if (jg > 0) tmem_terms<RC, RP, NP, true>(o_at, acc);
            tc_fence_before();
            const float s = column_sum<RC>(l, lane);
            if (lane < RC) sb.wsum[g][w][lane] = s;
            if (has_d) {
#pragma unroll
                for (int r = 0; r < RC; r++) s_x[(g * RC + r) * D + d] = acc[r];
            }
            if (row < RC) sb.xref[g][row] = jg == 0 ? kUnset : sb.ref[g][row];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sb.x_ready);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sb.abort_flag) atomicExch(&g_narrow_status, 1);
    if (warp == 15) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

constexpr size_t kSmemMost = 227 * 1024 - (sizeof(Bars) + 1023) / 1024 * 1024 - 1024;     // dynamic: beside Bars, and 1024 bytes to align

template <int D, int RC, int NQ, int NP>
cudaError_t launch_terms(const TreeParams &p, TcArgs &a, cudaStream_t st) {
    constexpr int RP = RC <= 16 ? 16 : 32;
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    constexpr size_t slot = kTile * D * 2, rest = 2 * kPBytes + 2 * (size_t)(RP * NQ * D * 2) + 2 * RC * D * sizeof(float);
    // an even number: a slot is K's or V's for good, so that its barriers have one producer and one consumer, each of which waits for
    // every phase in turn (a barrier's parity says nothing to one that skips phases)
    constexpr int slots = (int)((kSmemMost - rest) / slot);
    static_assert(slots >= 4, "two slots each of K and V");
    a.stages = slots > kMaxSlots ? kMaxSlots : slots & ~1;
    if (dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(tree_narrow_kernel<D, RC, NQ, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSmemMost + 1024));
        if (e != cudaSuccess) return e;
        if (dev < 64) ready[dev] = true;
    }
    return launch_dependent(tree_narrow_kernel<D, RC, NQ, NP>, dim3(sm_count()), kThreads, a.stages * slot + rest + 1024, st, p, a);
}
template <int D, int RC>
cudaError_t launch_rc(const TreeParams &p, TcArgs &a, cudaStream_t st) {
    if (a.p_terms == 3) return a.q_terms == 3 ? launch_terms<D, RC, 3, 3>(p, a, st) : launch_terms<D, RC, 1, 3>(p, a, st);
    return a.q_terms == 3 ? launch_terms<D, RC, 3, 2>(p, a, st) : launch_terms<D, RC, 1, 2>(p, a, st);
}
template <int D> cudaError_t launch_narrow_d(const TreeParams &p, TcArgs &a, cudaStream_t st) {
    const int R = p.n * p.G;
    if (R > 16) {
        if constexpr (D == 64)
            if (a.q_terms == 3) return launch_terms<D, 32, 3, 2>(p, a, st);
        return launch_terms<D, 32, 1, 2>(p, a, st);
    }
    return R <= 4 ? launch_rc<D, 4>(p, a, st) : (R <= 8 ? launch_rc<D, 8>(p, a, st) : launch_rc<D, 16>(p, a, st));
}

}  // namespace

// P's terms are columns of one 64-column operand; 96 columns of Q at head size 128 would leave two slots.  So the rule is the operand's width,
// not a crossing of two times: fp32 results go from 84 us at 16 rows to 195 at 24, where the wide kernel has to take them.
// 32 sequences of 2 - 4 K rows, 32 q / 8 kv heads of 128, here and in tree_wide_tc.cu: bf16, 8 rows 76 and 96 us, 16 rows 79 and 95,
// 24 rows 91 and 97, 32 rows 96 and 99; fp32 q and results, 8 rows 76 and 193, 16 rows 84 and 192.  64 sequences, 9 q / 3 kv heads of 64,
// fp32 q and bf16 results: 15 rows 47 and 72, 30 rows 69 and 74.
bool tree_narrow_takes(int R, int q_terms, int p_terms, int head_dim) {
    return R <= 16 || (R <= 32 && p_terms == 2 && (q_terms == 1 || head_dim == 64));
}

cudaError_t launch_tree_narrow(const TreeParams &p, TcArgs &a, int head_dim, cudaStream_t st) {
    return head_dim == 64 ? launch_narrow_d<64>(p, a, st) : launch_narrow_d<128>(p, a, st);
}

int tree_narrow_status(int reset, int *status_out) {
    return read_status_word("attn_decode_tree_status", g_narrow_status, reset, status_out);
}

}  // namespace treetc
}  // namespace nimllm
