// tree_decode_tc.cu -- the attention of tree_decode.cu for bf16 caches, on the Blackwell tensor cores.
//
// The query rows of a (sequence, KV head) -- (token, head) pairs -- are the M = 128 rows of tcgen05 products, cached rows come
// in tiles of 64:   S = Q K^T  (128 x 64, fp32 in TMEM),  P = exp2(S c - m),  O_tile = P V  (128 x D, fp32 in TMEM).
//
//   warps 0-3  softmax, one thread per TMEM lane.  The tile's O is added to fp32 registers instead of being accumulated in TMEM:
//              thousands of rows added up by the tensor core would lose what 32-bit results promise.
//   warps 4-5  producers: K and V rows of a tile into a ring of shared-memory stages with cp.async, swizzled as the MMA reads
//              them.  No tensor map, because a block may start at any 16-byte offset (kv_off) and end at any row; rows past the
//              sequence are filled with zeros, never read.
//   warp 6     Q of the next (sequence, KV head) while the last tiles of the one before are worked on
//   warp 7     issues the MMAs: S of tile j + 1 before P V of tile j
//
// Copies: with R <= 32 (64) query rows the Q tile holds them 4 (2) times and every copy takes a quarter (half) of a tile's
// columns; the P columns of the others stay zero.  The copies are independent softmaxes over disjoint rows, joined at the end of
// a segment.  All four warps then work on a tile that has only 32 rows of scores.
//
// Precision: the products are exact in fp32 accumulation, so the only roundings to bf16 are those of P and of an fp32 q.  Both are
// split: an fp32 q into three bf16 terms (2^-26 left), P into two terms for bf16 results (2^-17) and three for fp32 results.
// The terms are further MMAs into the same accumulator.
//
// Every wait is bounded as in prefill_tc.cu: after about 2 s without progress the CTA aborts and raises the status word.
#include "tree_finish.cuh"

namespace nimllm {

namespace {

using namespace tc;
using namespace treetc;

__device__ int g_tree_status = 0;      // sticky, nimllm_attn_decode_tree_status

constexpr int kTile = 64;              // cached rows of a tile
constexpr int kRows = 128;             // MMA rows
constexpr int kMaxStages = 10;
constexpr int kThreads = 256;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColP = 64, kColO = 192;    // S | P terms (3 x 32) | O x 2
constexpr int kQBox = kRows * 128, kKvBox = kTile * 128;  // bytes of a 64-column box

struct Bars {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t q_full, q_empty, s_full, s_free, p_ready, pv_done, epi, drain;
    uint32_t tmem_base;
    volatile int abort_flag;
    SpanStart start;
    int valid[kMaxStages];             // bit 0, 1: the pages of the tile's two halves exist
    float2 ml[kRows];                  // copies: maximum and sum of every lane, then of every row
};

// the rows of a tile that query row (token) attends, one bit each
__device__ __forceinline__ uint64_t visible_rows(const TreeParams &p, const SeqWork &w, int b, int token, int t0, int valid) {
    const int n_left = w.total - t0;                       // > 0
    uint64_t vis = 0;
    const int committed = w.len - t0;                      // rows of the tile before the drafts
    if (committed >= kTile) {
        vis = ~0ull;
    } else {
        const int j0 = committed > 0 ? 0 : -committed, at = committed > 0 ? committed : 0;   // draft j0 is row `at` of the tile
        uint64_t bits;
        if (p.mask) {
            const uint64_t *m = p.mask + ((int64_t)b * p.n + token) * p.words;
            const int k = j0 >> 6, sh = j0 & 63;
            bits = m[k] >> sh;
            if (sh && k + 1 < p.words) bits |= m[k + 1] << (64 - sh);
        } else {
            const int n = token + 1 - j0;                  // drafts j0 .. token
            bits = n <= 0 ? 0ull : (n >= 64 ? ~0ull : (1ull << n) - 1);
        }
        vis = (committed > 0 ? (1ull << committed) - 1 : 0ull) | (bits << at);
    }
    if (n_left < kTile) vis &= (1ull << n_left) - 1;
    if (!(valid & 1)) vis &= 0xffffffff00000000ull;
    if (!(valid & 2)) vis &= 0x00000000ffffffffull;
    return vis;
}

template <int D, int C>
__global__ void __launch_bounds__(kThreads, 1) tree_tc_kernel(TreeParams p, TcArgs a) {
    constexpr int RPT = kRows / C;             // query rows of a tile
    constexpr int NC = kTile / C;              // columns of a copy
    constexpr int kBoxes = D / 64;
    constexpr int kQTerm = kRows * D * 2, kKv = kTile * D * 2, kStage = 2 * kKv;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Bars sb;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *s_q = smem, *s_kv = smem + a.q_terms * kQTerm;
    float *s_out = reinterpret_cast<float *>(s_kv + a.stages * kStage);      // copies: [128][33]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    launch_dependents();
    grid_dependency_wait();

    const int n_units = span_begin<RPT, kTile, kThreads>(p, a, sb.start);
    if (n_units == 0) return;
    if (threadIdx.x == 0) {
        sb.abort_flag = 0;
        for (int s = 0; s < a.stages; s++) { mbar_init(&sb.full[s], 65); mbar_init(&sb.empty[s], 1); }
        mbar_init(&sb.q_full, 32); mbar_init(&sb.q_empty, 1);
        mbar_init(&sb.s_full, 1); mbar_init(&sb.s_free, 4);
        mbar_init(&sb.p_ready, 4); mbar_init(&sb.pv_done, 1);
        mbar_init(&sb.epi, 4); mbar_init(&sb.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // rows of the Q tile that no query row fills stay zero (or hold an earlier segment's rows): finite, never used
    for (int x = threadIdx.x; x < a.q_terms * kQTerm / 16; x += kThreads) reinterpret_cast<uint4 *>(s_q)[x] = make_uint4(0, 0, 0, 0);
    fence_async();
    if (warp == 7) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sb.tmem_base)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sb.tmem_base;
    volatile int *abort_flag = &sb.abort_flag;
    SpanWalk<RPT, kTile> walk(p, sb.start.b, sb.start.h, sb.start.i, n_units);
    Segment sg;
    bool ok = true;

    if (warp == 4 || warp == 5) {
        // ---------------------------------------------------------------- K and V rows
        constexpr int kChunks = D / 8;                     // 16-byte pieces of a row
        constexpr int kStep = 64 / kChunks;                // rows per round of the 64 threads
        const int t = threadIdx.x - 128;
        const int c = t % kChunks, r_in = t / kChunks;
        const uint32_t kv = smem_u32(s_kv);
        const __nv_bfloat16 *kg = reinterpret_cast<const __nv_bfloat16 *>(p.k) + c * 8, *vg = reinterpret_cast<const __nv_bfloat16 *>(p.v) + c * 8;
        int k = 0;                                         // tiles issued
        while (ok && walk.next(sg)) {
            for (int i = sg.i0; ok && i < sg.i1; i++, k++) {
                const int slot = k % a.stages, t0 = i * kTile;
                const int n = min(kTile, sg.w.total - t0);
                // the two halves of a tile lie in one page each (page_rows >= 32)
                const int64_t h0 = cache_row(p.rows, sg.b, sg.kvh, t0);
                const int64_t h1 = n > 32 ? cache_row(p.rows, sg.b, sg.kvh, t0 + 32) : 0;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.empty[slot], ((k / a.stages) & 1) ^ 1, abort_flag)))) break;
                if (t == 0) {                              // the 65th arrival publishes the word
                    sb.valid[slot] = (h0 >= 0 ? 1 : 0) | (h1 >= 0 ? 2 : 0);
                    mbar_arrive(&sb.full[slot]);
                }
                const uint32_t dst = kv + slot * kStage + (c >> 3) * kKvBox;
#pragma unroll
                for (int r0 = 0; r0 < kTile; r0 += kStep) {
                    const int r = r0 + r_in;
                    const int64_t base = r < 32 ? h0 : h1;
                    const bool have = r < n && base >= 0;
                    const int64_t off = have ? base + (int64_t)(r & 31) * D : 0;
                    const uint32_t d = dst + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                    cp_async16(d, kg + off, have ? 16 : 0);
                    cp_async16(d + kKv, vg + off, have ? 16 : 0);
                }
                cp_async_arrive(&sb.full[slot]);
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 6) {
        // ---------------------------------------------------------------- Q
        const uint32_t qs = smem_u32(s_q);
        int seg = 0;
        while (ok && walk.next(sg)) {
            if (seg > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(&sb.q_empty, (seg - 1) & 1, abort_flag)))) break;
            const int q0 = sg.qt * RPT, rows = min(RPT, sg.w.R - q0);
            if (p.q_dtype == NIMLLM_BF16) {
                constexpr int kChunks = D / 8, kStep = 32 / kChunks;
                const int c = lane % kChunks;
                const uint32_t dst = qs + (c >> 3) * kQBox;
                for (int r0 = 0; r0 < rows; r0 += 4 * kStep) {
                    uint4 x[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const int r = r0 + u * kStep + lane / kChunks;
                        if (r < rows)
                            x[u] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const __nv_bfloat16 *>(p.q) + tree_out_row(p, sg.b, sg.kvh, q0 + r) * D + c * 8);
                    }
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const int r = r0 + u * kStep + lane / kChunks;
                        if (r < rows)
#pragma unroll
                            for (int y = 0; y < C; y++) {
                                const int rr = y * RPT + r;
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)),
                                             "r"(x[u].x), "r"(x[u].y), "r"(x[u].z), "r"(x[u].w) : "memory");
                            }
                    }
                }
            } else {
                constexpr int kChunks = D / 4, kStep = 32 / kChunks;      // 4 values a lane
                const int c = lane % kChunks;
                const uint32_t dst = qs + (c >> 4) * kQBox;
                for (int r0 = 0; r0 < rows; r0 += 4 * kStep) {
                    float4 x[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const int r = r0 + u * kStep + lane / kChunks;
                        if (r < rows) x[u] = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p.q) + tree_out_row(p, sg.b, sg.kvh, q0 + r) * D + c * 4);
                    }
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const int r = r0 + u * kStep + lane / kChunks;
                        if (r < rows) {
                            float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                            for (int term = 0; term < a.q_terms; term++) {
                                const uint32_t lo = pack_bf16(v[0], v[1]), hi = pack_bf16(v[2], v[3]);
                                v[0] -= bf16lo(lo); v[1] -= bf16hi(lo); v[2] -= bf16lo(hi); v[3] -= bf16hi(hi);
#pragma unroll
                                for (int y = 0; y < C; y++) {
                                    const int rr = y * RPT + r;
                                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(dst + term * kQTerm + rr * 128 + ((((c & 15) >> 1) ^ (rr & 7)) << 4) + (c & 1) * 8),
                                                 "r"(lo), "r"(hi) : "memory");
                                }
                            }
                        }
                    }
                }
            }
            fence_async();
            mbar_arrive(&sb.q_full);
            seg++;
        }
    } else if (warp == 7) {
        // ---------------------------------------------------------------- MMA issuer (converged, one elected lane executes)
        const uint32_t leader = elect_one();
        constexpr uint32_t idesc_qk = instr_desc(kRows, kTile, 0, 0), idesc_pv = instr_desc(kRows, D, 0, 1);
        constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
        constexpr uint32_t kLboK = 1u << 16, kLboV = (uint32_t)(kKvBox >> 4) << 16;
        const uint32_t q_lo = ((smem_u32(s_q) >> 4) & 0x3FFFu) | kLboK, kv_base = smem_u32(s_kv);
        int k = 0, seg = 0;                                // tiles issued (P V), segments begun
        auto issue_s = [&](int tile) -> bool {
            if (!mbar_wait(&sb.full[tile % a.stages], (tile / a.stages) & 1, abort_flag)) return false;
            if (tile > 0 && !mbar_wait(&sb.s_free, (tile - 1) & 1, abort_flag)) return false;
            fence_async();
            tc_fence_after();
            const uint32_t k_lo = (((kv_base + (uint32_t)(tile % a.stages) * kStage) >> 4) & 0x3FFFu) | kLboK;
            for (int t = 0; t < a.q_terms; t++)
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++)
                    mma_ss_if(leader, tmem + kColS, make_desc(q_lo + t * (kQTerm >> 4) + (ks >> 2) * (kQBox >> 4) + (ks & 3) * 2, kDescHi),
                              make_desc(k_lo + (ks >> 2) * (kKvBox >> 4) + (ks & 3) * 2, kDescHi), idesc_qk, (t > 0 || ks > 0) ? 1u : 0u);
            tc_commit_if(leader, &sb.s_full);
            return true;
        };
        auto issue_pv = [&](int tile) -> bool {
            if (!mbar_wait(&sb.p_ready, tile & 1, abort_flag)) return false;
            tc_fence_after();
            const uint32_t v_lo = (((kv_base + (uint32_t)(tile % a.stages) * kStage + kKv) >> 4) & 0x3FFFu) | kLboV;
            for (int t = 0; t < a.p_terms; t++)
#pragma unroll
                for (int ks = 0; ks < kTile / 16; ks++)
                    mma_ts_if(leader, tmem + kColO + (tile & 1) * D, tmem + kColP + t * 32 + ks * 8, make_desc(v_lo + ks * 128, kDescHi), idesc_pv,
                              (t > 0 || ks > 0) ? 1u : 0u);
            tc_commit_if(leader, &sb.pv_done);
            tc_commit_if(leader, &sb.empty[tile % a.stages]);
            return true;
        };
        while (ok && walk.next(sg)) {
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.q_full, seg & 1, abort_flag)))) break;
            const int n = sg.i1 - sg.i0;
            if (!(ok = __all_sync(0xffffffffu, issue_s(k)))) break;
            if (n == 1) tc_commit_if(leader, &sb.q_empty);
            for (int j = 0; j < n; j++, k++) {
                if (j + 1 < n) {
                    if (!(ok = __all_sync(0xffffffffu, issue_s(k + 1)))) break;
                    if (j + 2 == n) tc_commit_if(leader, &sb.q_empty);
                }
                if (!(ok = __all_sync(0xffffffffu, issue_pv(k)))) break;
            }
            seg++;
        }
        tc_commit_if(leader, &sb.drain);
        mbar_wait(&sb.drain, 0, abort_flag);
    } else {
        // ---------------------------------------------------------------- softmax
        const int row = threadIdx.x;                       // TMEM lane
        const int copy = row / RPT, r = row % RPT;
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        const float c = p.scale_log2e;
        {   // the P columns of the other copies stay zero from here on
            uint32_t z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 96; x += 8) tmem_st8(lanes + kColP + x, z);
            tc_wait_st();
        }
        int k = 0, epi = 0;
        float acc[D];
        auto epi_sync = [&]() -> bool {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sb.epi);
            const bool good = __all_sync(0xffffffffu, mbar_wait(&sb.epi, epi & 1, abort_flag));
            epi++;
            return good;
        };
        auto add_o = [&](int tile) {
#pragma unroll
            for (int x = 0; x < D; x += 32) {
                uint32_t o[32];
                tmem_ld32(lanes + kColO + (tile & 1) * D + x, o);
                tc_wait_ld();
#pragma unroll
                for (int y = 0; y < 32; y++) acc[x + y] += __uint_as_float(o[y]);
            }
        };
        while (ok && walk.next(sg)) {
            const int qr = sg.qt * RPT + r;
            const bool live = qr < sg.w.R;
            const bool busy = __any_sync(0xffffffffu, live);           // a warp without query rows only keeps step
            const int token = live ? qr / p.G : 0;
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int x = 0; x < D; x++) acc[x] = 0.f;
            for (int i = sg.i0; i < sg.i1; i++, k++) {
                const int t0 = i * kTile;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.s_full, k & 1, abort_flag)))) break;
                tc_fence_after();
                float x[NC];
                const uint32_t s_at = lanes + kColS + copy * NC;
                if (busy) {
                    uint32_t *xr = reinterpret_cast<uint32_t *>(x);
                    if constexpr (NC == 16) tmem_ld16(s_at, xr);
                    else tmem_ld32(s_at, xr);
                    if constexpr (NC == 64) tmem_ld32(s_at + 32, xr + 32);
                    tc_wait_ld();
                }
                const int valid = sb.valid[k % a.stages];
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sb.s_free);
                float corr = 1.f, safe = 0.f;
                if (busy) {
#pragma unroll
                    for (int y = 0; y < NC; y++) x[y] *= c;
                    if (p.raw && live) {
                        float *raw = p.raw + ((int64_t)sg.b * p.Hq + sg.kvh * p.G + qr) * p.raw_ld + t0 + copy * NC;
#pragma unroll
                        for (int y = 0; y < NC; y += 4) *reinterpret_cast<float4 *>(raw + y) = make_float4(x[y], x[y + 1], x[y + 2], x[y + 3]);
                    }
                    if (t0 + kTile > sg.w.len || valid != 3) {
                        const uint64_t vis = (live ? visible_rows(p, sg.w, sg.b, token, t0, valid) : ~0ull) >> (copy * NC);
#pragma unroll
                        for (int y = 0; y < NC; y++)
                            if (!((vis >> y) & 1)) x[y] = -INFINITY;
                    }
                    float m0 = fmaxf(x[0], x[1]), m1 = fmaxf(x[2], x[3]);
#pragma unroll
                    for (int y = 4; y < NC; y += 4) { m0 = max3(m0, x[y], x[y + 1]); m1 = max3(m1, x[y + 2], x[y + 3]); }
                    const float m_new = fmaxf(m, fmaxf(m0, m1));
                    safe = m_new == -INFINITY ? 0.f : m_new;
                    corr = ex2(m - safe);
                    m = m_new;
                }
                if (i > sg.i0) {
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.pv_done, (k - 1) & 1, abort_flag)))) break;
                    tc_fence_after();
                }
                if (busy) {
                    float s0 = 0.f, s1 = 0.f;
                    const uint32_t p_at = lanes + kColP + copy * (NC / 2);
#pragma unroll
                    for (int y0 = 0; y0 < NC; y0 += 16) {
                        uint32_t t0_[8], t1_[8], t2_[8];
#pragma unroll
                        for (int y = 0; y < 16; y += 2) {
                            float e0 = ex2(x[y0 + y] - safe), e1 = ex2(x[y0 + y + 1] - safe);
                            s0 += e0;
                            s1 += e1;
                            uint32_t h = pack_bf16(e0, e1);
                            t0_[y / 2] = h;
                            e0 -= bf16lo(h); e1 -= bf16hi(h);
                            h = pack_bf16(e0, e1);
                            t1_[y / 2] = h;
                            e0 -= bf16lo(h); e1 -= bf16hi(h);
                            t2_[y / 2] = pack_bf16(e0, e1);
                        }
                        tmem_st8(p_at + y0 / 2, t0_);
                        tmem_st8(p_at + 32 + y0 / 2, t1_);
                        if (a.p_terms == 3) tmem_st8(p_at + 64 + y0 / 2, t2_);
                    }
                    l = l * corr + (s0 + s1);
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sb.p_ready);
                if (busy && i > sg.i0) {
                    add_o(k - 1);
                    if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
                        for (int y = 0; y < D; y++) acc[y] *= corr;
                    }
                }
            }
            if (!ok) break;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.pv_done, (k - 1) & 1, abort_flag)))) break;
            tc_fence_after();
            if (busy) add_o(k - 1);
            tc_fence_before();

            constexpr int W = D + 4;
            float *rec = sg.whole ? nullptr : p.recs + ((int64_t)blockIdx.x * 2 + sg.slot) * kRecRows * W;
            if constexpr (C == 1) {
                if (live) {
                    const float inv = l > 0.f ? 1.f / l : 0.f;
                    const int64_t orow = tree_out_row(p, sg.b, sg.kvh, qr);
#pragma unroll
                    for (int d = 0; d < D; d += 4) {
                        const float4 v = make_float4(acc[d] * inv, acc[d + 1] * inv, acc[d + 2] * inv, acc[d + 3] * inv);
                        if (rec) *reinterpret_cast<float4 *>(rec + r * W + d) = v;
                        else store_row4<D>(p, orow, d, v);
                    }
                    if (rec) *reinterpret_cast<float4 *>(rec + r * W + D) = make_float4(m * kLn2, l, 0.f, 0.f);
                    else store_row_stats<D>(p, orow, m, l);
                }
            } else {
                sb.ml[row] = make_float2(m, l);
                if (!(ok = epi_sync())) break;
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int y = 0; y < C; y++) M = fmaxf(M, sb.ml[y * RPT + r].x);
                const float safe = M == -INFINITY ? 0.f : M;
#pragma unroll
                for (int y = 0; y < C; y++) { const float2 v = sb.ml[y * RPT + r]; L += v.y * ex2(v.x - safe); }
                const float f = (L > 0.f ? 1.f / L : 0.f) * ex2(m - safe);
                const int rows = min(RPT, sg.w.R - sg.qt * RPT);
#pragma unroll
                for (int d0 = 0; d0 < D; d0 += 32) {
#pragma unroll
                    for (int y = 0; y < 32; y++) s_out[row * 33 + y] = acc[d0 + y] * f;
                    if (!(ok = epi_sync())) break;
                    for (int e = row; e < rows * 8; e += kRows) {
                        const int rr = e >> 3, d = (e & 7) * 4;
                        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int y = 0; y < C; y++)
#pragma unroll
                            for (int z = 0; z < 4; z++) v[z] += s_out[(y * RPT + rr) * 33 + d + z];
                        const float4 o = make_float4(v[0], v[1], v[2], v[3]);
                        if (rec) *reinterpret_cast<float4 *>(rec + rr * W + d0 + d) = o;
                        else store_row4<D>(p, tree_out_row(p, sg.b, sg.kvh, sg.qt * RPT + rr), d0 + d, o);
                    }
                    if (!(ok = epi_sync())) break;
                }
                if (!ok) break;
                if (copy == 0 && live) {
                    if (rec) *reinterpret_cast<float4 *>(rec + r * W + D) = make_float4(M * kLn2, L, 0.f, 0.f);
                    else store_row_stats<D>(p, tree_out_row(p, sg.b, sg.kvh, qr), M, L);
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sb.abort_flag) atomicExch(&g_tree_status, 1);
    if (warp == 7) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

constexpr size_t kSmemMost = 227 * 1024 - (sizeof(Bars) + 1023) / 1024 * 1024 - 1024;     // dynamic: beside Bars, and 1024 bytes to align

template <int D, int C>
cudaError_t launch_c(const TreeParams &p, TcArgs &a, cudaStream_t st) {
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const size_t q = (size_t)a.q_terms * kRows * D * 2, stage = 2 * kTile * D * 2, join = C > 1 ? kRows * 33 * sizeof(float) : 0;
    int stages = (int)((kSmemMost - q - join) / stage);
    a.stages = stages > kMaxStages ? kMaxStages : stages;
    if (dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(tree_tc_kernel<D, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSmemMost + 1024));
        if (e != cudaSuccess) return e;
        if (dev < 64) ready[dev] = true;
    }
    return launch_dependent(tree_tc_kernel<D, C>, dim3(sm_count()), kThreads, q + join + a.stages * stage + 1024, st, p, a);
}

template <int D>
cudaError_t launch_d(const TreeParams &p, TcArgs &a, cudaStream_t st) {
    const int R = p.n * p.G;
    const bool narrow = tree_narrow_takes(R, a.q_terms, a.p_terms, D);
    const int rpt = narrow ? kNarrowRows : (R <= 32 ? 32 : (R <= 64 ? 64 : 128));
    cudaError_t e;
    if (narrow) e = launch_tree_narrow(p, a, D, st);
    else e = rpt == 32 ? launch_c<D, 4>(p, a, st) : (rpt == 64 ? launch_c<D, 2>(p, a, st) : launch_c<D, 1>(p, a, st));
    if (e != cudaSuccess) return e;
    FinishArgs f = {};
    f.tc = a; f.rpt = rpt; f.tile = narrow ? kNarrowTile : kTile; f.workers = sm_count();
    return launch_finish<D>(p, f, st);
}

}  // namespace

size_t tree_tc_workspace_bytes(int batch, int n, int n_head, int n_kv_head, int head_dim) {
    (void)n; (void)n_head; (void)n_kv_head;
    return rec_bytes(head_dim) + (size_t)sm_count() * sizeof(int4) + ((size_t)batch + 1) * sizeof(int64_t);
}

int launch_tree_tc(const char *who, TreeParams &p, int head_dim, void *workspace, cudaStream_t st) {
    TcArgs a = {};
    p.recs = (float *)workspace;
    a.starts = (int4 *)((unsigned char *)workspace + rec_bytes(head_dim));
    a.cum = (int64_t *)(a.starts + sm_count());
    a.q_terms = p.q_dtype == NIMLLM_F32 ? 3 : 1;
    a.p_terms = (p.out && p.out_dtype == NIMLLM_F32) || p.partials_out ? 3 : 2;
    a.stages = 0;
    const cudaError_t e = head_dim == 64 ? launch_d<64>(p, a, st) : launch_d<128>(p, a, st);
    if (e != cudaSuccess) return fail(NIMLLM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return NIMLLM_OK;
}

// Reads (and clears) a sticky word of the current device.
template <typename T> static int read_status(T &word, int reset, int *out) {
    int st = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&st, word, sizeof(int));
    if (e == cudaSuccess && reset && st != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(word, &zero, sizeof(int));
    }
    if (e != cudaSuccess) return fail(NIMLLM_ERR_CUDA, "attn_decode_tree_status: %s", cudaGetErrorString(e));
    *out = st;
    return NIMLLM_OK;
}

}  // namespace nimllm

extern "C" int nimllm_attn_decode_tree_status(int reset) {
    int wide = 0, narrow = 0;
    int rc = nimllm::read_status(nimllm::g_tree_status, reset, &wide);
    if (!rc) rc = nimllm::treetc::tree_narrow_status(reset, &narrow);
    return rc ? -rc : (wide | narrow);
}
