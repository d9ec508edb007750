// tree_wide_tc.cu -- tree and scored decode over bf16 caches with many query rows per KV head, on the tensor cores; and the choice
// between this kernel and the one for few rows (tree_narrow_tc.cu).
//
// The query rows of a (sequence, KV head) -- (token, head) pairs -- are the M = 128 rows of tcgen05 products, cached rows come
// in tiles of 64:   S = Q K^T  (128 x 64, fp32 in TMEM),  P = exp2(S c - ref),  O += P V  (128 x D, fp32 in TMEM, P from TMEM).
//
//   warps 0-3, 4-7   two softmax groups, one thread per query row (= TMEM lane).  Up to 128 rows: both have the same rows and take the
//                    tiles in turn, group 0 joins the two results in TMEM at the end of a segment.  More: 256 rows share every tile,
//                    half of them in each group, so that a cached row is still read once.
//   warps 8-11       K rows (8, 9) and V rows (10, 11) into a ring of slots with cp.async, swizzled as the MMA reads them.  No tensor
//                    map, because a block may start at any 16-byte offset (kv_off), a page may end anywhere and a sequence at any row;
//                    rows past it are filled with zeros, never read.
//   warps 12, 15     walk of the CTA's span (12) and Q of the segments to come
//   warps 13, 14     issue Q K^T and P V, each in order and waiting for its own operands alone
//
// ref is a query row's running maximum, taken anew only when a score passes it by more than 2^32: rounding is relative to P's own
// size, and fp32 has the range.  O is then rescaled in TMEM, which costs nothing while it does not happen.
//
// Precision: the products are exact in fp32 accumulation, so the only roundings to bf16 are those of P and of an fp32 q.  For fp32
// results both are split into three bf16 terms (2^-26 left), further MMAs into the same accumulator, and O is taken from TMEM into
// registers every few tiles: thousands of rows added up by the tensor core would lose what 32-bit results promise.  For bf16 results
// P is rounded to bf16 like the result itself (the sum is taken of the rounded values, so that a single large weight stays exact): results
// are off by 2.3e-3 of their norm where the rounding of the result alone is 1.7e-3.  With a second term the trees measured below took 160 us
// for 148, and 196 for 174 call by call; fp32 results have the weights in 32 bits.
// That is the precision of more than 32 query rows only: 17 - 32 rows of an fp32 q with heads of 128, which the narrow kernel does not
// take, have two terms (2^-17 left) as its rows have: 32 sequences of 2 - 4 K rows, 20 query rows, 130 us.  Scored decode has two as
// well, so that l is the sum of the weights themselves, which the scores are divided by (32 sequences of 2 - 4 K rows, 40 heads of 128:
// 102 us, with one term 100).
//
// Measured (graph replay): 8 trees of 64 tokens over 9 - 16 K rows in pages, 32 q / 8 kv heads of 128, bf16: 148 us (172 call by call from
// Python; 8 us more without the rows' policy of leaving L2 first, which keeps records, Q and code there).  The rows' bytes at the measured
// peak of HBM are 65 us, the products at the library's matrix rate 64.  A tile takes 2700 cycles, 2200 of them from its first product to its
// last: 24 products that follow one another every 93 cycles or so, 64 columns wide or 128, while the tensor pipe is active for 36 % of the
// cycles.  Its exponentials take 1024 of the two groups' turns.  Tiles of 128 rows, which need 16 products for the
// same work, were built with one S of both groups and with P over S, before that policy: 179 and 199 us for 168, because a group then
// waits for the other's reading of S or for its own P.
//
// Every wait is bounded as in prefill_tc.cu: after about 2 s without progress the CTA aborts and raises the status word.
#include "tree_finish.cuh"

namespace nimllm {
namespace treetc {

namespace {

using namespace tc;

__device__ int g_wide_status = 0;      // sticky, nimllm_attn_decode_tree_status

constexpr int kTile = 64;              // cached rows of a tile
constexpr int kRows = 128;             // MMA rows
constexpr int kMaxSlots = 16;
constexpr int kThreads = 512;
constexpr int kWindow = 4;             // fp32 results: tiles between two readings of O
constexpr float kGrow = 32.f;          // log2 units by which a score may pass the reference
constexpr float kUnset = -1e30f;       // reference of a query row that has attended nothing yet: any score passes it
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kGroupCols = 256, kColP = 64, kColO = 128;      // a group: S | P (fp32 results: over S, third term) | O
constexpr int kQBox = kRows * 128, kKvBox = kTile * 128;           // bytes of a 64-column box
constexpr int kSegs = 8, kValid = 32;

struct SegEntry {
    int b, kvh, qt, i0, i1, len, total, R, flags;  // b < 0: the end; flags: 1 whole, 2 the second record slot
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
    int valid[kValid];                 // by tile: bits 0, 1: the pages of its two halves exist
    float2 other[kRows];               // group 1's reference and sum of every row
};

// segment s of the queue, in every lane; false at the end and when a wait gave up (ok says which)
__device__ __forceinline__ bool next_segment(Bars &sb, int s, SegEntry &e, bool &ok, int lane) {
    ok = __all_sync(0xffffffffu, mbar_wait(&sb.seg_full[s % kSegs], (s / kSegs) & 1, &sb.abort_flag));
    if (!ok) return false;
    e = sb.segs[s % kSegs];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sb.seg_empty[s % kSegs]);
    return e.b >= 0;
}

// the rows of a tile that query row (token) attends, one bit each
__device__ __forceinline__ uint64_t visible_rows(const TreeParams &p, const SegEntry &w, int b, int token, int t0, int valid) {
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

__device__ __forceinline__ uint64_t pair2(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpair2(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2_f32(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t mul2_f32(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// 32 scaled scores, less the reference, -> NP terms of P (16 packed columns each); adds the exponentials (NP = 1: rounded) to l
template <int NP> __device__ __forceinline__ void exps32(const float *x, float ref, float &l, uint32_t pk[NP][16]) {
    const uint64_t nr = pair2(-ref, -ref);
    uint64_t sum = 0ull;
#pragma unroll
    for (int y = 0; y < 32; y += 2) {
        float e0, e1;
        unpair2(add2_f32(pair2(x[y], x[y + 1]), nr), e0, e1);
        e0 = ex2(e0);
        e1 = ex2(e1);
        uint64_t e = pair2(e0, e1);
        uint32_t h = pack_bf16(e0, e1);
        pk[0][y / 2] = h;
        sum = add2_f32(sum, NP == 1 ? pair2(bf16lo(h), bf16hi(h)) : e);
#pragma unroll
        for (int t = 1; t < NP; t++) {
            e = add2_f32(e, pair2(-bf16lo(h), -bf16hi(h)));
            unpair2(e, e0, e1);
            h = pack_bf16(e0, e1);
            pk[t][y / 2] = h;
        }
    }
    float s0, s1;
    unpair2(sum, s0, s1);
    l += s0 + s1;
}
__device__ __forceinline__ void scale32(float *x, float c) {
    const uint64_t c2 = pair2(c, c);
#pragma unroll
    for (int y = 0; y < 32; y += 2) unpair2(mul2_f32(pair2(x[y], x[y + 1]), c2), x[y], x[y + 1]);
}
__device__ __forceinline__ float max32(const float *x) {
    float m0 = fmaxf(x[0], x[1]), m1 = fmaxf(x[2], x[3]);
#pragma unroll
    for (int y = 4; y < 32; y += 4) { m0 = max3(m0, x[y], x[y + 1]); m1 = max3(m1, x[y + 2], x[y + 3]); }
    return fmaxf(m0, m1);
}
__device__ __forceinline__ void hide32(float *x, uint32_t vis) {
#pragma unroll
    for (int y = 0; y < 32; y++)
        if (!((vis >> y) & 1)) x[y] = -INFINITY;
}

// NQ, NP: terms of q (1, 3) and of P (1, 2, 3); SPLIT: 256 query rows a tile, half of them per group (else 128, the tiles in turn)
template <int D, int NQ, int NP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) tree_wide_kernel(TreeParams p, TcArgs a) {
    constexpr int RPT = SPLIT ? 2 * kRows : kRows;
    constexpr int kQTerm = kRows * D * 2, kQTile = NQ * kQTerm, kSlot = kTile * D * 2;
    constexpr int kQBufs = !SPLIT && NQ == 1 ? 2 : 1;
    constexpr int kOWindow = NP == 3 ? kWindow : 1 << 30;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Bars sb;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *s_q = smem, *s_kv = smem + (SPLIT ? 2 : kQBufs) * kQTile;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    launch_dependents();
    grid_dependency_wait();
    const int n_units = span_begin<RPT, kTile, kThreads>(p, a, sb.start);
    if (n_units == 0) return;
    if (threadIdx.x == 0) {
        sb.abort_flag = 0;
        for (int s = 0; s < a.stages; s++) { mbar_init(&sb.full[s], 65); mbar_init(&sb.empty[s], 1); }
        for (int s = 0; s < kSegs; s++) { mbar_init(&sb.seg_full[s], 1); mbar_init(&sb.seg_empty[s], 15); }
        for (int g = 0; g < 2; g++) {
            mbar_init(&sb.q_full[g], 64); mbar_init(&sb.q_empty[g], 1);
            mbar_init(&sb.s_full[g], 1); mbar_init(&sb.s_free[g], 4);
            mbar_init(&sb.p_ready[g], 4); mbar_init(&sb.pv_done[g], 1);
        }
        mbar_init(&sb.q_asked, 64); mbar_init(&sb.x_ready, 4); mbar_init(&sb.x_free, 4); mbar_init(&sb.drain[0], 1); mbar_init(&sb.drain[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // rows of the Q tile that no query row fills stay zero (or hold an earlier segment's rows): finite, never used
    for (int x = threadIdx.x; x < (SPLIT ? 2 : kQBufs) * kQTile / 16; x += kThreads) reinterpret_cast<uint4 *>(s_q)[x] = make_uint4(0, 0, 0, 0);
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
        // ---------------------------------------------------------------- even slots are K's, odd ones V's
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        constexpr int kChunks = D / 8, kStep = 64 / kChunks;
        const int which = (warp - 8) >> 1, t = (int)threadIdx.x - 256 - which * 64, c = t % kChunks, r_in = t / kChunks;
        const uint32_t kv = smem_u32(s_kv);
        const uint64_t policy = evict_first_policy();
        const __nv_bfloat16 *src = reinterpret_cast<const __nv_bfloat16 *>(which ? p.v : p.k) + c * 8;
        int k = 0, slot = which, phase = 1;
        for (int seg = 0; next_segment(sb, seg, sg, ok, lane); seg++) {
            // the loads of the first Q go out before a ring full of rows queues up in front of them
            if (seg == 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(&sb.q_asked, 0, abort_flag)))) break;
            for (int i = sg.i0; i < sg.i1; i++, k++) {
                const int t0 = i * kTile, n = min(kTile, sg.total - t0);
                // a half of a tile lies in one page (page_rows >= 32)
                const int64_t h0 = cache_row(p.rows, sg.b, sg.kvh, t0), h1 = n > 32 ? cache_row(p.rows, sg.b, sg.kvh, t0 + 32) : 0;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.empty[slot], phase, abort_flag)))) break;
                if (t == 0) {                              // the 65th arrival publishes the tile's word
                    if (which == 0) sb.valid[k % kValid] = (h0 >= 0 ? 1 : 0) | (h1 >= 0 ? 2 : 0);
                    mbar_arrive(&sb.full[slot]);
                }
                const uint32_t dst = kv + slot * kSlot + (c >> 3) * kKvBox;
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int64_t h = y ? h1 : h0;
                    const int r_end = h >= 0 ? n - y * 32 : 0;
                    const __nv_bfloat16 *g = src + (h >= 0 ? h : 0) + r_in * D;
#pragma unroll
                    for (int r0 = 0; r0 < 32; r0 += kStep) {
                        const int rr = y * 32 + r0 + r_in;
                        const bool have = r0 + r_in < r_end;
                        cp_async16(dst + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), have ? g + r0 * D : src, have ? 16 : 0, policy);
                    }
                }
                cp_async_arrive(&sb.full[slot]);
                slot += 2;
                if (slot >= a.stages) { slot = which; phase ^= 1; }
            }
            if (!ok) break;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 12 || warp == 15) {
        // ---------------------------------------------------------------- segments and Q
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        SpanWalk<RPT, kTile> walk(p, sb.start.b, sb.start.h, sb.start.i, n_units);
        const int half = warp == 15;
        for (int seg = 0;; seg++) {
            if (warp == 12) {
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.seg_empty[seg % kSegs], ((seg / kSegs) & 1) ^ 1, abort_flag)))) break;
                Segment s;
                const bool more = walk.next(s);
                sg = more ? SegEntry{s.b, s.kvh, s.qt, s.i0, s.i1, s.w.len, s.w.total, s.w.R, (s.whole ? 1 : 0) | (s.slot ? 2 : 0)}
                          : SegEntry{-1, 0, 0, 0, 0, 0, 0, 0, 0};
                if (lane == 0) {
                    sb.segs[seg % kSegs] = sg;
                    mbar_arrive(&sb.seg_full[seg % kSegs]);
                }
                if (!more) break;
            } else if (!next_segment(sb, seg, sg, ok, lane)) {
                break;
            }
            const int buf = seg % kQBufs;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.q_empty[buf], ((seg / kQBufs) & 1) ^ 1, abort_flag)))) break;
            const uint32_t qs = smem_u32(s_q) + (SPLIT ? 0 : buf * kQTile);
            const int q0 = sg.qt * RPT, rows = min(RPT, sg.R - q0);
            if constexpr (NQ == 1) {
                constexpr int kChunks = D / 8, kStep = 32 / kChunks;
                const int c = lane % kChunks;
                const __nv_bfloat16 *qg = reinterpret_cast<const __nv_bfloat16 *>(p.q) + c * 8;
                for (int r = half * kStep + lane / kChunks; r < rows; r += 2 * kStep)
                    cp_async16(qs + (r >> 7) * kQTile + (c >> 3) * kQBox + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4),
                               qg + tree_out_row(p, sg.b, sg.kvh, q0 + r) * D, 16);
                if (seg == 0) mbar_arrive(&sb.q_asked);
                asm volatile("cp.async.wait_all;" ::: "memory");
            } else {
                constexpr int kChunks = D / 4, kStep = 32 / kChunks;      // four values a lane
                static_assert(kStep == 128 / D, "");
                const int c = lane % kChunks;
                const float *qg = reinterpret_cast<const float *>(p.q) + c * 4;
                for (int r0 = half * kStep; r0 < rows; r0 += 16 * kStep) {
                    float4 x[8];
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const int r = r0 + u * 2 * kStep + lane / kChunks;
                        if (r < rows) x[u] = *reinterpret_cast<const float4 *>(qg + tree_out_row(p, sg.b, sg.kvh, q0 + r) * D);
                    }
                    if (seg == 0 && r0 == half * kStep) mbar_arrive(&sb.q_asked);
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const int r = r0 + u * 2 * kStep + lane / kChunks;
                        if (r < rows) {
                            float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
                            for (int term = 0; term < NQ; term++) {
                                const uint32_t lo = pack_bf16(v[0], v[1]), hi = pack_bf16(v[2], v[3]);
                                v[0] -= bf16lo(lo); v[1] -= bf16hi(lo); v[2] -= bf16lo(hi); v[3] -= bf16hi(hi);
                                asm volatile("st.shared.v2.b32 [%0], {%1, %2};"
                                             ::"r"(qs + (r >> 7) * kQTile + term * kQTerm + (c >> 4) * kQBox + (r & 127) * 128 + ((((c & 15) >> 1) ^ (r & 7)) << 4) + (c & 1) * 8),
                                             "r"(lo), "r"(hi) : "memory");
                            }
                        }
                    }
                }
            }
            if (NQ > 1 && seg == 0 && half * (128 / D) >= rows) mbar_arrive(&sb.q_asked);      // this warp has no row
            fence_async();
            mbar_arrive(&sb.q_full[buf]);
        }
    } else if (warp == 13) {
        // ---------------------------------------------------------------- S (the warp stays converged, one elected lane executes)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const uint32_t leader = elect_one();
        constexpr uint32_t idesc = instr_desc(kRows, kTile, 0, 0);
        constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29), kLbo = 1u << 16;
        const uint32_t kv_base = smem_u32(s_kv), q_base = smem_u32(s_q);
        int k = 0, slot = 0, phase = 0;
        for (int seg = 0; next_segment(sb, seg, sg, ok, lane); seg++) {
            const int buf = seg % kQBufs;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.q_full[buf], (seg / kQBufs) & 1, abort_flag)))) break;
            for (int i = sg.i0; i < sg.i1; i++, k++) {
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.full[slot], phase, abort_flag)))) break;
                const uint32_t k_lo = (((kv_base + (uint32_t)slot * kSlot) >> 4) & 0x3FFFu) | kLbo;
                for (int g = SPLIT ? 0 : (k & 1); g < (SPLIT ? 2 : (k & 1) + 1); g++) {
                    const int cg = SPLIT ? k : k >> 1;
                    // fp32 results: P lies over S, so the products of the tile before have to be done
                    if (cg > 0) ok = __all_sync(0xffffffffu, mbar_wait(NP == 3 ? &sb.pv_done[g] : &sb.s_free[g], (cg - 1) & 1, abort_flag));
                    if (!ok) break;
                    fence_async();
                    tc_fence_after();
                    const uint32_t q_lo = (((q_base + (SPLIT ? g : buf) * kQTile) >> 4) & 0x3FFFu) | kLbo;
                    // smallest terms first: the sum is short of bits only from where the large ones have come in
#pragma unroll
                    for (int t = NQ - 1; t >= 0; t--)
#pragma unroll
                        for (int ks = 0; ks < D / 16; ks++)
                            mma_ss_if(leader, tmem + g * kGroupCols, make_desc(q_lo + t * (kQTerm >> 4) + (ks >> 2) * (kQBox >> 4) + (ks & 3) * 2, kDescHi),
                                      make_desc(k_lo + (ks >> 2) * (kKvBox >> 4) + (ks & 3) * 2, kDescHi), idesc, (t < NQ - 1 || ks > 0) ? 1u : 0u);
                    tc_commit_if(leader, &sb.s_full[g]);
                }
                if (!ok) break;
                tc_commit_if(leader, &sb.empty[slot]);
                slot += 2;
                if (slot >= a.stages) { slot = 0; phase ^= 1; }
            }
            if (!ok) break;
            tc_commit_if(leader, &sb.q_empty[buf]);
        }
        tc_commit_if(leader, &sb.drain[0]);
        mbar_wait(&sb.drain[0], 0, abort_flag);
    } else if (warp == 14) {
        // ---------------------------------------------------------------- O
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const uint32_t leader = elect_one();
        constexpr uint32_t idesc = instr_desc(kRows, D, 0, 1);
        constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29), kLbo = (uint32_t)(kKvBox >> 4) << 16;
        const uint32_t kv_base = smem_u32(s_kv);
        int k = 0, slot = 1, phase = 0;
        for (int seg = 0; next_segment(sb, seg, sg, ok, lane); seg++) {
            const int n = sg.i1 - sg.i0;
            for (int j = 0; j < n; j++, k++) {
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.full[slot], phase, abort_flag)))) break;
                const uint32_t v_lo = (((kv_base + (uint32_t)slot * kSlot) >> 4) & 0x3FFFu) | kLbo;
                for (int g = SPLIT ? 0 : (k & 1); g < (SPLIT ? 2 : (k & 1) + 1); g++) {
                    const int cg = SPLIT ? k : k >> 1, jg = SPLIT ? j : j >> 1;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(&sb.p_ready[g], cg & 1, abort_flag)))) break;
                    fence_async();
                    tc_fence_after();
                    const uint32_t at = tmem + g * kGroupCols;
#pragma unroll
                    for (int t = NP - 1; t >= 0; t--)
#pragma unroll
                        for (int ks = 0; ks < kTile / 16; ks++) {
                            // P: 8 packed columns a step (fp32 results: two terms over the 32 columns of S that they came from)
                            const uint32_t pa = NP == 3 && t < 2 ? at + (ks >> 1) * 32 + t * 16 + (ks & 1) * 8 : at + kColP + (NP == 3 ? 0 : t * 32) + ks * 8;
                            mma_ts_if(leader, at + kColO, pa, make_desc(v_lo + ks * 128, kDescHi), idesc, t < NP - 1 || ks > 0 || jg % kOWindow != 0 ? 1u : 0u);
                        }
                    tc_commit_if(leader, &sb.pv_done[g]);
                }
                if (!ok) break;
                tc_commit_if(leader, &sb.empty[slot]);
                slot += 2;
                if (slot >= a.stages) { slot = 1; phase ^= 1; }
            }
            if (!ok) break;
        }
        tc_commit_if(leader, &sb.drain[1]);
        mbar_wait(&sb.drain[1], 0, abort_flag);
    } else {
        // ---------------------------------------------------------------- softmax groups
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        const int g = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + g * kGroupCols;
        const float c = p.scale_log2e;
        constexpr int W = D + 4;
        int k = 0, cg = 0;
        float acc[NP == 3 ? D : 1];
        auto wait = [&](uint64_t *bar, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)); };
        // O joins the registers (fp32 results)
        auto take_o = [&]() {
            if constexpr (NP == 3) {
#pragma unroll
                for (int y0 = 0; y0 < D; y0 += 32) {
                    uint32_t o[32];
                    tmem_ld32(at + kColO + y0, o);
                    tc_wait_ld();
#pragma unroll
                    for (int y = 0; y < 32; y++) acc[y0 + y] += __uint_as_float(o[y]);
                }
            }
        };
        for (int seg = 0; next_segment(sb, seg, sg, ok, lane); seg++) {
            const int qr = sg.qt * RPT + (SPLIT ? g * kRows : 0) + row;
            const bool live = qr < sg.R;
            const bool busy = __any_sync(0xffffffffu, live);           // a warp without query rows only keeps step
            const int token = live ? qr / p.G : 0;
            float ref = kUnset, l = 0.f;
            if constexpr (NP == 3) {
#pragma unroll
                for (int y = 0; y < D; y++) acc[y] = 0.f;
            }
            int jg = 0;
            for (int i = sg.i0 + (!SPLIT && (k & 1) != g ? 1 : 0); i < sg.i1; i += SPLIT ? 1 : 2) {
                const int t0 = i * kTile;
                if (!(ok = wait(&sb.s_full[g], cg & 1))) break;
                // P may be written, O read or rescaled; group 0 has read the O of the segment before
                if (cg > 0 && !(ok = wait(&sb.pv_done[g], (cg - 1) & 1))) break;
                if (!SPLIT && g == 1 && jg == 0 && seg > 0 && !(ok = wait(&sb.x_free, (seg - 1) & 1))) break;
                tc_fence_after();
                if (busy) {
                    const int valid = sb.valid[(k + i - sg.i0) % kValid];
                    const bool tail = t0 + kTile > sg.len || valid != 3;
                    uint64_t vis = ~0ull;
                    if (tail && live) vis = visible_rows(p, sg, sg.b, token, t0, valid);
                    float *raw = p.raw && live ? p.raw + ((int64_t)sg.b * p.Hq + sg.kvh * p.G + qr) * p.raw_ld + t0 : nullptr;
                    // S: for bf16 results all of it stays in registers; for fp32 results, whose O is there, it is fetched twice
                    float x[NP == 3 ? 32 : 64];
                    uint32_t *xr = reinterpret_cast<uint32_t *>(x);
                    auto half = [&](int y, float *v) {                          // scaled, stored and masked
                        scale32(v, c);
                        if (raw) {
#pragma unroll
                            for (int z = 0; z < 32; z += 4) *reinterpret_cast<float4 *>(raw + y + z) = make_float4(v[z], v[z + 1], v[z + 2], v[z + 3]);
                        }
                        if (tail) hide32(v, (uint32_t)(vis >> y));
                    };
                    float top;
                    if constexpr (NP == 3) {
                        tmem_ld32(at + 32, xr);
                        tc_wait_ld();
                        half(32, x);
                        top = max32(x);
                        tmem_ld32(at, xr);
                        tc_wait_ld();
                        half(0, x);
                        top = fmaxf(top, max32(x));
                    } else {
                        tmem_ld32(at, xr);
                        tmem_ld32(at + 32, xr + 32);
                        tc_wait_ld();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sb.s_free[g]);
                        half(0, x);
                        half(32, x + 32);
                        top = fmaxf(max32(x), max32(x + 32));
                    }
                    if (NP == 3 && jg > 0 && jg % kOWindow == 0) take_o();
                    // a reference that was passed by far (or is not there yet) gives way; what has been added up follows
                    const bool grown = top > ref + kGrow && top < INFINITY;
                    if (__any_sync(0xffffffffu, grown)) {
                        const float f = grown ? ex2(ref - top) : 1.f;
                        if (grown) ref = top;
                        l *= f;
                        if constexpr (NP == 3) {
#pragma unroll
                            for (int y = 0; y < D; y++) acc[y] *= f;
                        }
                        if (jg % kOWindow != 0) {
#pragma unroll 1
                            for (int y0 = 0; y0 < D; y0 += 32) {
                                uint32_t o[32];
                                tmem_ld32(at + kColO + y0, o);
                                tc_wait_ld();
#pragma unroll
                                for (int y = 0; y < 32; y++) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                                tmem_st32(at + kColO + y0, o);
                            }
                        }
                    }
                    uint32_t pk[NP][16];
                    exps32<NP>(x, ref, l, pk);
                    if constexpr (NP == 3) {
                        tmem_st16(at, pk[0]);
                        tmem_st16(at + 16, pk[1]);
                        tmem_st16(at + kColP, pk[2]);
                        tmem_ld32(at + 32, xr);
                        tc_wait_ld();
                        raw = nullptr;                                         // stored above
                        half(32, x);
                        exps32<NP>(x, ref, l, pk);
                        tmem_st16(at + 32, pk[0]);
                        tmem_st16(at + 48, pk[1]);
                        tmem_st16(at + kColP + 16, pk[2]);
                    } else {
#pragma unroll
                        for (int t = 0; t < NP; t++) tmem_st16(at + kColP + t * 32, pk[t]);
                        exps32<NP>(x + 32, ref, l, pk);
#pragma unroll
                        for (int t = 0; t < NP; t++) tmem_st16(at + kColP + t * 32 + 16, pk[t]);
                    }
                    tc_wait_st();
                } else if (NP != 3 && lane == 0) {
                    mbar_arrive(&sb.s_free[g]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sb.p_ready[g]);
                jg++;
                cg++;
            }
            if (!ok) break;
            k += sg.i1 - sg.i0;

            // ---- end of the segment
            if (jg > 0 && !(ok = wait(&sb.pv_done[g], (cg - 1) & 1))) break;
            if (!SPLIT && g == 1 && jg == 0 && seg > 0 && !(ok = wait(&sb.x_free, (seg - 1) & 1))) break;
            tc_fence_after();
            if (busy && jg > 0) take_o();
            if (!SPLIT && g == 1) {
                // the other group joins: sums through shared memory, O where it is (fp32 results: put back there)
                if constexpr (NP == 3) {
                    if (busy) {
#pragma unroll
                        for (int y0 = 0; y0 < D; y0 += 32) tmem_st32(at + kColO + y0, reinterpret_cast<uint32_t *>(acc) + y0);
                        tc_wait_st();
                    }
                }
                sb.other[row] = make_float2(ref, l);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sb.x_ready);
                continue;
            }
            float m = ref, f0 = l != 0.f ? 1.f : 0.f, f1 = 0.f;      // 0: the group has nothing; a sum that is NaN counts
            if (!SPLIT) {
                if (!(ok = wait(&sb.x_ready, seg & 1))) break;
                tc_fence_after();
                const float2 o = sb.other[row];
                m = fmaxf(ref, o.x);
                f0 = ex2(ref - m);
                f1 = ex2(o.x - m);
                const float sum = l * f0 + o.y * f1;
                f0 = l != 0.f ? f0 : 0.f;
                f1 = o.y != 0.f ? f1 : 0.f;
                l = sum;
            }
            if (busy) {
                const float inv = inverse_sum(l);                  // may be NaN: a group that has nothing stays at 0
                f0 *= inv;
                if (!SPLIT) f1 = f1 != 0.f ? f1 * inv : 0.f;
                m = m == kUnset ? -INFINITY : m;
                const int64_t orow = tree_out_row(p, sg.b, sg.kvh, qr);
                float *rec = sg.flags & 1 ? nullptr : p.recs + ((int64_t)blockIdx.x * 2 + (sg.flags >> 1)) * a.rec_rows * W + ((SPLIT ? g * kRows : 0) + row) * 4;
                const bool any1 = !SPLIT && __any_sync(0xffffffffu, f1 != 0.f);      // split rows have no second O: no columns behind group 1's
                // O in TMEM: rolled, for less code to fetch once a segment (48 rows over 2 - 4 K 106 -> 96 us); O in registers has fixed names
#pragma unroll (NP == 3 ? D / 16 : 1)
                for (int y0 = 0; y0 < D; y0 += 16) {
                    float v[16];
                    if constexpr (NP == 3) {
#pragma unroll
                        for (int y = 0; y < 16; y++) v[y] = acc[y0 + y] * f0;
                    } else {
                        tmem_ld16(at + kColO + y0, reinterpret_cast<uint32_t *>(v));
                        tc_wait_ld();
#pragma unroll
                        for (int y = 0; y < 16; y++) v[y] = f0 != 0.f ? v[y] * f0 : 0.f;   // a group without tiles has no O
                    }
                    if (any1) {
                        float u[16];
                        tmem_ld16(at + kGroupCols + kColO + y0, reinterpret_cast<uint32_t *>(u));
                        tc_wait_ld();
#pragma unroll
                        for (int y = 0; y < 16; y++) v[y] += f1 != 0.f ? u[y] * f1 : 0.f;
                    }
                    if (live) {
                        if (rec) {
#pragma unroll
                            for (int y = 0; y < 16; y += 4) *reinterpret_cast<float4 *>(rec + (y0 + y) * a.rec_rows) = make_float4(v[y], v[y + 1], v[y + 2], v[y + 3]);
                        } else {
#pragma unroll
                            for (int y = 0; y < 16; y += 8) store_row8<D>(p, orow, y0 + y, v + y);
                        }
                    }
                }
                if (live) {
                    if (rec) {
                        *reinterpret_cast<float4 *>(rec + D * a.rec_rows) = make_float4(m * kLn2, l, 0.f, 0.f);
                        mark_cut(p, orow);
                    } else {
                        store_row_stats<D>(p, orow, m, l);
                    }
                }
            }
            tc_fence_before();
            if (!SPLIT) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&sb.x_free);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sb.abort_flag) atomicExch(&g_wide_status, 1);
    if (warp == 15) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

constexpr size_t kSmemMost = 227 * 1024 - (sizeof(Bars) + 1023) / 1024 * 1024 - 1024;     // dynamic: beside Bars, and 1024 bytes to align

template <int D, int NQ, int NP, bool SPLIT>
cudaError_t launch_terms(const TreeParams &p, TcArgs &a, cudaStream_t st) {
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    constexpr size_t q = (size_t)(SPLIT || NQ == 1 ? 2 : 1) * NQ * kRows * D * 2, slot = kTile * D * 2;
    constexpr int slots = (int)((kSmemMost - q) / slot);
    static_assert(slots >= 4, "two slots each of K and V");
    a.stages = slots > kMaxSlots ? kMaxSlots : slots & ~1;      // even: a slot is K's or V's for good (tree_narrow_tc.cu)
    if (dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(tree_wide_kernel<D, NQ, NP, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSmemMost + 1024));
        if (e != cudaSuccess) return e;
        if (dev < 64) ready[dev] = true;
    }
    return launch_dependent(tree_wide_kernel<D, NQ, NP, SPLIT>, dim3(sm_count()), kThreads, q + a.stages * slot + 1024, st, p, a);
}

// 256 rows share a tile where Q has one term; three leave too few slots, and at head size 64 no second Q to fetch ahead.  Measured with
// and without: heads of 128, one term, 256 rows over 9 - 16 K 152.2 and 153.4 us, 160 rows over 2 - 4 K 94.9 and 96.8; heads of 64,
// three terms, 192 rows 103 and 91 us
bool splits(int R, int q_terms) { return R > kRows && q_terms == 1; }
int rows_per_tile(int R, int q_terms, int p_terms, int head_dim) {
    return tree_narrow_takes(R, q_terms, p_terms, head_dim) ? kNarrowRows : (splits(R, q_terms) ? 2 * kRows : kRows);
}

template <int D, int NQ, int NP>
cudaError_t launch_wide(const TreeParams &p, TcArgs &a, cudaStream_t st) {
    if constexpr (NQ == 1)
        if (splits(p.n * p.G, NQ)) return launch_terms<D, NQ, NP, true>(p, a, st);
    return launch_terms<D, NQ, NP, false>(p, a, st);
}

template <int D>
cudaError_t launch_d(const TreeParams &p, TcArgs &a, cudaStream_t st) {
    const int R = p.n * p.G;
    const bool narrow = tree_narrow_takes(R, a.q_terms, a.p_terms, D);
    cudaError_t e;
    // terms of P: three for 32-bit results, else one where its rounding is no larger than the result's.  Two for rows that the narrow kernel
    // leaves, and where scores are kept: their softmax has the same sum l, which one term would have to round with P
    const int np = a.p_terms == 3 ? 3 : (R <= kNarrowRows || p.score ? 2 : 1);
    if (narrow) e = launch_tree_narrow(p, a, D, st);
    else if (a.q_terms == 1) e = np == 1 ? launch_wide<D, 1, 1>(p, a, st) : (np == 2 ? launch_wide<D, 1, 2>(p, a, st) : launch_wide<D, 1, 3>(p, a, st));
    else e = np == 1 ? launch_wide<D, 3, 1>(p, a, st) : (np == 2 ? launch_wide<D, 3, 2>(p, a, st) : launch_wide<D, 3, 3>(p, a, st));
    if (e != cudaSuccess) return e;
    FinishArgs f = {};
    f.tc = a; f.rpt = rows_per_tile(R, a.q_terms, a.p_terms, D); f.tile = narrow ? kNarrowTile : kTile; f.workers = sm_count(); f.by_col = !narrow;
    return launch_finish<D>(p, f, st);
}

}  // namespace
}  // namespace treetc

using namespace treetc;

// enough for either q and out type: the rows of a record slot grow with the query rows alone
static int record_rows(int R) { return R <= kNarrowRows ? 128 : (R <= kRows ? kRows : 2 * kRows); }
static size_t tc_record_bytes(int R, int head_dim) { return (size_t)sm_count() * 2 * record_rows(R) * rec_stride(head_dim) * sizeof(float); }

size_t tree_tc_workspace_bytes(int batch, int n, int n_head, int n_kv_head, int head_dim) {
    return tc_record_bytes(n * (n_head / n_kv_head), head_dim) + (size_t)sm_count() * sizeof(int4) + ((size_t)batch + 1) * sizeof(int64_t);
}

int launch_tree_tc(const char *who, TreeParams &p, int head_dim, void *workspace, cudaStream_t st) {
    TcArgs a = {};
    p.recs = (float *)workspace;
    a.rec_rows = record_rows(p.n * p.G);
    a.starts = (int4 *)((unsigned char *)workspace + tc_record_bytes(p.n * p.G, head_dim));
    a.cum = (int64_t *)(a.starts + sm_count());
    a.q_terms = p.q_dtype == NIMLLM_F32 ? 3 : 1;
    a.p_terms = (p.out && p.out_dtype == NIMLLM_F32) || p.partials_out ? 3 : 2;
    const cudaError_t e = head_dim == 64 ? launch_d<64>(p, a, st) : launch_d<128>(p, a, st);
    if (e != cudaSuccess) return fail(NIMLLM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return NIMLLM_OK;
}

}  // namespace nimllm

extern "C" int nimllm_attn_decode_tree_status(int reset) {
    int wide = 0, narrow = 0;
    int rc = nimllm::read_status_word("attn_decode_tree_status", nimllm::treetc::g_wide_status, reset, &wide);
    if (!rc) rc = nimllm::treetc::tree_narrow_status(reset, &narrow);
    return rc ? -rc : (wide | narrow);
}
