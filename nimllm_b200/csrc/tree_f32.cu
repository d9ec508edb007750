// tree_f32.cu -- tree and scored decode over fp32 caches, on the CUDA cores: fp32 products, as the reference's cache asks for.
//
// Up to 16 query rows per KV head (tree_f32_narrow_kernel) the cached rows are streamed: a warp takes eight rows of a tile (16 of
// head_dim 64), a row lies across 32 (16) lanes with 16 bytes each, and the partial products of 32 (16) scores are summed by one halving
// exchange, which leaves one score per lane -- a shuffle per score.  K of the next tile is fetched while V is worked on and the
// other way round.  The list of tiles is cut into equal spans like the tensor-core kernels' (tree_tc.cuh).
//
// More query rows (tree_f32_tiled_kernel) are bound by the multiply-adds: a CTA has 32 or 64 query rows and one chunk of cached
// rows, a thread a (2 or 4) x (BN / 8) block of the score tile and the same rows' D / 8 output columns, as in prefill_f32.cu.
//
// Measured (graph replay): scored decode of 16 sequences of 4 - 8 K rows, 32 q / 8 kv heads of 128: 144 us, 124 at the measured peak of
// HBM; 7 drafts of one sequence of 505 rows 15 us, its next token 11 us (latency: two launches, a tile, the join); 4 trees of 64 tokens
// over 4 - 8 K rows 774 us, 34 TFLOP/s of multiply-adds, about half of what the CUDA cores have.
#include "tree_finish.cuh"

namespace nimllm {
namespace treetc {

namespace {

constexpr float kUnset = -1e30f;       // reference of a query row that has attended nothing yet: any score passes it
constexpr float kGrow = 8.f;           // log2 units by which a score may pass the reference

__device__ __forceinline__ uint64_t pair2(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpair2(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

constexpr int kWarps = 8;              // one CTA per SM: a thread has 255 registers for rows under way
template <int D> constexpr int warp_rows() { return D == 64 ? 16 : 8; }      // eight 16-byte loads of K and of V per lane
template <int D> constexpr int narrow_tile() { return kWarps * warp_rows<D>(); }
constexpr int kNarrowRpt = 16;

template <int D, int RC>
__global__ void __launch_bounds__(kWarps * 32, 1) tree_f32_narrow_kernel(TreeParams p, TcArgs a) {
    constexpr int WARPS = kWarps, THREADS = WARPS * 32, TILE = narrow_tile<D>(), ROWS = warp_rows<D>();
    constexpr int LANES = D / 4, H = 32 / LANES;           // lanes of a row, rows of a load
    constexpr int NL = ROWS / H;                           // loads of a warp's rows
    constexpr int U = LANES / RC;                          // loads of a step: U * RC scores, one per lane
    constexpr int NS = NL / U;                             // steps
    static_assert(U >= 1 && NS * U == NL, "steps");
    extern __shared__ float sm[];
    float *s_q = sm, *s_acc = s_q + RC * D;                // q rows | every warp's output [WARPS][RC][D]
    float *s_p = s_acc + WARPS * RC * D;                   // weights: [WARPS][H][NL * RC]
    float2 *s_ml = reinterpret_cast<float2 *>(s_p + WARPS * ROWS * RC);     // [WARPS][RC]
    __shared__ SpanStart start;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = lane % LANES, sub = lane / LANES;
    launch_dependents();
    grid_dependency_wait();
    const int n_units = span_begin<kNarrowRpt, TILE, THREADS>(p, a, start);
    if (n_units == 0) return;
    SpanWalk<kNarrowRpt, TILE> walk(p, start.b, start.h, start.i, n_units);
    Segment sg;
    const float *kg = reinterpret_cast<const float *>(p.k) + c * 4, *vg = reinterpret_cast<const float *>(p.v) + c * 4;
    float *sp = s_p + warp * ROWS * RC + sub * NL * RC;
    while (walk.next(sg)) {
        const int R = sg.w.R, total = sg.w.total, len = sg.w.len;
        __syncthreads();                                   // the segment before has been stored
        for (int x = tid; x < RC * D; x += THREADS) {
            const int r = x / D;
            s_q[x] = r < R ? load_as_f32(p.q, p.q_dtype, tree_out_row(p, sg.b, sg.kvh, r) * D + x % D) : 0.f;
        }
        __syncthreads();
        const int64_t base = p.rows.table ? 0 : cache_row(p.rows, sg.b, sg.kvh, 0);
        const int mine = warp * ROWS;
        uint4 kx[NL], vx[NL];
        // a warp's rows lie in one page; rows past the sequence or without a page are zeros
        auto fetch = [&](uint4 *x, const float *g, int t) {
            const int r0 = t * TILE + mine;
            int64_t at = -1;
            if (r0 < total) at = p.rows.table ? cache_row(p.rows, sg.b, sg.kvh, r0) : base + (int64_t)r0 * D;
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int r = j * H + sub;
                x[j] = at >= 0 && r0 + r < total ? ldg_stream(g + at + (int64_t)r * D) : make_uint4(0, 0, 0, 0);
            }
        };
        uint64_t acc[RC][2];
#pragma unroll
        for (int r = 0; r < RC; r++) acc[r][0] = acc[r][1] = 0ull;
        float ref = kUnset, l = 0.f;                       // of query row c % RC
        const int my_r = c % RC;
        fetch(kx, kg, sg.i0);
        fetch(vx, vg, sg.i0);
        for (int t = sg.i0; t < sg.i1; t++) {
            const int r0 = t * TILE + mine;
            float xs[NS];
#pragma unroll
            for (int st = 0; st < NS; st++) {
                float part[U * RC];
#pragma unroll
                for (int r = 0; r < RC; r++) {
                    const float4 q = *reinterpret_cast<const float4 *>(s_q + r * D + c * 4);
                    const uint64_t q01 = pair2(q.x, q.y), q23 = pair2(q.z, q.w);
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const uint4 k = kx[st * U + u];
                        float e, o;
                        unpair2(fma2(q23, pair2(__uint_as_float(k.z), __uint_as_float(k.w)), mul2(q01, pair2(__uint_as_float(k.x), __uint_as_float(k.y)))), e, o);
                        part[u * RC + r] = e + o;
                    }
                }
                // halving exchange over the lanes of a row: lane c is left with the sum of part[c]
#pragma unroll
                for (int h = LANES / 2; h > 0; h >>= 1) {
                    const bool up = c & h;
#pragma unroll
                    for (int i = 0; i < h; i++) {
                        const float give = up ? part[i] : part[i + h], keep = up ? part[i + h] : part[i];
                        part[i] = keep + __shfl_xor_sync(0xffffffffu, give, h);
                    }
                }
                xs[st] = part[0] * p.scale_log2e;
            }
            if (t + 1 < sg.i1) fetch(kx, kg, t + 1);
            float top = -INFINITY;
            const bool tail = r0 + ROWS > len || p.rows.table;
#pragma unroll
            for (int st = 0; st < NS; st++) {
                const int row = r0 + (st * U + c / RC) * H + sub;
                bool see = row < total && my_r < R;
                if (see && tail) {
                    if (row >= len) see = tree_sees(p, sg.b, my_r / p.G, row - len);
                    if (see && p.rows.table) see = cache_row(p.rows, sg.b, sg.kvh, row) >= 0;
                }
                if (see && p.raw) p.raw[((int64_t)sg.b * p.Hq + sg.kvh * p.G + my_r) * p.raw_ld + row] = xs[st];
                if (!see) xs[st] = -INFINITY;
                top = fmaxf(top, xs[st]);
            }
            if (__any_sync(0xffffffffu, top > ref + kGrow && top < INFINITY)) {
                // the references follow the maxima, and with them what has been added up
#pragma unroll
                for (int off = RC; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                const float old = ref;
                if (top > ref && top < INFINITY) ref = top;
                const float f = ex2(old - ref);
                l *= f;
#pragma unroll
                for (int r = 0; r < RC; r++) {
                    const float fr = __shfl_sync(0xffffffffu, f, r);
                    acc[r][0] = mul2(acc[r][0], pair2(fr, fr));
                    acc[r][1] = mul2(acc[r][1], pair2(fr, fr));
                }
            }
            __syncwarp();                                  // the weights of the tile before have been read
#pragma unroll
            for (int st = 0; st < NS; st++) {
                const float w = ex2(xs[st] - ref);
                l += w;
                sp[st * LANES + c] = w;
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const uint64_t v01 = pair2(__uint_as_float(vx[j].x), __uint_as_float(vx[j].y)), v23 = pair2(__uint_as_float(vx[j].z), __uint_as_float(vx[j].w));
#pragma unroll
                for (int r = 0; r < RC; r += 4) {
                    const float4 w = *reinterpret_cast<const float4 *>(sp + j * RC + r);
                    const float ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        acc[r + i][0] = fma2(pair2(ws[i], ws[i]), v01, acc[r + i][0]);
                        acc[r + i][1] = fma2(pair2(ws[i], ws[i]), v23, acc[r + i][1]);
                    }
                }
            }
            if (t + 1 < sg.i1) fetch(vx, vg, t + 1);
        }
        // ---- the warps' results meet in shared memory
#pragma unroll
        for (int off = RC; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
        if (lane < RC) s_ml[warp * RC + lane] = make_float2(ref, l);
#pragma unroll
        for (int r = 0; r < RC; r++) {
            float4 o;
            unpair2(acc[r][0], o.x, o.y);
            unpair2(acc[r][1], o.z, o.w);
            if (H == 2) {
                o.x += __shfl_xor_sync(0xffffffffu, o.x, 16); o.y += __shfl_xor_sync(0xffffffffu, o.y, 16);
                o.z += __shfl_xor_sync(0xffffffffu, o.z, 16); o.w += __shfl_xor_sync(0xffffffffu, o.w, 16);
            }
            if (sub == 0) *reinterpret_cast<float4 *>(s_acc + (warp * RC + r) * D + c * 4) = o;
        }
        __syncthreads();
        constexpr int W = D + 4;
        float *rec = sg.whole ? nullptr : p.recs + ((int64_t)blockIdx.x * 2 + sg.slot) * a.rec_rows * W;
        for (int e = tid; e < R * (D / 4); e += THREADS) {
            const int r = e / (D / 4), col = e % (D / 4) * 4;
            float M = kUnset, L = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) M = fmaxf(M, s_ml[w * RC + r].x);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float2 ml = s_ml[w * RC + r];
                const float f = ml.y != 0.f ? ex2(ml.x - M) : 0.f;
                L += ml.y * f;
                const float4 x = *reinterpret_cast<const float4 *>(s_acc + (w * RC + r) * D + col);
                o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y); o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
            }
            const float inv = inverse_sum(L);
            o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
            const int64_t orow = tree_out_row(p, sg.b, sg.kvh, r);
            const float m = M == kUnset ? -INFINITY : M;
            if (rec) {
                *reinterpret_cast<float4 *>(rec + r * W + col) = o;
                if (col == 0) {
                    *reinterpret_cast<float4 *>(rec + r * W + D) = make_float4(m * kLn2, L, 0.f, 0.f);
                    mark_cut(p, orow);
                }
            } else {
                store_row4<D>(p, orow, col, o);
                if (col == 0) store_row_stats<D>(p, orow, m, L);
            }
        }
    }
}

template <int D, int RC>
cudaError_t launch_narrow(const TreeParams &p, TcArgs &a, cudaStream_t st) {
    constexpr size_t smem = (RC * D + kWarps * RC * D + kWarps * warp_rows<D>() * RC) * sizeof(float) + kWarps * RC * sizeof(float2);
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !ready[dev])) {
        e = cudaFuncSetAttribute(tree_f32_narrow_kernel<D, RC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess && dev < 64) ready[dev] = true;
    }
    if (e == cudaSuccess) e = launch_dependent(tree_f32_narrow_kernel<D, RC>, dim3(sm_count()), kWarps * 32, smem, st, p, a);
    if (e != cudaSuccess) return e;
    FinishArgs f = {};
    f.tc = a; f.rpt = kNarrowRpt; f.tile = narrow_tile<D>(); f.workers = sm_count();
    return launch_finish<D>(p, f, st);
}

// ------------------------------------------------------------------------------------------------ many query rows
template <int D> constexpr int tiled_bn() { return D == 64 ? 64 : 32; }
template <int D, int TI> constexpr size_t tiled_smem() {
    return ((size_t)(16 * TI + 2 * tiled_bn<D>()) * (D + 4) + (size_t)16 * TI * (tiled_bn<D>() + 4)) * sizeof(float);
}

// Thread (rg, cg) of the 16 x 8 threads takes query rows rg + 16 i, cached rows cg + 8 j and output columns cg * 4 + 32 u: with rows
// padded by 4 floats those strides keep the 16-byte reads of a quarter-warp on different banks.
template <int D, int TI>
__global__ void __launch_bounds__(128) tree_f32_tiled_kernel(TreeParams p) {
    constexpr int TM = 16 * TI, BN = tiled_bn<D>(), LD = D + 4, LP = BN + 4, NJ = BN / 8, NU = D / 32;
    extern __shared__ __align__(16) float sm[];
    float *s_q = sm, *s_k = s_q + TM * LD, *s_v = s_k + BN * LD, *s_p = s_v + BN * LD;
    launch_dependents();
    grid_dependency_wait();
    const int chunk = blockIdx.x, b = blockIdx.z;
    const int q_tiles = (p.n * p.G + TM - 1) / TM;
    const int kvh = blockIdx.y / q_tiles, q0 = (blockIdx.y % q_tiles) * TM;
    const int len = tree_committed(p, b), total = len + tree_drafts(p, b, len);
    const int R = tree_tokens(p, b) * p.G;                 // live query rows
    if (q0 >= R) return;
    const int n_chunks = total <= p.chunk_rows ? 1 : (total + p.chunk_rows - 1) / p.chunk_rows;
    if (chunk >= n_chunks) return;
    const int r_begin = chunk * p.chunk_rows, r_end = min(total, r_begin + p.chunk_rows);
    const int tid = threadIdx.x, rg = tid >> 3, cg = tid & 7;

    for (int x = tid; x < TM * (D / 4); x += 128) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (q0 + r < R) {
            const int64_t at = tree_out_row(p, b, kvh, q0 + r) * D + d;
            if (p.q_dtype == NIMLLM_F32) {
                v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p.q) + at);
            } else {
                const uint2 u = *reinterpret_cast<const uint2 *>(reinterpret_cast<const __nv_bfloat16 *>(p.q) + at);
                v = make_float4(bf16lo(u.x), bf16hi(u.x), bf16lo(u.y), bf16hi(u.y));
            }
        }
        *reinterpret_cast<float4 *>(s_q + r * LD + d) = v;
    }
    float m[TI], l[TI];
    uint64_t o[TI][NU * 2];
#pragma unroll
    for (int i = 0; i < TI; i++) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int u = 0; u < NU * 2; u++) o[i][u] = 0ull;
    }
    const float *kg = reinterpret_cast<const float *>(p.k), *vg = reinterpret_cast<const float *>(p.v);
    for (int r0 = r_begin; r0 < r_end; r0 += BN) {
        __syncthreads();                                   // the tile before has been used
        // rows past the chunk and rows without a page are zeros
#pragma unroll 4
        for (int x = tid; x < BN * (D / 4); x += 128) {
            const int r = x / (D / 4), d = x % (D / 4) * 4;
            const int64_t at = r0 + r < r_end ? cache_row(p.rows, b, kvh, r0 + r) : -1;
            const uint32_t dk = (uint32_t)__cvta_generic_to_shared(s_k + r * LD + d), dv = (uint32_t)__cvta_generic_to_shared(s_v + r * LD + d);
            cp_async16(dk, kg + (at >= 0 ? at + d : 0), at >= 0 ? 16 : 0);
            cp_async16(dv, vg + (at >= 0 ? at + d : 0), at >= 0 ? 16 : 0);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        uint64_t s[TI][NJ];
#pragma unroll
        for (int i = 0; i < TI; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++) s[i][j] = 0ull;
#pragma unroll 2
        for (int d = 0; d < D; d += 4) {
            float4 qf[TI], kf[NJ];
#pragma unroll
            for (int i = 0; i < TI; i++) qf[i] = *reinterpret_cast<const float4 *>(s_q + (rg + 16 * i) * LD + d);
#pragma unroll
            for (int j = 0; j < NJ; j++) kf[j] = *reinterpret_cast<const float4 *>(s_k + (cg + 8 * j) * LD + d);
#pragma unroll
            for (int i = 0; i < TI; i++)
#pragma unroll
                for (int j = 0; j < NJ; j++)
                    s[i][j] = fma2(pair2(qf[i].z, qf[i].w), pair2(kf[j].z, kf[j].w), fma2(pair2(qf[i].x, qf[i].y), pair2(kf[j].x, kf[j].y), s[i][j]));
        }
        const bool tail = r0 + BN > len || r0 + BN > r_end || p.rows.table;      // rows that not every token attends, or no rows
#pragma unroll
        for (int i = 0; i < TI; i++) {
            const int qr = q0 + rg + 16 * i, token = qr / p.G;
            float x[NJ], mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int r = r0 + cg + 8 * j;
                float e, od;
                unpair2(s[i][j], e, od);
                x[j] = (e + od) * p.scale_log2e;
                if (p.raw && qr < R && r < r_end) p.raw[((int64_t)b * p.Hq + kvh * p.G + qr) * p.raw_ld + r] = x[j];
                if (tail) {
                    bool see = r < r_end && qr < R;
                    if (see && r >= len) see = tree_sees(p, b, token, r - len);
                    if (see && p.rows.table) see = cache_row(p.rows, b, kvh, r) >= 0;
                    if (!see) x[j] = -INFINITY;
                }
                mx = fmaxf(mx, x[j]);
            }
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float m_new = fmaxf(m[i], mx), safe = m_new == -INFINITY ? 0.f : m_new;
            const float corr = ex2(m[i] - safe);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const float w = ex2(x[j] - safe);
                sum += w;
                s_p[(rg + 16 * i) * LP + cg + 8 * j] = w;
            }
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            l[i] = l[i] * corr + sum;
            m[i] = m_new;
#pragma unroll
            for (int u = 0; u < NU * 2; u++) o[i][u] = mul2(o[i][u], pair2(corr, corr));
        }
        __syncwarp();                                      // a row's weights are written and read by the same 8 lanes
#pragma unroll 2
        for (int j = 0; j < BN; j += 4) {
            float4 pf[TI];
#pragma unroll
            for (int i = 0; i < TI; i++) pf[i] = *reinterpret_cast<const float4 *>(s_p + (rg + 16 * i) * LP + j);
#pragma unroll
            for (int jj = 0; jj < 4; jj++) {
                float4 vf[NU];
#pragma unroll
                for (int u = 0; u < NU; u++) vf[u] = *reinterpret_cast<const float4 *>(s_v + (j + jj) * LD + cg * 4 + 32 * u);
#pragma unroll
                for (int i = 0; i < TI; i++) {
                    const float w = jj == 0 ? pf[i].x : jj == 1 ? pf[i].y : jj == 2 ? pf[i].z : pf[i].w;
                    const uint64_t ww = pair2(w, w);
#pragma unroll
                    for (int u = 0; u < NU; u++) {
                        o[i][2 * u] = fma2(ww, pair2(vf[u].x, vf[u].y), o[i][2 * u]);
                        o[i][2 * u + 1] = fma2(ww, pair2(vf[u].z, vf[u].w), o[i][2 * u + 1]);
                    }
                }
            }
        }
        __syncwarp();                                      // before the next tile's weights overwrite these
    }
    constexpr int W = D + 4;
#pragma unroll
    for (int i = 0; i < TI; i++) {
        const int qr = q0 + rg + 16 * i;
        if (qr >= R) continue;
        const float inv = inverse_sum(l[i]);
        const int64_t orow = tree_out_row(p, b, kvh, qr);
        float *rec = n_chunks > 1 ? p.recs + ((int64_t)chunk * p.B * p.n * p.Hq + orow) * W : nullptr;
#pragma unroll
        for (int u = 0; u < NU; u++) {
            float4 v;
            unpair2(o[i][2 * u], v.x, v.y);
            unpair2(o[i][2 * u + 1], v.z, v.w);
            v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
            if (rec) *reinterpret_cast<float4 *>(rec + cg * 4 + 32 * u) = v;
            else store_row4<D>(p, orow, cg * 4 + 32 * u, v);
        }
        if (cg == 0) {
            if (rec) {
                *reinterpret_cast<float4 *>(rec + D) = make_float4(m[i] * kLn2, l[i], 0.f, 0.f);
                mark_cut(p, orow);
            } else {
                store_row_stats<D>(p, orow, m[i], l[i]);
            }
        }
    }
}

template <int D, int TI>
cudaError_t launch_tiled(TreeParams &p, int max_total, cudaStream_t st) {
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !ready[dev])) {
        e = cudaFuncSetAttribute(tree_f32_tiled_kernel<D, TI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tiled_smem<D, TI>());
        if (e == cudaSuccess && dev < 64) ready[dev] = true;
    }
    const int q_tiles = (p.n * p.G + 16 * TI - 1) / (16 * TI);
    p.max_chunks = (int)(((int64_t)max_total + p.chunk_rows - 1) / p.chunk_rows);
    if (p.max_chunks < 1) p.max_chunks = 1;
    if (e == cudaSuccess) e = launch_dependent(tree_f32_tiled_kernel<D, TI>, dim3(p.max_chunks, p.Hkv * q_tiles, p.B), 128, tiled_smem<D, TI>(), st, p);
    FinishArgs f = {};
    return e == cudaSuccess ? launch_finish<D>(p, f, st) : e;
}

// 8 sequences of 2 - 4 K rows, heads of 128, streamed and tiled: 4 rows 46 and 173 us, 8 rows 56 and 173, 16 rows 88 and 174
bool narrow_rows(int R) { return R <= kNarrowRpt; }
// the same with tiles of 32 and of 64 query rows: 32 rows 177 and 219 us, 48 rows 327 and 224, 64 rows 328 and 232
int tile_rows(int R) { return R <= 32 ? 32 : 64; }

// rows of a chunk: enough CTAs for four on every SM, whole tiles, and no more pieces of a row than a block joins
int chunk_of(int batch, int R, int n_kv_head, int head_dim, int max_total) {
    const int bn = head_dim == 64 ? tiled_bn<64>() : tiled_bn<128>();
    const int64_t tiles = (int64_t)batch * n_kv_head * ((R + tile_rows(R) - 1) / tile_rows(R));
    int64_t c = (tiles * max_total + 4 * sm_count() - 1) / (4 * sm_count());
    const int64_t least = ((int64_t)max_total + kMaxPieces - 1) / kMaxPieces;
    c = c < least ? least : c;
    c = (c + bn - 1) / bn * bn;
    return (int)(c < bn ? bn : (c > (1 << 30) ? 1 << 30 : c));
}

template <int D> cudaError_t launch_d(TreeParams &p, void *workspace, int max_total, cudaStream_t st) {
    const int R = p.n * p.G;
    p.recs = (float *)workspace;
    if (narrow_rows(R)) {
        TcArgs a = {};
        a.rec_rows = kNarrowRpt;
        a.starts = (int4 *)((unsigned char *)workspace + (size_t)sm_count() * 2 * kNarrowRpt * rec_stride(D) * sizeof(float));
        a.cum = (int64_t *)(a.starts + sm_count());
        return R <= 4 ? launch_narrow<D, 4>(p, a, st) : (R <= 8 ? launch_narrow<D, 8>(p, a, st) : launch_narrow<D, 16>(p, a, st));
    }
    p.chunk_rows = chunk_of(p.B, R, p.Hkv, D, max_total);
    return tile_rows(R) == 32 ? launch_tiled<D, 2>(p, max_total, st) : launch_tiled<D, 4>(p, max_total, st);
}

}  // namespace
}  // namespace treetc

size_t tree_f32_workspace_bytes(int batch, int n, int n_head, int n_kv_head, int head_dim, int max_total) {
    using namespace treetc;
    const int R = n * (n_head / n_kv_head);
    if (narrow_rows(R))
        return (size_t)sm_count() * (2 * kNarrowRpt * rec_stride(head_dim) * sizeof(float) + sizeof(int4)) + ((size_t)batch + 1) * sizeof(int64_t);
    const int chunk = chunk_of(batch, R, n_kv_head, head_dim, max_total);
    const int64_t chunks = ((int64_t)max_total + chunk - 1) / chunk;
    return chunks <= 1 ? 0 : (size_t)chunks * batch * n * n_head * rec_stride(head_dim) * sizeof(float);
}

int launch_tree_f32(const char *who, TreeParams &p, int head_dim, int max_total, void *workspace, cudaStream_t st) {
    const cudaError_t e = head_dim == 64 ? treetc::launch_d<64>(p, workspace, max_total, st) : treetc::launch_d<128>(p, workspace, max_total, st);
    if (e != cudaSuccess) return fail(NIMLLM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return NIMLLM_OK;
}

}  // namespace nimllm
