// rope_at.cu -- rotation of q and k at a position of its own per token, with the append of the rows to the cache.
//
// For the pairs (x0, x1) of the first rot_dim columns of a head -- (f, f + rot_dim/2) in the half layout, (2f, 2f + 1) in
// the interleaved one -- and the table row of the token's position:
//     y0 = x0 c - x1 s,  y1 = x0 s + x1 c           gradient: the same with -s (the transposed matrix)
// The other columns pass.  rope_append.cu ties the row of a token to its position; here both are given, because the tokens
// of a drafted tree share positions and the rows of an evicted cache have left theirs.
//
// HBM-bound elementwise work.  A thread moves pairs of vectors of V elements (16 bytes each where the head allows: V = 8 for
// bf16, 4 for fp32; else 4), all of them rotated or all of them passed.
//
// Measured (graph replay): gradient of 4 x 8192 tokens, 32 + 8 heads of 128, bf16: 127 us = 5.3 TB/s; 61 trees of 24 tokens into pages:
// 10.3 us (5.6 us of memory time, the rest is launch and three loads in a row, pos, tables and the page entry); one token 4.1 us.
#include <math.h>

#include "cache_rows.cuh"

namespace nimllm {

namespace {

struct RopeAtParams {
    const void *q, *k, *v;
    void *q_out, *k_out;
    void *k_cache, *v_cache;
    const float *cos_tab, *sin_tab;
    const int32_t *pos, *row0;
    int first_row;
    CacheRows rows;
    int B, n, Hq, Hkv, D, rot;
    int table_rows;
    float sign;
    int zero_padding;        // gradient: tokens without a position get 0 (the forward did not read them)
    int n_q, n_k, n_v;       // slots: query heads, K heads, V heads
    int items, lanes, per_token;   // pairs of vectors of a head, threads of a token that have the same one, threads of a token
};

template <typename T, int V> __device__ __forceinline__ void load_vec(const T *p, float *f) {
    static_assert(sizeof(T) == 4 && V == 4, "table entries");
    const float4 x = *reinterpret_cast<const float4 *>(p);
    f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
}
template <typename T, int V> struct Unpack {
    __device__ static void go(const uint4 &u, float *f) {
        if constexpr (sizeof(T) == 4) Elem<float>::unpack(u, f);
        else if constexpr (V == 8) Elem<__nv_bfloat16>::unpack(u, f);
        else { f[0] = bf16lo(u.x); f[1] = bf16hi(u.x); f[2] = bf16lo(u.y); f[3] = bf16hi(u.y); }
    }
};
template <typename T, int V> __device__ __forceinline__ void store_vec(T *p, const float *f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    } else if constexpr (V == 8) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    } else {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
    }
}

// Slots 0.. are the query heads, then the K heads, then the V heads.  A thread has one pair of vectors of a token and takes kHeads of
// the token's slots, `lanes` apart: the token's row, position and table entries are fetched and the places worked out once for all of
// them, and the loads of all of them are in flight together.
template <typename ActT, typename CacheT, int V, bool INTERLEAVED, int HEADS>
__global__ void __launch_bounds__(256) rope_at_kernel(RopeAtParams p) {
    launch_dependents();
    grid_dependency_wait();
    const int idx = blockIdx.x * 256 + threadIdx.x;        // < 2^31: checked on the host
    const int token = idx / p.per_token;
    if (token >= p.B * p.n) return;
    const int in = idx - token * p.per_token;
    const int first = in / p.items, item = in - first * p.items;
    const int b = token / p.n, t = token - b * p.n;
    const int slots = p.n_q + p.n_k + p.n_v;

    const int row = (p.row0 ? p.row0[b] : p.first_row) + t;
    const int pos = p.pos ? p.pos[token] : row;
    const bool live = pos >= 0 && (p.rot == 0 || pos < p.table_rows);
    // the first elements of the two vectors
    const bool turned = item * 2 * V < p.rot;
    const int half = p.rot / 2;
    const int e0 = turned && !INTERLEAVED ? item * V : item * 2 * V;
    const int e1 = turned && !INTERLEAVED ? e0 + half : e0 + V;

    uint4 x0[HEADS], x1[HEADS];                            // V elements each, as they lie in memory
    if (live) {
#pragma unroll
        for (int h = 0; h < HEADS; h++) {
            const int slot = first + h * p.lanes;
            if (slot < slots) {
                const bool is_q = slot < p.n_q, is_v = slot >= p.n_q + p.n_k;
                const int head = is_q ? slot : (is_v ? slot - p.n_q - p.n_k : slot - p.n_q);
                const ActT *x = reinterpret_cast<const ActT *>(is_q ? p.q : (is_v ? p.v : p.k)) + ((int64_t)token * (is_q ? p.Hq : p.Hkv) + head) * p.D;
                if constexpr (sizeof(ActT) * V == 16) {
                    x0[h] = *reinterpret_cast<const uint4 *>(x + e0);
                    x1[h] = *reinterpret_cast<const uint4 *>(x + e1);
                } else {
                    const uint2 y0 = *reinterpret_cast<const uint2 *>(x + e0), y1 = *reinterpret_cast<const uint2 *>(x + e1);
                    x0[h] = make_uint4(y0.x, y0.y, 0, 0);
                    x1[h] = make_uint4(y1.x, y1.y, 0, 0);
                }
            }
        }
    }
    float c[V], s[V];
    if (live && turned) {
        const float *ct = p.cos_tab + (int64_t)pos * half + item * V, *st = p.sin_tab + (int64_t)pos * half + item * V;
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            load_vec<float, 4>(ct + i, c + i);
            load_vec<float, 4>(st + i, s + i);
        }
#pragma unroll
        for (int i = 0; i < V; i++) s[i] *= p.sign;
    }
    const bool in_cache = p.k_cache && live && row >= 0 && row < p.rows.cap;
#pragma unroll
    for (int h = 0; h < HEADS; h++) {
        const int slot = first + h * p.lanes;
        if (slot >= slots) break;
        const bool is_q = slot < p.n_q, is_v = slot >= p.n_q + p.n_k;
        const int head = is_q ? slot : (is_v ? slot - p.n_q - p.n_k : slot - p.n_q);
        ActT *out = reinterpret_cast<ActT *>(is_q ? p.q_out : (is_v ? nullptr : p.k_out));
        if (out) out += ((int64_t)token * (is_q ? p.Hq : p.Hkv) + head) * p.D;
        float f0[V], f1[V];
        if (live) {
            Unpack<ActT, V>::go(x0[h], f0);
            Unpack<ActT, V>::go(x1[h], f1);
            if (turned && !is_v) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    // pair i: (f0[i], f1[i]) in the half layout, two neighbours of the 2V elements in the interleaved one
                    float &u = INTERLEAVED ? (2 * i < V ? f0[(2 * i) % V] : f1[(2 * i) % V]) : f0[i];
                    float &w = INTERLEAVED ? (2 * i < V ? f0[(2 * i + 1) % V] : f1[(2 * i + 1) % V]) : f1[i];
                    const float y0 = u * c[i] - w * s[i], y1 = u * s[i] + w * c[i];
                    u = y0;
                    w = y1;
                }
            }
        } else {
            if (!p.zero_padding) continue;
#pragma unroll
            for (int i = 0; i < V; i++) f0[i] = f1[i] = 0.f;
        }
        if (out) {
            store_vec<ActT, V>(out + e0, f0);
            store_vec<ActT, V>(out + e1, f1);
        }
        if (!is_q && in_cache) {
            const int64_t at = cache_row(p.rows, b, head, row);
            if (at >= 0) {
                CacheT *dst = reinterpret_cast<CacheT *>(is_v ? p.v_cache : p.k_cache) + at;
                store_vec<CacheT, V>(dst + e0, f0);
                store_vec<CacheT, V>(dst + e1, f1);
            }
        }
    }
}

template <typename ActT, typename CacheT, int V, int HEADS>
cudaError_t launch_heads(RopeAtParams p, int layout, cudaStream_t st) {
    const int slots = p.n_q + p.n_k + p.n_v;
    p.items = p.D / (2 * V);
    p.lanes = (slots + HEADS - 1) / HEADS;
    p.per_token = p.lanes * p.items;
    const int64_t threads = (int64_t)p.B * p.n * p.per_token;
    if (threads > 0x7fffff00) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)((threads + 255) / 256));
    return layout == NIMLLM_ROPE_INTERLEAVED ? launch_dependent(rope_at_kernel<ActT, CacheT, V, true, HEADS>, grid, 256, 0, st, p)
                                             : launch_dependent(rope_at_kernel<ActT, CacheT, V, false, HEADS>, grid, 256, 0, st, p);
}
template <typename ActT, typename CacheT, int V>
cudaError_t launch_v(const RopeAtParams &p, int layout, cudaStream_t st) {
    // four heads a thread share the table's loads once that still leaves every SM full of threads: the gradient of 4 x 8192 tokens
    // takes 126.9 us, 129.4 with one head a thread; a decode step of 200 tokens 4.4 us with one, 6.4 with four
    const int64_t threads = (int64_t)p.B * p.n * (p.n_q + p.n_k + p.n_v) * (p.D / (2 * V));
    return threads >= (int64_t)sm_count() * 2048 * 4 ? launch_heads<ActT, CacheT, V, 4>(p, layout, st) : launch_heads<ActT, CacheT, V, 1>(p, layout, st);
}

int launch_rope_at(const char *who, const RopeAtParams &p, int layout, int act_dtype, int cache_dtype, cudaStream_t st) {
    if ((int64_t)p.B * p.n * (p.n_q + p.n_k + p.n_v) == 0) return NIMLLM_OK;
    cudaError_t e;
    if (act_dtype == NIMLLM_F32) {
        e = cache_dtype == NIMLLM_F32 ? launch_v<float, float, 4>(p, layout, st) : launch_v<float, __nv_bfloat16, 4>(p, layout, st);
    } else if (p.D % 16 == 0 && p.rot % 16 == 0) {
        e = cache_dtype == NIMLLM_F32 ? launch_v<__nv_bfloat16, float, 8>(p, layout, st) : launch_v<__nv_bfloat16, __nv_bfloat16, 8>(p, layout, st);
    } else {
        e = cache_dtype == NIMLLM_F32 ? launch_v<__nv_bfloat16, float, 4>(p, layout, st) : launch_v<__nv_bfloat16, __nv_bfloat16, 4>(p, layout, st);
    }
    if (e != cudaSuccess) return fail(NIMLLM_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return NIMLLM_OK;
}

int check_rotation(const char *who, int act_dtype, const float *cos_tab, const float *sin_tab, int rot_dim, int layout, int table_rows,
                   int batch, int n, int n_head, int n_kv_head, int head_dim) {
    if ((int64_t)batch * n > 0x7fffffff) return fail(NIMLLM_ERR_UNSUPPORTED, "%s: %d x %d tokens", who, batch, n);
    if (batch < 0 || n < 0 || n_head < 0 || n_kv_head < 0 || head_dim <= 0 || head_dim % 8 != 0)
        return fail(NIMLLM_ERR_ARG, "%s: bad shape B=%d n=%d Hq=%d Hkv=%d D=%d", who, batch, n, n_head, n_kv_head, head_dim);
    if (!dtype_ok(act_dtype)) return fail(NIMLLM_ERR_ARG, "%s: unknown dtype", who);
    if ((cos_tab == nullptr) != (sin_tab == nullptr)) return fail(NIMLLM_ERR_ARG, "%s: give both RoPE tables or neither", who);
    if (layout != NIMLLM_ROPE_HALF && layout != NIMLLM_ROPE_INTERLEAVED) return fail(NIMLLM_ERR_ARG, "%s: unknown layout %d", who, layout);
    if (cos_tab && (rot_dim <= 0 || rot_dim % 8 != 0 || rot_dim > head_dim || table_rows <= 0))
        return fail(NIMLLM_ERR_ARG, "%s: rot_dim %d must be a multiple of 8 up to head_dim %d, table_rows %d > 0", who, rot_dim, head_dim, table_rows);
    if (((uintptr_t)cos_tab | (uintptr_t)sin_tab) & 15) return fail(NIMLLM_ERR_ARG, "%s: the tables must be 16-byte aligned", who);
    return NIMLLM_OK;
}

int rope_append_at(const char *who, const CacheRows *rows, const void *q, void *q_out, int n_head, const void *k_new, void *k_out,
                   const void *v_new, int act_dtype, const float *cos_tab, const float *sin_tab, int rot_dim, int layout, int table_rows,
                   const int32_t *pos, const int32_t *row0, int first_row, void *k_cache, void *v_cache, int cache_dtype, int batch,
                   int n, int n_kv_head, int head_dim, void *stream) {
    if (int rc = check_rotation(who, act_dtype, cos_tab, sin_tab, rot_dim, layout, table_rows, batch, n, n_head, n_kv_head, head_dim)) return rc;
    if ((q == nullptr) != (q_out == nullptr)) return fail(NIMLLM_ERR_ARG, "%s: give q and q_out or neither", who);
    if ((k_out && !k_new) || (k_cache && (!k_new || !v_new))) return fail(NIMLLM_ERR_ARG, "%s: null k_new / v_new", who);
    if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k_new | (uintptr_t)k_out | (uintptr_t)v_new) & 15)
        return fail(NIMLLM_ERR_ARG, "%s: q, k_new, v_new and the outputs must be 16-byte aligned", who);
    RopeAtParams p = {};
    p.q = q; p.q_out = q_out; p.k = k_new; p.k_out = k_out; p.v = v_new;
    p.k_cache = k_cache; p.v_cache = v_cache; p.cos_tab = cos_tab; p.sin_tab = sin_tab;
    p.pos = pos; p.row0 = row0; p.first_row = first_row;
    if (rows) p.rows = *rows;
    p.B = batch; p.n = n; p.Hq = n_head; p.Hkv = n_kv_head; p.D = head_dim; p.rot = cos_tab ? rot_dim : 0;
    p.table_rows = table_rows; p.sign = 1.f; p.zero_padding = 0;
    p.n_q = q ? n_head : 0; p.n_k = (k_out || k_cache) ? n_kv_head : 0; p.n_v = k_cache ? n_kv_head : 0;
    return launch_rope_at(who, p, layout, act_dtype, k_cache ? cache_dtype : act_dtype, (cudaStream_t)stream);
}

}  // namespace

}  // namespace nimllm

using namespace nimllm;

extern "C" {

int nimllm_rope_tables_scaled_host(float *cos_tab, float *sin_tab, int max_pos, int rot_dim, double base, int kind, double factor,
                                   double low, double high, int orig_len, double gain) {
    if (!cos_tab || !sin_tab || max_pos < 0 || rot_dim <= 0 || (rot_dim & 1) || !(base > 0))
        return fail(NIMLLM_ERR_ARG, "rope_tables_scaled_host: bad arguments");
    if (kind < NIMLLM_ROPE_SCALE_NONE || kind > NIMLLM_ROPE_SCALE_RAMP)
        return fail(NIMLLM_ERR_ARG, "rope_tables_scaled_host: unknown kind %d", kind);
    if (kind != NIMLLM_ROPE_SCALE_NONE && !(factor > 0))
        return fail(NIMLLM_ERR_ARG, "rope_tables_scaled_host: factor must be positive");
    if (kind == NIMLLM_ROPE_SCALE_BASE && rot_dim <= 2)
        return fail(NIMLLM_ERR_ARG, "rope_tables_scaled_host: a stretched base needs rot_dim > 2");
    if (kind == NIMLLM_ROPE_SCALE_RAMP && (!(high > low) || orig_len <= 0))
        return fail(NIMLLM_ERR_ARG, "rope_tables_scaled_host: the ramp needs high > low and orig_len > 0");
    if (kind == NIMLLM_ROPE_SCALE_BASE) base *= pow(factor, (double)rot_dim / (rot_dim - 2));
    const int half = rot_dim / 2;
    for (int f = 0; f < half; f++) {
        double w = pow(base, -2.0 * f / rot_dim);
        if (kind == NIMLLM_ROPE_SCALE_LINEAR) w /= factor;
        if (kind == NIMLLM_ROPE_SCALE_RAMP) {
            // turns that the frequency makes over the trained length: few -> interpolated, many -> as trained
            const double turns = orig_len * w / (2 * M_PI);
            double keep = (turns - low) / (high - low);
            keep = keep < 0 ? 0 : (keep > 1 ? 1 : keep);
            w = keep * w + (1 - keep) * w / factor;
        }
        // 64 bits up to the table: at position 10^5 an angle in 32 bits is 4e-3 off
        for (int pos = 0; pos < max_pos; pos++) {
            cos_tab[(size_t)pos * half + f] = (float)(gain * cos(pos * w));
            sin_tab[(size_t)pos * half + f] = (float)(gain * sin(pos * w));
        }
    }
    return NIMLLM_OK;
}

int nimllm_rope_append_at(const void *q, void *q_out, int n_head, const void *k_new, void *k_out, const void *v_new, int act_dtype,
                          const float *rope_cos, const float *rope_sin, int rot_dim, int layout, int table_rows, const int32_t *pos,
                          const int32_t *row0, int first_row, void *k_cache, void *v_cache, int cache_dtype, const int64_t *kv_off,
                          int64_t seq_stride, int64_t head_stride, int max_seq, int batch, int n, int n_kv_head, int head_dim,
                          void *stream) {
    const char *who = "rope_append_at";
    if ((k_cache == nullptr) != (v_cache == nullptr)) return fail(NIMLLM_ERR_ARG, "%s: give both cache pointers or neither", who);
    CacheRows rows;
    if (k_cache)
        if (int rc = contiguous_rows(rows, who, k_cache, v_cache, cache_dtype, kv_off, seq_stride, head_stride, max_seq, head_dim)) return rc;
    return rope_append_at(who, k_cache ? &rows : nullptr, q, q_out, n_head, k_new, k_out, v_new, act_dtype, rope_cos, rope_sin, rot_dim,
                          layout, table_rows, pos, row0, first_row, k_cache, v_cache, cache_dtype, batch, n, n_kv_head, head_dim, stream);
}

int nimllm_rope_append_at_paged(const void *q, void *q_out, int n_head, const void *k_new, void *k_out, const void *v_new, int act_dtype,
                                const float *rope_cos, const float *rope_sin, int rot_dim, int layout, int table_rows,
                                const int32_t *pos, const int32_t *row0, int first_row, void *k_pages, void *v_pages, int cache_dtype,
                                const int32_t *page_table, int max_pages, int page_rows, int n_pages, int batch, int n, int n_kv_head,
                                int head_dim, void *stream) {
    const char *who = "rope_append_at_paged";
    CacheRows rows;
    if (int rc = paged_rows(rows, who, k_pages, v_pages, cache_dtype, page_table, max_pages, page_rows, n_pages, n_kv_head, head_dim)) return rc;
    return rope_append_at(who, &rows, q, q_out, n_head, k_new, k_out, v_new, act_dtype, rope_cos, rope_sin, rot_dim, layout, table_rows, pos,
                          row0, first_row, k_pages, v_pages, cache_dtype, batch, n, n_kv_head, head_dim, stream);
}

int nimllm_rope_at_bwd(const void *dq_rot, void *dq, int n_head, const void *dk_rot, void *dk, int dtype, const float *rope_cos,
                       const float *rope_sin, int rot_dim, int layout, int table_rows, const int32_t *pos, int pos0, int batch, int n,
                       int n_kv_head, int head_dim, void *stream) {
    const char *who = "rope_at_bwd";
    if (!rope_cos || !rope_sin) return fail(NIMLLM_ERR_ARG, "%s: null RoPE tables", who);
    if (int rc = check_rotation(who, dtype, rope_cos, rope_sin, rot_dim, layout, table_rows, batch, n, n_head, n_kv_head, head_dim)) return rc;
    if ((dq_rot == nullptr) != (dq == nullptr) || (dk_rot == nullptr) != (dk == nullptr) || (!dq && !dk))
        return fail(NIMLLM_ERR_ARG, "%s: give each gradient with its output", who);
    if (((uintptr_t)dq_rot | (uintptr_t)dq | (uintptr_t)dk_rot | (uintptr_t)dk) & 15)
        return fail(NIMLLM_ERR_ARG, "%s: the gradients must be 16-byte aligned", who);
    RopeAtParams p = {};
    p.q = dq_rot; p.q_out = dq; p.k = dk_rot; p.k_out = dk; p.cos_tab = rope_cos; p.sin_tab = rope_sin;
    p.pos = pos; p.first_row = pos0; p.B = batch; p.n = n; p.Hq = n_head; p.Hkv = n_kv_head; p.D = head_dim; p.rot = rot_dim;
    p.table_rows = table_rows; p.sign = -1.f; p.zero_padding = 1;
    p.n_q = dq ? n_head : 0; p.n_k = dk ? n_kv_head : 0; p.n_v = 0;
    return launch_rope_at(who, p, layout, dtype, dtype, (cudaStream_t)stream);
}

}  // extern "C"
