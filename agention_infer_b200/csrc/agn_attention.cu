// Attention of query rows over the KV cache that agn_kv_write_f32 fills.
//
//   out[t, h, :] = sum_j p_j V[s, j, h / G, :],  p = softmax_j(scale * q[t, h, :] . K[s, j, h / G, :]),  j = 0 .. pos[t]
//
// (`launch_attention`, src/ops/wgpu_backend/resident.rs:551-565; kernels `attention_scores`, `attention_softmax`,
// `attention_output` and their `_q8_0` forms, src/ops/kernels_wgpu.rs:749-980; CPU `attention_into`,
// src/model/llama/cpu_path.rs:160-192).  G = n_q_heads / n_kv_heads query heads share a KV head.
#include <math.h>

#include "agn_common.cuh"

namespace {

struct AttnArgs {
    const void *q;
    void *out;
    const unsigned char *k_cache, *v_cache;
    const int32_t *pos, *seq;
    int64_t T, n_seqs, max_seq;
    int n_q, n_kv, hd, pos_start, bytes_per_token;
    float scale;
    uint32_t *flags;
};

// Visible slots of row t and the first byte of its sequence's cache; 0 slots for an empty row or one outside the cache.
__device__ __forceinline__ int attn_row(const AttnArgs &a, int64_t t, int64_t *seq_off) {
    const int64_t p = a.pos ? (int64_t)a.pos[t] : (int64_t)a.pos_start + t;
    const int64_t s = a.seq ? (int64_t)a.seq[t] : 0;
    *seq_off = 0;
    if (p < -1 || p >= a.max_seq || s < 0 || s >= a.n_seqs) {
        atomicOr(a.flags, AGN_FLAG_OOB_ATTN);
        return 0;
    }
    *seq_off = s * a.max_seq * a.bytes_per_token;
    return (int)(p + 1);
}

template <int KV> __device__ __forceinline__ float kv_value(const unsigned char *row, int i) {
    if (KV == 0) return __half2float(reinterpret_cast<const __half *>(row)[i]);
    if (KV == 1) {
        const unsigned char *b = row + (i >> 5) * 34;
        return __half2float(*reinterpret_cast<const __half *>(b)) * (float)(signed char)b[2 + (i & 31)];
    }
    const unsigned char *b = row + (i >> 5) * 36;
    return *reinterpret_cast<const float *>(b) * ((float)(int)b[4 + (i & 31)] - 128.0f);
}

// One CTA of 128 threads per (row, query head): 128 slots at a time, a slot per thread for the scores and a dimension
// (or two) per thread for the output, with the running maximum and sum of the softmax in f32.
template <typename T, int KV> __global__ void __launch_bounds__(128) attn_row_kernel(AttnArgs a) {
    agn_pdl_prologue();
    __shared__ float sq[256], sp[128], red[4];
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, kvh = h / (a.n_q / a.n_kv), tid = threadIdx.x;
    int64_t off;
    const int n = attn_row(a, t, &off);
    const int64_t qoff = (t * a.n_q + h) * a.hd;
    for (int d = tid; d < a.hd; d += 128) sq[d] = ActVec<T>::load1(static_cast<const T *>(a.q) + qoff, d) * a.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int j0 = 0; j0 < n; j0 += 128) {
        const int cnt = min(128, n - j0);
        float s = -INFINITY;
        if (tid < cnt) {
            const unsigned char *row = a.k_cache + off + (int64_t)(j0 + tid) * a.bytes_per_token;
            s = 0.0f;
            for (int d = 0; d < a.hd; d++) s = __fmaf_rn(sq[d], kv_value<KV>(row, kvh * a.hd + d), s);
        }
        const float wm = agn_warp_max(s);
        if ((tid & 31) == 0) red[tid >> 5] = wm;
        __syncthreads();
        const float mt = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), mn = fmaxf(m, mt);
        const float c = expf(m - mn);
        m = mn;
        sp[tid] = tid < cnt ? expf(s - mn) : 0.0f;
        __syncthreads();
        o0 *= c; o1 *= c; l *= c;
        for (int j = 0; j < cnt; j++) {
            const unsigned char *row = a.v_cache + off + (int64_t)(j0 + j) * a.bytes_per_token;
            l += sp[j];
            if (tid < a.hd) o0 = __fmaf_rn(sp[j], kv_value<KV>(row, kvh * a.hd + tid), o0);
            if (tid + 128 < a.hd) o1 = __fmaf_rn(sp[j], kv_value<KV>(row, kvh * a.hd + tid + 128), o1);
        }
        __syncthreads();
    }
    const float inv = n > 0 ? 1.0f / l : 0.0f;
    if (tid < a.hd) ActVec<T>::store1(static_cast<T *>(a.out) + qoff, tid, n > 0 ? o0 * inv : 0.0f);
    if (tid + 128 < a.hd) ActVec<T>::store1(static_cast<T *>(a.out) + qoff, tid + 128, n > 0 ? o1 * inv : 0.0f);
}

bool attn_shape_ok(int64_t T, int n_q, int n_kv, int hd, int64_t max_seq) {
    return T >= 0 && T <= 0x7fffffffLL && n_q > 0 && n_kv > 0 && n_q % n_kv == 0 && n_q <= 65535 && hd > 0 && hd <= 256 && hd % 32 == 0 &&
           max_seq > 0 && max_seq <= 0x7fffffffLL;
}

template <typename T>
int32_t attention_kv(agn_ctx *ctx, const T *q, T *out, int32_t kv_dtype, const void *k_cache, const void *v_cache, int64_t rows,
                     int32_t n_q, int32_t n_kv, int32_t hd, const int32_t *pos, int32_t pos_start, const int32_t *seq,
                     int64_t n_seqs, int64_t max_seq, float scale, void *workspace, size_t workspace_bytes) {
    AGN_CHECK_CTX(ctx);
    if (kv_dtype != AGN_F16 && kv_dtype != AGN_Q8_0 && kv_dtype != AGN_KV_Q8_0_WORDS)
        return agn_fail(ctx, AGN_EUNSUPPORTED_DTYPE, "attention_kv: KV dtype %d is neither f16 (1), q8_0 (8) nor q8_0 in words (1008)", kv_dtype);
    if (!attn_shape_ok(rows, n_q, n_kv, hd, max_seq) || n_seqs <= 0)
        return agn_fail(ctx, AGN_EINVAL, "attention_kv: T=%lld n_q_heads=%d n_kv_heads=%d head_dim=%d (a multiple of 32 up to 256) n_seqs=%lld "
                        "max_seq_len=%lld", (long long)rows, n_q, n_kv, hd, (long long)n_seqs, (long long)max_seq);
    if (!(scale > 0.0f) || isinf(scale)) return agn_fail(ctx, AGN_EINVAL, "attention_kv: scale=%g must be positive and finite", (double)scale);
    if (!pos && seq) return agn_fail(ctx, AGN_EINVAL, "attention_kv: seq needs pos (rows without positions are consecutive slots of one sequence)");
    if (!pos && (pos_start < 0 || (int64_t)pos_start + rows > max_seq))
        return agn_fail(ctx, AGN_EINVAL, "attention_kv: rows %d .. %lld outside the cache of %lld slots", pos_start,
                        (long long)pos_start + rows - 1, (long long)max_seq);
    if (rows == 0) return AGN_OK;
    if (!q || !out || !k_cache || !v_cache) return agn_fail(ctx, AGN_EINVAL, "attention_kv: null pointer");
    if (static_cast<const void *>(q) == out) return agn_fail(ctx, AGN_EINVAL, "attention_kv: out must not alias q");
    if (!agn_aligned16(q) || !agn_aligned16(out)) return agn_fail(ctx, AGN_EINVAL, "attention_kv: q and out must be 16-byte aligned");
    const int ca = kv_dtype == AGN_KV_Q8_0_WORDS ? 4 : 2;
    if (!agn_aligned(k_cache, ca) || !agn_aligned(v_cache, ca))
        return agn_fail(ctx, AGN_EINVAL, "attention_kv: caches must be %d-byte aligned", ca);
    AGN_CUDA(ctx, cudaSetDevice(ctx->device));
    AttnArgs a;
    a.q = q; a.out = out; a.k_cache = static_cast<const unsigned char *>(k_cache); a.v_cache = static_cast<const unsigned char *>(v_cache);
    a.pos = pos; a.seq = seq; a.T = rows; a.n_seqs = n_seqs; a.max_seq = max_seq; a.n_q = n_q; a.n_kv = n_kv; a.hd = hd; a.pos_start = pos_start;
    a.bytes_per_token = (int)agn_kv_bytes_per_token(kv_dtype, (int64_t)n_kv * hd); a.scale = scale; a.flags = ctx->d_flags;
    const dim3 grid((unsigned)rows, (unsigned)n_q);
    if (kv_dtype == AGN_F16) agn_launch(ctx, attn_row_kernel<T, 0>, grid, dim3(128), 0, a);
    else if (kv_dtype == AGN_Q8_0) agn_launch(ctx, attn_row_kernel<T, 1>, grid, dim3(128), 0, a);
    else agn_launch(ctx, attn_row_kernel<T, 2>, grid, dim3(128), 0, a);
    ctx->flags_dirty = true;
    AGN_LAUNCHED(ctx, "attention_kv");
    (void)workspace; (void)workspace_bytes;
    return AGN_OK;
}

}  // namespace

extern "C" int64_t agn_attention_kv_workspace_bytes(int64_t T, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int64_t max_seq_len,
                                                    int32_t has_pos) {
    if (!attn_shape_ok(T, n_q_heads, n_kv_heads, head_dim, max_seq_len)) return 0;
    (void)has_pos;
    return 0;
}

extern "C" int32_t agn_attention_kv_f32(agn_ctx *ctx, const float *q, float *out, int32_t kv_dtype, const void *k_cache, const void *v_cache,
                                        int64_t T, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, const int32_t *pos,
                                        int32_t pos_start, const int32_t *seq, int64_t n_seqs, int64_t max_seq_len, float scale,
                                        void *workspace, size_t workspace_bytes) {
    return attention_kv<float>(ctx, q, out, kv_dtype, k_cache, v_cache, T, n_q_heads, n_kv_heads, head_dim, pos, pos_start, seq, n_seqs,
                               max_seq_len, scale, workspace, workspace_bytes);
}

extern "C" int32_t agn_attention_kv_f16(agn_ctx *ctx, const void *q, void *out, int32_t kv_dtype, const void *k_cache, const void *v_cache,
                                        int64_t T, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, const int32_t *pos,
                                        int32_t pos_start, const int32_t *seq, int64_t n_seqs, int64_t max_seq_len, float scale,
                                        void *workspace, size_t workspace_bytes) {
    return attention_kv<__half>(ctx, static_cast<const __half *>(q), static_cast<__half *>(out), kv_dtype, k_cache, v_cache, T, n_q_heads,
                                n_kv_heads, head_dim, pos, pos_start, seq, n_seqs, max_seq_len, scale, workspace, workspace_bytes);
}
