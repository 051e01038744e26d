// The gated delta rule, the recurrence of the engine's linear-attention layers (GatedDeltaNet, src/model/llama/cpu_path.rs:397-688;
// GPU kernels src/ops/kernels_wgpu.rs:331-559).  Per value head, with a state S [head_k, head_v]:
//
//   S_t = a_t S_{t-1} + k_t d_t^T,   d_t = beta_t (v_t - a_t S_{t-1}^T k_t),   o_t = S_t^T q_t,   a_t = exp(g_t)
//
// q and k are divided by their 2-norm first (l2norm_eps >= 0) and q is multiplied by `scale`.
#include <math.h>

#include "agn_common.cuh"

namespace {

struct DeltaArgs {
    const float *q, *k, *v, *g, *beta, *state_in;
    float *state_out, *out;
    const int32_t *cu;  // n_seqs + 1 row offsets, or null: sequences of T / n_seqs rows
    int64_t T, n_seqs, q_stride, k_stride, v_stride;
    int n_k, n_v, dv;
    float scale, eps;
    uint32_t *flags;
};

// Rows [*b, *e) of sequence s.  Offsets outside [0, T] or out of order are cut and reported.
__device__ __forceinline__ void delta_rows(const DeltaArgs &a, int64_t s, int64_t *b, int64_t *e) {
    if (!a.cu) {
        const int64_t n = a.T / a.n_seqs;
        *b = s * n;
        *e = *b + n;
        return;
    }
    const int64_t b0 = a.cu[s], e0 = a.cu[s + 1];
    *b = b0 < 0 ? 0 : b0 > a.T ? a.T : b0;
    *e = e0 < *b ? *b : e0 > a.T ? a.T : e0;
    if ((*b != b0 || *e != e0) && threadIdx.x == 0) atomicOr(a.flags, AGN_FLAG_BAD_SEQLENS);
}

// Recurrent form, for few tokens a sequence: what it has to move is the state, read once and written once (HBM-bound from a few
// sequences on).  A CTA holds 32 columns of one head's state in registers: they evolve independently of the other columns, so a
// single sequence of 32 heads of 128 already gives 128 CTAs.  Thread (row group rg = 0..15, column quad c4): rows rg + 16 i.
// k^T S and q^T S are taken from the same old state in one pass (o = a q^T S + (q.k) d), so a token costs one exchange
// between the four warps.
constexpr int TB = 8;  // tokens whose q, k, v are staged at a time
template <int DK> __global__ void __launch_bounds__(128) delta_recurrent_kernel(DeltaArgs a) {
    agn_pdl_prologue();
    constexpr int R = DK / 16;
    __shared__ __align__(16) float sq[TB][DK], sk[TB][DK], sv[TB][32];
    __shared__ float sa[TB], sb[TB], sqk[TB];
    __shared__ __align__(16) float red[2][4][2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = blockIdx.x * 32, h = blockIdx.y, hk = h / (a.n_v / a.n_k);
    const int64_t s = blockIdx.z;
    int64_t b, e;
    delta_rows(a, s, &b, &e);
    const int rg = warp * 4 + (lane >> 3), c4 = (lane & 7) * 4;
    const int64_t soff = ((s * a.n_v + h) * DK + rg) * a.dv + c0 + c4;
    float4 S[R];
#pragma unroll
    for (int i = 0; i < R; i++)
        S[i] = a.state_in ? *reinterpret_cast<const float4 *>(a.state_in + soff + (int64_t)16 * i * a.dv) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int64_t t0 = b; t0 < e; t0 += TB) {
        const int cnt = (int)(e - t0 < TB ? e - t0 : TB);
        __syncthreads();
        for (int i = warp; i < cnt; i += 4) {
            const int64_t t = t0 + i;
            constexpr int V = DK / 32;
            float qv[V], kv[V], qq = 0.0f, kk = 0.0f, qk = 0.0f;
#pragma unroll
            for (int j = 0; j < V; j++) {
                qv[j] = a.q[t * a.q_stride + hk * DK + lane + 32 * j];
                kv[j] = a.k[t * a.k_stride + hk * DK + lane + 32 * j];
                qq = __fmaf_rn(qv[j], qv[j], qq);
                kk = __fmaf_rn(kv[j], kv[j], kk);
            }
            float fq = a.scale, fk = 1.0f;
            if (a.eps >= 0.0f) {
                fq *= rsqrtf(agn_warp_sum(qq) + a.eps);
                fk = rsqrtf(agn_warp_sum(kk) + a.eps);
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                qv[j] *= fq;
                kv[j] *= fk;
                qk = __fmaf_rn(qv[j], kv[j], qk);
                sq[i][lane + 32 * j] = qv[j];
                sk[i][lane + 32 * j] = kv[j];
            }
            qk = agn_warp_sum(qk);
            sv[i][lane] = a.v[t * a.v_stride + h * a.dv + c0 + lane];
            if (lane == 0) {
                sa[i] = expf(a.g[t * a.n_v + h]);
                sb[i] = a.beta[t * a.n_v + h];
                sqk[i] = qk;
            }
        }
        __syncthreads();
        for (int i = 0; i < cnt; i++) {
            float4 dk = make_float4(0.0f, 0.0f, 0.0f, 0.0f), dq = dk;
            float kr[R];
#pragma unroll
            for (int j = 0; j < R; j++) {
                const float qr = sq[i][rg + 16 * j];
                kr[j] = sk[i][rg + 16 * j];
                dk.x = __fmaf_rn(kr[j], S[j].x, dk.x); dk.y = __fmaf_rn(kr[j], S[j].y, dk.y);
                dk.z = __fmaf_rn(kr[j], S[j].z, dk.z); dk.w = __fmaf_rn(kr[j], S[j].w, dk.w);
                dq.x = __fmaf_rn(qr, S[j].x, dq.x); dq.y = __fmaf_rn(qr, S[j].y, dq.y);
                dq.z = __fmaf_rn(qr, S[j].z, dq.z); dq.w = __fmaf_rn(qr, S[j].w, dq.w);
            }
#pragma unroll
            for (int o = 8; o <= 16; o <<= 1) {
                dk.x += __shfl_xor_sync(0xffffffffu, dk.x, o); dk.y += __shfl_xor_sync(0xffffffffu, dk.y, o);
                dk.z += __shfl_xor_sync(0xffffffffu, dk.z, o); dk.w += __shfl_xor_sync(0xffffffffu, dk.w, o);
                dq.x += __shfl_xor_sync(0xffffffffu, dq.x, o); dq.y += __shfl_xor_sync(0xffffffffu, dq.y, o);
                dq.z += __shfl_xor_sync(0xffffffffu, dq.z, o); dq.w += __shfl_xor_sync(0xffffffffu, dq.w, o);
            }
            float(*rd)[2][32] = red[i & 1];  // two buffers: one barrier a token is enough
            if (lane < 8) *reinterpret_cast<float4 *>(&rd[warp][0][c4]) = dk;
            else if (lane < 16) *reinterpret_cast<float4 *>(&rd[warp][1][c4]) = dq;
            __syncthreads();
            const float al = sa[i], be = sb[i], qk = sqk[i];
            float d[4], o[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float sk4 = (rd[0][0][c4 + c] + rd[1][0][c4 + c]) + (rd[2][0][c4 + c] + rd[3][0][c4 + c]);
                const float sq4 = (rd[0][1][c4 + c] + rd[1][1][c4 + c]) + (rd[2][1][c4 + c] + rd[3][1][c4 + c]);
                d[c] = be * __fmaf_rn(-al, sk4, sv[i][c4 + c]);
                o[c] = __fmaf_rn(qk, d[c], al * sq4);
            }
#pragma unroll
            for (int j = 0; j < R; j++) {
                S[j].x = __fmaf_rn(kr[j], d[0], al * S[j].x); S[j].y = __fmaf_rn(kr[j], d[1], al * S[j].y);
                S[j].z = __fmaf_rn(kr[j], d[2], al * S[j].z); S[j].w = __fmaf_rn(kr[j], d[3], al * S[j].w);
            }
            if (rg == 0) *reinterpret_cast<float4 *>(a.out + (t0 + i) * (int64_t)a.n_v * a.dv + (int64_t)h * a.dv + c0 + c4) = make_float4(o[0], o[1], o[2], o[3]);
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++) *reinterpret_cast<float4 *>(a.state_out + soff + (int64_t)16 * i * a.dv) = S[i];
}

bool delta_shape_ok(int64_t T, int64_t n_seqs, int n_k, int n_v, int dk, int dv) {
    return T >= 0 && T <= 0x7fffffffLL && n_seqs > 0 && n_seqs <= 65535 && n_k > 0 && n_v > 0 && n_v % n_k == 0 && n_v <= 65535 && (dk == 64 || dk == 128) &&
           dv > 0 && dv % 32 == 0 && dv <= 256;
}

}  // namespace

extern "C" int64_t agn_gated_delta_rule_workspace_bytes(int64_t T, int64_t n_seqs, int32_t n_k_heads, int32_t n_v_heads, int32_t head_k,
                                                        int32_t head_v) {
    if (!delta_shape_ok(T, n_seqs, n_k_heads, n_v_heads, head_k, head_v)) return 0;
    return 0;
}

extern "C" int32_t agn_gated_delta_rule_f32(agn_ctx *ctx, const float *q, const float *k, const float *v, const float *g, const float *beta,
                                            const float *state_in, float *state_out, float *out, int64_t T, int64_t n_seqs,
                                            const int32_t *cu_seqlens, int32_t n_k_heads, int32_t n_v_heads, int32_t head_k, int32_t head_v,
                                            int64_t q_stride, int64_t k_stride, int64_t v_stride, float scale, float l2norm_eps,
                                            void *workspace, size_t workspace_bytes) {
    AGN_CHECK_CTX(ctx);
    if (!delta_shape_ok(T, n_seqs, n_k_heads, n_v_heads, head_k, head_v))
        return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: T=%lld n_seqs=%lld n_k_heads=%d n_v_heads=%d head_k=%d (64, 128) head_v=%d (a multiple of "
                        "32 up to 256)", (long long)T, (long long)n_seqs, n_k_heads, n_v_heads, head_k, head_v);
    if (!cu_seqlens && T % n_seqs)
        return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: %lld rows are not %lld sequences of one length (pass cu_seqlens)", (long long)T, (long long)n_seqs);
    if (q_stride < (int64_t)n_k_heads * head_k || k_stride < (int64_t)n_k_heads * head_k || v_stride < (int64_t)n_v_heads * head_v)
        return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: a row stride is smaller than the row");
    if (!isfinite(scale) || isnan(l2norm_eps)) return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: scale and l2norm_eps must be numbers");
    if (!state_out || (T > 0 && (!q || !k || !v || !g || !beta || !out))) return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: null pointer");
    if (!agn_aligned16(state_in) || !agn_aligned16(state_out) || !agn_aligned16(q) || !agn_aligned16(k) || !agn_aligned16(v) || !agn_aligned16(out) ||
        q_stride % 4 || k_stride % 4 || v_stride % 4)
        return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: q, k, v, out and the states must be 16-byte aligned, row strides multiples of 4");
    if (out && (out == q || out == k || out == v)) return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: out must not alias q, k or v");
    AGN_CUDA(ctx, cudaSetDevice(ctx->device));
    DeltaArgs a;
    a.q = q; a.k = k; a.v = v; a.g = g; a.beta = beta; a.state_in = state_in; a.state_out = state_out; a.out = out; a.cu = cu_seqlens;
    a.T = T; a.n_seqs = n_seqs; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.n_k = n_k_heads; a.n_v = n_v_heads; a.dv = head_v; a.scale = scale; a.eps = l2norm_eps; a.flags = ctx->d_flags;
    const dim3 grid((unsigned)(head_v / 32), (unsigned)n_v_heads, (unsigned)n_seqs);
    if (head_k == 64) agn_launch(ctx, delta_recurrent_kernel<64>, grid, dim3(128), 0, a);
    else agn_launch(ctx, delta_recurrent_kernel<128>, grid, dim3(128), 0, a);
    if (cu_seqlens) ctx->flags_dirty = true;
    AGN_LAUNCHED(ctx, "gated_delta_recurrent");
    (void)workspace; (void)workspace_bytes;
    return AGN_OK;
}
