// The norm behind a recurrent mixer, fused with its gate:
//
//   out[r, i] = (w[i] * x[r, i]) / sqrt(sum_i x[r, i]^2 / n + eps) * gate[r, i] / (1 + exp(-gate[r, i]))
//
// over rows of one head each (n = head size, one weight for all heads).  HBM-bound, 12 bytes a value in f32 (10 with a 16-bit
// result).
#include <math.h>

#include "agn_common.cuh"
#include "agn_row_math.cuh"

namespace {

// A warp takes R rows, each in registers (VPT vectors of four per lane), all loads ahead of the first use, so that x is read once and enough bytes are on their
// way.  VEC false: scalar accesses for rows whose length or address does not allow vectors.
template <typename OT, int VPT, int R, bool VEC>
__global__ void __launch_bounds__(128) gated_norm_warp_kernel(const float *__restrict__ x, const float *__restrict__ gate, const float *__restrict__ w, OT *__restrict__ out,
                                                              int64_t rows, int n, float inv_n, float eps) {
    agn_pdl_prologue();
    const int lane = threadIdx.x & 31;
    const int64_t r0 = ((int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * R;
    if (r0 >= rows) return;
    float4 xv[R][VPT], gv[R][VPT];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const float *xr = x + (r0 + r) * n, *gr = gate + (r0 + r) * n;
        const bool there = r0 + r < rows;
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int i = 4 * (lane + 32 * k);
            xv[r][k] = gv[r][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (VEC) {
                if (there && i < n) { xv[r][k] = ActVec<float>::load(xr, i >> 2); gv[r][k] = ActVec<float>::load(gr, i >> 2); }
            } else if (there) {
                if (i < n) { xv[r][k].x = xr[i]; gv[r][k].x = gr[i]; }
                if (i + 1 < n) { xv[r][k].y = xr[i + 1]; gv[r][k].y = gr[i + 1]; }
                if (i + 2 < n) { xv[r][k].z = xr[i + 2]; gv[r][k].z = gr[i + 2]; }
                if (i + 3 < n) { xv[r][k].w = xr[i + 3]; gv[r][k].w = gr[i + 3]; }
            }
        }
    }
    float4 wv[VPT];
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const int i = 4 * (lane + 32 * k);
        if (VEC) wv[k] = i < n ? __ldg(reinterpret_cast<const float4 *>(w + i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        else wv[k] = make_float4(i < n ? w[i] : 0.0f, i + 1 < n ? w[i + 1] : 0.0f, i + 2 < n ? w[i + 2] : 0.0f, i + 3 < n ? w[i + 3] : 0.0f);
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < VPT; k++) acc = agn_sum_sq4(xv[r][k], acc);
        const float inv = agn_inv_rms(agn_warp_sum(acc.x + acc.y), inv_n, eps);
        if (r0 + r >= rows) continue;
        OT *o = out + (r0 + r) * n;
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int i = 4 * (lane + 32 * k);
            if (i >= n) continue;
            const float4 y = agn_silu_mul4(gv[r][k], agn_scale4(agn_mul4(wv[k], xv[r][k]), inv));
            if (VEC) {
                ActVec<OT>::store(o, i >> 2, y);
            } else {
                ActVec<OT>::store1(o, i, y.x);
                if (i + 1 < n) ActVec<OT>::store1(o, i + 1, y.y);
                if (i + 2 < n) ActVec<OT>::store1(o, i + 2, y.z);
                if (i + 3 < n) ActVec<OT>::store1(o, i + 3, y.w);
            }
        }
    }
}

template <typename OT, int VPT, int R>
void launch_rows(agn_ctx *ctx, bool vec, const float *x, const float *gate, const float *w, OT *out, int64_t rows, int n, float eps) {
    const int per = 4 * R;  // rows of a CTA
    const dim3 grid((unsigned)((rows + per - 1) / per));
    if (vec) agn_launch(ctx, gated_norm_warp_kernel<OT, VPT, R, true>, grid, dim3(128), 0, x, gate, w, out, rows, n, 1.0f / (float)n, eps);
    else agn_launch(ctx, gated_norm_warp_kernel<OT, VPT, R, false>, grid, dim3(128), 0, x, gate, w, out, rows, n, 1.0f / (float)n, eps);
}

template <typename OT, int VPT>
void launch_vpt(agn_ctx *ctx, bool vec, const float *x, const float *gate, const float *w, OT *out, int64_t rows, int n, float eps) {
    // Two short rows per warp once they fill the GPU that way: 131072 rows of 128 in 31 us (6.4 TB/s); one row 36 us, four 31.4.  Fewer rows are
    // over sooner the more warps they are.
    constexpr int R = VPT == 1 ? 2 : 1;
    if (R > 1 && rows >= (int64_t)4 * R * 8 * ctx->sm_count) launch_rows<OT, VPT, R>(ctx, vec, x, gate, w, out, rows, n, eps);
    else launch_rows<OT, VPT, 1>(ctx, vec, x, gate, w, out, rows, n, eps);
}

template <typename OT>
int32_t gated_norm(agn_ctx *ctx, const float *x, const float *gate, const float *w, OT *out, int64_t rows, int64_t n, float eps) {
    if (rows < 0 || n <= 0 || n > 1024)
        return agn_fail(ctx, AGN_EINVAL, "rms_norm_silu_gate: rows=%lld n=%lld (1 .. 1024)", (long long)rows, (long long)n);
    if (rows > 4LL * 0x7fffffffLL) return agn_fail(ctx, AGN_EINVAL, "rms_norm_silu_gate: too many rows");
    if (rows == 0) return AGN_OK;
    if (!x || !gate || !w || !out) return agn_fail(ctx, AGN_EINVAL, "rms_norm_silu_gate: null pointer");
    if (!agn_aligned(x, 4) || !agn_aligned(gate, 4) || !agn_aligned(w, 4) || !agn_aligned(out, (int)sizeof(OT)))
        return agn_fail(ctx, AGN_EINVAL, "rms_norm_silu_gate: pointers must be aligned to their element type");
    AGN_CUDA(ctx, cudaSetDevice(ctx->device));
    const bool vec = n % 4 == 0 && agn_aligned16(x) && agn_aligned16(gate) && agn_aligned16(w) && agn_aligned(out, ActVec<OT>::ALIGN);
    if (n <= 128) launch_vpt<OT, 1>(ctx, vec, x, gate, w, out, rows, (int)n, eps);
    else if (n <= 256) launch_vpt<OT, 2>(ctx, vec, x, gate, w, out, rows, (int)n, eps);
    else if (n <= 512) launch_vpt<OT, 4>(ctx, vec, x, gate, w, out, rows, (int)n, eps);
    else launch_vpt<OT, 8>(ctx, vec, x, gate, w, out, rows, (int)n, eps);
    AGN_LAUNCHED(ctx, "rms_norm_silu_gate");
    return AGN_OK;
}

}  // namespace

extern "C" int32_t agn_rms_norm_silu_gate_f32(agn_ctx *ctx, const float *x, const float *gate, const float *w, float *out, int64_t rows,
                                              int64_t n, float eps) {
    AGN_CHECK_CTX(ctx);
    return gated_norm<float>(ctx, x, gate, w, out, rows, n, eps);
}

extern "C" int32_t agn_rms_norm_silu_gate_f32_out16(agn_ctx *ctx, const float *x, const float *gate, const float *w, void *out, int64_t rows,
                                                    int64_t n, float eps, int32_t out_dtype) {
    AGN_CHECK_CTX(ctx);
    if (out_dtype != AGN_F16 && out_dtype != AGN_BF16)
        return agn_fail(ctx, AGN_EUNSUPPORTED_DTYPE, "rms_norm_silu_gate: output dtype %d is neither f16 (1) nor bf16 (30)", out_dtype);
    if (static_cast<const void *>(x) == out || static_cast<const void *>(gate) == out)
        return rows == 0 ? AGN_OK : agn_fail(ctx, AGN_EINVAL, "rms_norm_silu_gate: a 16-bit output must not alias an input");
    if (out_dtype == AGN_F16) return gated_norm<__half>(ctx, x, gate, w, static_cast<__half *>(out), rows, n, eps);
    return gated_norm<__nv_bfloat16>(ctx, x, gate, w, static_cast<__nv_bfloat16 *>(out), rows, n, eps);
}
