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

// A warp per row, the row in registers (VPT vectors of four per lane), so that x is read once; VEC false: scalar accesses for
// rows whose length or address does not allow vectors.
template <typename OT, int VPT, bool VEC>
__global__ void __launch_bounds__(256) gated_norm_warp_kernel(const float *__restrict__ x, const float *__restrict__ gate,
                                                              const float *__restrict__ w, OT *__restrict__ out, int64_t rows, int n,
                                                              float inv_n, float eps) {
    agn_pdl_prologue();
    const int lane = threadIdx.x & 31;
    const int64_t r = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (r >= rows) return;
    const float *xr = x + r * n, *gr = gate + r * n;
    float4 xv[VPT], gv[VPT];
    float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const int i = 4 * (lane + 32 * k);
        xv[k] = gv[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (VEC) {
            if (i < n) { xv[k] = ActVec<float>::load(xr, i >> 2); gv[k] = ActVec<float>::load(gr, i >> 2); }
        } else {
            if (i < n) { xv[k].x = xr[i]; gv[k].x = gr[i]; }
            if (i + 1 < n) { xv[k].y = xr[i + 1]; gv[k].y = gr[i + 1]; }
            if (i + 2 < n) { xv[k].z = xr[i + 2]; gv[k].z = gr[i + 2]; }
            if (i + 3 < n) { xv[k].w = xr[i + 3]; gv[k].w = gr[i + 3]; }
        }
    }
#pragma unroll
    for (int k = 0; k < VPT; k++) acc = agn_sum_sq4(xv[k], acc);
    const float inv = agn_inv_rms(agn_warp_sum(acc.x + acc.y), inv_n, eps);
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        const int i = 4 * (lane + 32 * k);
        if (i >= n) continue;
        float4 wv;
        if (VEC) {
            wv = __ldg(reinterpret_cast<const float4 *>(w + i));
        } else {
            wv = make_float4(w[i], i + 1 < n ? w[i + 1] : 0.0f, i + 2 < n ? w[i + 2] : 0.0f, i + 3 < n ? w[i + 3] : 0.0f);
        }
        const float4 y = agn_silu_mul4(gv[k], agn_scale4(agn_mul4(wv, xv[k]), inv));
        if (VEC) {
            ActVec<OT>::store(out + r * n, i >> 2, y);
        } else {
            ActVec<OT>::store1(out + r * n, i, y.x);
            if (i + 1 < n) ActVec<OT>::store1(out + r * n, i + 1, y.y);
            if (i + 2 < n) ActVec<OT>::store1(out + r * n, i + 2, y.z);
            if (i + 3 < n) ActVec<OT>::store1(out + r * n, i + 3, y.w);
        }
    }
}

template <typename OT, int VPT>
void launch_vpt(agn_ctx *ctx, bool vec, const float *x, const float *gate, const float *w, OT *out, int64_t rows, int n, float eps) {
    const int warps = 4;
    const dim3 grid((unsigned)((rows + warps - 1) / warps));
    if (vec) agn_launch(ctx, gated_norm_warp_kernel<OT, VPT, true>, grid, dim3(32 * warps), 0, x, gate, w, out, rows, n, 1.0f / (float)n, eps);
    else agn_launch(ctx, gated_norm_warp_kernel<OT, VPT, false>, grid, dim3(32 * warps), 0, x, gate, w, out, rows, n, 1.0f / (float)n, eps);
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
