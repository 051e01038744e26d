// Joins the shares of the slots that the prompt kernels took of a row.
#include <math.h>

#include "agn_attention_decode.cuh"

namespace {

constexpr int JOIN_WARPS = 8;

// One warp per (token, query head), four values per lane and step: out = sum_x c_x o_x / sum_x c_x l_x with c_x = 2^(m_x - max m).
__global__ void __launch_bounds__(32 * JOIN_WARPS) attn_split_join_kernel(const __grid_constant__ DecodeArgs d, AttnSplit split, int kv_dtype, const int *odd, int64_t odd_tiles, int group) {
    agn_pdl_prologue();
    __shared__ float weight[JOIN_WARPS][ATTN_MAX_SMS];
    const AttnArgs &a = d.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = a.hd;
    const int64_t row = (int64_t)blockIdx.x * JOIN_WARPS + warp, stride = a.T * a.n_q * (int64_t)(hd + 4);
    if (row >= a.T * a.n_q) return;
    const float *part = split.part + row * (hd + 4);
    float M = -INFINITY, L = 0.0f;
    for (int x = lane; x < split.splits; x += 32) M = fmaxf(M, weight[warp][x] = part[x * stride + hd]);
    M = agn_warp_max(M);
    for (int x = lane; x < split.splits; x += 32) {
        const float m = weight[warp][x], l = part[x * stride + hd + 1], c = ex2(m - (M == -INFINITY ? 0.0f : M));
        weight[warp][x] = m == -INFINITY && l == 0.0f ? -1.0f : c;  // -1: nothing in it, not even sums
        L = __fmaf_rn(c, l, L);  // NaN where all of a share's scores are: its maximum is still -inf
    }
    L = agn_warp_sum(L);
    __syncwarp();
    const float inv = M == -INFINITY ? NAN : 1.0f / L;  // all scores -inf: 0 / 0
    bool any = false;
    const int kvh = (int)(row % a.n_q) / (a.n_q / a.n_kv), last = a.pos_start + (int)(row / a.n_q);
    const int *flags = odd + kvh * odd_tiles;
    if (kv_dtype >= 0) {
        for (int t = lane; t <= last / group; t += 32) any |= flags[t] != 0;
        any = __any_sync(0xffffffffu, any);
    }
    for (int i = 4 * lane; i < hd; i += 128) {
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int x = 0; x < split.splits; x++) {
            const float c = weight[warp][x];
            if (c < 0.0f) continue;
            const float4 v = *reinterpret_cast<const float4 *>(part + x * stride + i);  // sums that are not finite count whatever their weight is
            o.x = __fmaf_rn(c, v.x, o.x); o.y = __fmaf_rn(c, v.y, o.y); o.z = __fmaf_rn(c, v.z, o.z); o.w = __fmaf_rn(c, v.w, o.w);
        }
        o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
        if (any) {
            const auto look = [&](int slot) { return flags[slot / group] != 0; };
            o.x += odd_value(a, kv_dtype, kvh * hd + i, last, look, group);
            o.y += odd_value(a, kv_dtype, kvh * hd + i + 1, last, look, group);
            o.z += odd_value(a, kv_dtype, kvh * hd + i + 2, last, look, group);
            o.w += odd_value(a, kv_dtype, kvh * hd + i + 3, last, look, group);
        }
        store_act4(d, row * hd, i >> 2, o);
    }
}

}  // namespace

int32_t agn_attention_join(agn_ctx *ctx, const AttnArgs &a, int kv_dtype, int act16, AttnSplit split, const int *odd, int64_t odd_tiles, int group) {
    DecodeArgs d = {};
    d.a = a;
    d.act16 = act16;
    agn_launch(ctx, attn_split_join_kernel, dim3((unsigned)((a.T * a.n_q + JOIN_WARPS - 1) / JOIN_WARPS)), dim3(32 * JOIN_WARPS), 0, d, split, odd ? kv_dtype : -1, odd, odd_tiles, group);
    AGN_LAUNCHED(ctx, "attention_kv_join");
    return AGN_OK;
}
