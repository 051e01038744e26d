// Attention of query rows over the KV cache that agn_kv_write_f32 fills.
//
//   out[t, h, :] = sum_j p_j V[s, j, h / G, :],  p = softmax_j(scale * q[t, h, :] . K[s, j, h / G, :]),  j = 0 .. pos[t]
//
// (`launch_attention`, src/ops/wgpu_backend/resident.rs:551-565; kernels `attention_scores`, `attention_softmax`,
// `attention_output` and their `_q8_0` forms, src/ops/kernels_wgpu.rs:749-980; CPU `attention_into`,
// src/model/llama/cpu_path.rs:160-192).  G = n_q_heads / n_kv_heads query heads share a KV head.
#include <math.h>

#include "agn_attention_decode.cuh"

namespace {

// Joins the parts of the rows that attn_decode_kernel shared out over several CTAs, and writes the rows that see nothing.  A CTA per (row, query head); a warp takes
// every eighth part, four at a time (all their loads at once: the kernel is a few waits for memory long), each with maximum and sums of its own, and the warps'
// results are joined in shared memory.  (16 rows of 8192 slots, both kernels: 58.4 us with 256 threads, 63.1 with 512, 60.1 with 128.)
constexpr int JOIN_THREADS = 256, JOIN_TEAMS = JOIN_THREADS / 32;
__global__ void __launch_bounds__(JOIN_THREADS) attn_join_kernel(const __grid_constant__ DecodeArgs d) {
    agn_pdl_prologue();
    __shared__ int64_t warp_sums[JOIN_TEAMS], mine[2];
    __shared__ __align__(16) float sums[JOIN_TEAMS][256];
    __shared__ float ms[JOIN_TEAMS], ls[JOIN_TEAMS];
    const AttnArgs &a = d.a;
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hd = a.hd;
    const int64_t out = (t * a.n_q + h) * hd;
    int64_t w = 0, n, all;
    if (a.T == 1) {
        n = all = attn_tiles(a, 0, d.tt);
    } else {
        int64_t r0, r1, pre;
        scan_rows(a, d.tt, warp_sums, &r0, &r1, &pre, &all);
        if (r0 <= t && t < r1) {
            for (int64_t r = r0; r < t; r++) pre += attn_tiles(a, r, d.tt);
            mine[0] = pre;
            mine[1] = attn_tiles(a, t, d.tt);
        }
        __syncthreads();
        w = mine[0];
        n = mine[1];
    }
    if (n == 0) {
        if (tid < hd) store_act(d, out + tid, 0.0f);
        return;
    }
    const AttnShares shares(all, d.parts);
    const int x0 = a.T == 1 ? 0 : shares.part(w), x1 = a.T == 1 ? d.parts - 1 : shares.part(w + n - 1);
    if (shares.start(x0) <= w && w + n <= shares.start(x0 + 1)) return;  // in one part: written there
    const float *part = d.part + (int64_t)h * (hd + 4);
    float M = -INFINITY, L = 0.0f;
    float4 o[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
    for (int x = x0 + warp; x <= x1; x += 4 * JOIN_TEAMS) {
        float m[4], l[4];
        float4 v[4][2];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int y = x + k * JOIN_TEAMS;
            const int64_t begin = shares.start(y);
            const bool there = y <= x1 && begin < shares.start(y + 1);  // a CTA without tiles left nothing
            // its first run of tiles is this row's unless the CTA began in an earlier row
            const float *p = part + (2 * (int64_t)y + (begin < w ? 1 : 0)) * d.slot_floats;
            m[k] = there ? p[hd] : -INFINITY;
            l[k] = there ? p[hd + 1] : 0.0f;
#pragma unroll
            for (int i = 0; i < 2; i++)
                v[k][i] = there && 4 * lane + 128 * i < hd ? *reinterpret_cast<const float4 *>(p + 4 * lane + 128 * i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        const float top = fmaxf(fmaxf(M, fmaxf(m[0], m[1])), fmaxf(m[2], m[3])), mu = top == -INFINITY ? 0.0f : top, c = ex2(M - mu);
        M = top;
        L *= c;
#pragma unroll
        for (int i = 0; i < 2; i++) { o[i].x *= c; o[i].y *= c; o[i].z *= c; o[i].w *= c; }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float f = ex2(m[k] - mu);
            L = __fmaf_rn(f, l[k], L);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                o[i].x = __fmaf_rn(f, v[k][i].x, o[i].x); o[i].y = __fmaf_rn(f, v[k][i].y, o[i].y);
                o[i].z = __fmaf_rn(f, v[k][i].z, o[i].z); o[i].w = __fmaf_rn(f, v[k][i].w, o[i].w);
            }
        }
    }
    if (lane == 0) {
        ms[warp] = M;
        ls[warp] = L;
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
        if (4 * lane + 128 * i < hd) *reinterpret_cast<float4 *>(&sums[warp][4 * lane + 128 * i]) = o[i];
    __syncthreads();
    if (tid >= hd) return;
    float top = -INFINITY, sum = 0.0f, y = 0.0f;
#pragma unroll
    for (int k = 0; k < JOIN_TEAMS; k++) top = fmaxf(top, ms[k]);
    const float mu = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < JOIN_TEAMS; k++) {
        const float f = ex2(ms[k] - mu);
        sum = __fmaf_rn(f, ls[k], sum);
        y = __fmaf_rn(f, sums[k][tid], y);
    }
    store_act(d, out + tid, y / sum);
}

// The decode kernel's shape for a call: heads to a CTA, warps to a head, tiles, stages.
struct DecodePlan {
    int tt, stages, hc, groups, row_stride, col_groups, chunks, parts;
    size_t smem;
};
constexpr int ATTN_SMEM = 106500;  // of the stages: two CTAs per SM beside their 9 KB of joining buffers

DecodePlan decode_plan(int64_t T, int n_q, int n_kv, int hd, int64_t max_seq, int block_bytes, bool f16, int sms) {
    DecodePlan p;
    p.hc = n_kv < 8 ? n_kv : 8;
    p.chunks = (n_kv + p.hc - 1) / p.hc;
    p.col_groups = (n_q / n_kv + 7) / 8;
    p.row_stride = attn_row_stride(p.hc * (hd / 32) * block_bytes);
    p.groups = 8 / p.hc;
    p.tt = attn_slots_per_warp(f16) * p.groups;
    p.stages = 3;
    if (2 * p.tt * p.row_stride * 3 > (hd <= 128 ? ATTN_SMEM : 215000)) p.stages = 2;
    p.smem = (size_t)p.stages * 2 * p.tt * p.row_stride + 16;
    p.parts = 0;
    if (T <= ATTN_MAX_SPLIT_ROWS) {
        const int64_t most = T * ((max_seq + p.tt - 1) / p.tt), fill = 2 * sms / (p.chunks * p.col_groups) > 0 ? 2 * sms / (p.chunks * p.col_groups) : 1;
        p.parts = (int)(most < fill ? most : fill);
    }
    return p;
}

bool attn_shape_ok(int64_t T, int n_q, int n_kv, int hd, int64_t max_seq) {
    return T >= 0 && T <= 0x7fffffffLL && n_q > 0 && n_kv > 0 && n_q % n_kv == 0 && n_q <= 65535 && hd > 0 && hd <= 256 && hd % 32 == 0 &&
           max_seq > 0 && max_seq <= 0x7fffff00LL;
}

// Two parts per CTA of the decode kernel; the CTAs are as many as the largest part of this architecture holds two of per SM.
int64_t attn_workspace(int64_t T, int n_q, int hd) {
    return T > 0 && T <= ATTN_MAX_SPLIT_ROWS ? (int64_t)2 * 2 * ATTN_MAX_SMS * n_q * (hd + 4) * 4 : 0;
}

// Few rows of one sequence are quicker as single rows (f32 over q8_0, single rows / chunks, us: 28/4 heads of 128 behind 8000 slots 8 rows 35 / 39, 12 rows 43 / 41, behind
// 1000 slots 12 rows 19 / 18; 32/8 heads of 128 behind 8000 slots 8 rows 53 / 56, 12 rows 70 / 57).
constexpr int CHUNK_MIN_TOKENS = 12;
bool chunk_fits(int64_t T, int n_q, int n_kv) { return T >= CHUNK_MIN_TOKENS && T * (n_q / n_kv) < (1LL << 30); }

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
    if (!agn_aligned(pos, 4) || !agn_aligned(seq, 4)) return agn_fail(ctx, AGN_EINVAL, "attention_kv: pos and seq must be 4-byte aligned");
    const bool prompt = !pos && sizeof(T) == 2 && agn_attention_prompt_fits(rows, n_q, n_kv, hd);
    const bool chunk = !pos && !prompt && chunk_fits(rows, n_q, n_kv);
    const int sms = ctx->sm_count < ATTN_MAX_SMS ? ctx->sm_count : ATTN_MAX_SMS;
    const int64_t end = (int64_t)pos_start + rows;
    const int64_t need = prompt ? agn_attention_prompt_workspace(end, rows, n_q, n_kv, hd, sms, false)
                         : chunk ? agn_attention_chunk_workspace(end, rows, n_q, n_kv, hd, sms, false) : attn_workspace(rows, n_q, hd);
    if (need > 0 && (!workspace || (int64_t)workspace_bytes < need || !agn_aligned16(workspace)))
        return agn_fail(ctx, AGN_EINVAL, "attention_kv: needs %lld bytes of 16-byte aligned workspace", (long long)need);
    AGN_CUDA(ctx, cudaSetDevice(ctx->device));
    AttnArgs a;
    a.q = q; a.out = out; a.k_cache = static_cast<const unsigned char *>(k_cache); a.v_cache = static_cast<const unsigned char *>(v_cache);
    a.pos = pos; a.seq = seq; a.T = rows; a.n_seqs = n_seqs; a.max_seq = max_seq; a.n_q = n_q; a.n_kv = n_kv; a.hd = hd; a.pos_start = pos_start;
    a.bytes_per_token = (int)agn_kv_bytes_per_token(kv_dtype, (int64_t)n_kv * hd); a.scale = scale; a.flags = ctx->d_flags;
    ctx->flags_dirty = true;
    if (prompt) return agn_attention_prompt_f16(ctx, a, kv_dtype, workspace);
    if (chunk) return agn_attention_chunk(ctx, a, kv_dtype, sizeof(T) == 2, workspace);
    const int block_bytes = kv_dtype == AGN_F16 ? 64 : kv_dtype == AGN_Q8_0 ? 34 : 36;
    const DecodePlan p = decode_plan(rows, n_q, n_kv, hd, max_seq, block_bytes, kv_dtype == AGN_F16, sms);
    DecodeArgs d;
    d.a = a; d.part = static_cast<float *>(workspace); d.parts = p.parts; d.act16 = sizeof(T) == 2; d.tt = p.tt; d.stages = p.stages; d.hc = p.hc;
    d.groups = p.groups; d.row_stride = p.row_stride; d.col_groups = p.col_groups; d.slot_floats = n_q * (hd + 4);
    // the widest copy that the caches' address, the row's and the heads' share of it allow
    const int last = (n_kv - (p.chunks - 1) * p.hc) * (hd / 32) * block_bytes;
    const uint64_t bits = (uint64_t)reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | (uint64_t)a.bytes_per_token |
                          (uint64_t)(p.hc * (hd / 32) * block_bytes) | (uint64_t)last | 16;
    d.granule = (int)(bits & (0 - bits));
    size_t smem = p.smem;
    if (d.granule < 4) { d.stages = 1; smem = (size_t)2 * p.tt * p.row_stride + 16; }
    const dim3 grid((unsigned)(p.parts ? p.parts : rows), (unsigned)(p.chunks * p.col_groups));
    const int32_t rc = kv_dtype == AGN_F16 ? agn_attention_decode_f16(ctx, d, grid, smem)
                       : kv_dtype == AGN_Q8_0 ? agn_attention_decode_q8(ctx, d, grid, smem) : agn_attention_decode_words(ctx, d, grid, smem);
    if (rc != AGN_OK || !p.parts) return rc;
    agn_launch(ctx, attn_join_kernel, dim3((unsigned)rows, (unsigned)n_q), dim3(JOIN_THREADS), 0, d);
    AGN_LAUNCHED(ctx, "attention_kv_decode");
    return AGN_OK;
}

}  // namespace

extern "C" int64_t agn_attention_kv_workspace_bytes(int64_t T, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int64_t max_seq_len,
                                                    int32_t has_pos) {
    if (!attn_shape_ok(T, n_q_heads, n_kv_heads, head_dim, max_seq_len)) return 0;
    int64_t need = attn_workspace(T, n_q_heads, head_dim);
    if (has_pos) return need;
    // for whichever activation type the rows have, and for rows that end anywhere in the cache
    const int64_t chunk = chunk_fits(T, n_q_heads, n_kv_heads) ? agn_attention_chunk_workspace(max_seq_len, T, n_q_heads, n_kv_heads, head_dim, ATTN_MAX_SMS, true) : 0;
    const int64_t prompt = agn_attention_prompt_fits(T, n_q_heads, n_kv_heads, head_dim)
                               ? agn_attention_prompt_workspace(max_seq_len, T, n_q_heads, n_kv_heads, head_dim, ATTN_MAX_SMS, true) : 0;
    if (chunk > need) need = chunk;
    return prompt > need ? prompt : need;
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
