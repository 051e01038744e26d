// Attention of query rows over the KV cache that agn_kv_write_f32 fills.
//
//   out[t, h, :] = sum_j p_j V[s, j, h / G, :],  p = softmax_j(scale * q[t, h, :] . K[s, j, h / G, :]),  j = 0 .. pos[t]
//
// (`launch_attention`, src/ops/wgpu_backend/resident.rs:551-565; kernels `attention_scores`, `attention_softmax`,
// `attention_output` and their `_q8_0` forms, src/ops/kernels_wgpu.rs:749-980; CPU `attention_into`,
// src/model/llama/cpu_path.rs:160-192).  G = n_q_heads / n_kv_heads query heads share a KV head.
#include <math.h>

#include "agn_attention.cuh"

namespace {

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

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], float a0, float a1, float a2, float a3, float b0, float b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)), "r"(__float_as_uint(b0)),
          "r"(__float_as_uint(b1)));
}
__device__ __forceinline__ void add4(float (&o)[4], const float (&x)[4]) {
    const float2 a = __fadd2_rn(make_float2(o[0], o[1]), make_float2(x[0], x[1])), b = __fadd2_rn(make_float2(o[2], o[3]), make_float2(x[2], x[3]));
    o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
}
template <int N> __device__ __forceinline__ void cp_async(uint32_t dst, const void *src, bool in) {  // zeros where it is not `in`
    if (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(in ? N : 0) : "memory");
}
// four signed (q8_0) or offset-binary (words) bytes, all as byte + 128
template <int KV> __device__ __forceinline__ uint32_t offset_bytes(uint32_t w) { return KV == KV_Q8 ? w ^ 0x80808080u : w; }
// two of them as exact f16: 0x6400 | u is 1024 + u
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t u, uint32_t sel) {
    const uint32_t h = __byte_perm(u, 0x64646464u, sel);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&h), __floats2half2_rn(1152.0f, 1152.0f));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// one of them as exact f32: 0x4B000000 | u is 2^23 + u
__device__ __forceinline__ float byte_to_float(uint32_t u, int i) {
    return __fsub_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 + i)), 8388736.0f);
}
// p = hi + lo, hi with tf32's 11 bits (cut) and lo what is left of it.  The values it is multiplied by may not be finite, or the scale in
// it: with an infinite value lo must not be 0 (0 * inf), with an infinite p it must not be inf - inf, for the sum of
// the two products to be what the one product would be.
template <int KV> __device__ __forceinline__ void split_tf32(float p, float &hi, float &lo) {
    hi = __uint_as_float(__float_as_uint(p) & 0xffffe000u);
    lo = KV == KV_F16 ? fmaxf(p - hi, 1.17549435e-38f) : fminf(p - hi, 1e35f);
}
// four / eight bytes at an address that is a multiple of 4, or (odd) 2 behind one
__device__ __forceinline__ uint32_t load4_at(const unsigned char *p, bool odd) {
    if (!odd) return *reinterpret_cast<const uint32_t *>(p);
    const uint32_t *w = reinterpret_cast<const uint32_t *>(p - 2);
    return __funnelshift_r(w[0], w[1], 16);
}
__device__ __forceinline__ void load8_at(const unsigned char *p, bool odd, uint32_t &x, uint32_t &y) {
    if (odd) {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(p - 2);
        const uint32_t w1 = w[1];
        x = __funnelshift_r(w[0], w1, 16);
        y = __funnelshift_r(w1, w[2], 16);
    } else {
        x = reinterpret_cast<const uint32_t *>(p)[0];
        y = reinterpret_cast<const uint32_t *>(p)[1];
    }
}
// ---- Decode: rows of any position and sequence ----------------------------------------------------------------------
//
// Bound by HBM: a slot's 2 * bytes_per_token bytes are read once for all query heads.  What a CTA works on is a run of tiles of
// `tt` slots: all rows' tiles are numbered one after the other and shared out evenly (so a batch of very different lengths, or one long row, fills
// the GPU alike); a row that falls into several CTAs is joined by attn_join_kernel.  Tiles arrive by cp.async in a ring of stages, all KV heads of a
// slot together, and each warp takes one KV head (and a share of the tile's slots where there are fewer than 8).
//
// Per 8 slots and head, on the matrix units so that the instructions per cached byte stay below what the stream allows:
//   S = Q K^T as m16n8k16 f16: rows 0-7 hold the upper halves of the (up to 8) query heads, rows 8-15 the lower halves
//     (q = hi + lo, each 11 bits, after a power of two has brought the row's largest value to [1, 2)), the columns are slots; the cached
//     bytes are exact in f16, so a score keeps 22 bits; block scales are applied to the f32 products of 32 dims.
//   O^T += V^T P^T as m16n8k8 tf32, twice: p * scale split into two tf32 parts (22 bits, any range), V's bytes exact in tf32.  The
//     accumulators of S are P^T's operand layout as they are (columns 2t, 2t+1 stand for slots t, t+4).
constexpr int ATTN_MAX_SMS = 148, ATTN_THREADS = 256, ATTN_WARPS = 8, ATTN_MAX_SPLIT_ROWS = 512;

struct DecodeArgs {
    AttnArgs a;
    float *part;          // [2 * parts][n_q][hd + 2]
    int parts;            // CTAs along x; 0: one CTA per row, no joining
    int tt, stages, hc, groups, row_stride, granule, col_groups, slot_floats;
};

struct RowCursor {
    int64_t row, off;
    int n, j;  // visible slots, next slot
};

__device__ __forceinline__ int64_t attn_tiles(const AttnArgs &a, int64_t t, int tt) {
    int64_t off;
    return ((int64_t)attn_row(a, t, &off) + tt - 1) / tt;
}

// Tiles of all rows before each thread's share of the rows, and of all rows.
__device__ __forceinline__ void scan_rows(const AttnArgs &a, int tt, int64_t *warp_sums, int64_t *r0, int64_t *r1, int64_t *before,
                                          int64_t *total) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    *r0 = a.T * tid / blockDim.x;
    *r1 = a.T * (tid + 1) / blockDim.x;
    int64_t sum = 0;
    for (int64_t t = *r0; t < *r1; t++) sum += attn_tiles(a, t, tt);
    int64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int64_t pre = 0, all = 0;
    for (int w = 0; w < nw; w++) {
        if (w < warp) pre += warp_sums[w];
        all += warp_sums[w];
    }
    *before = pre + inc - sum;
    *total = all;
}

template <typename T, int KV, int NB, int U> __global__ void __launch_bounds__(ATTN_THREADS, NB <= 4 ? 2 : 1) attn_decode_kernel(DecodeArgs d) {
    agn_pdl_prologue();
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float xch[ATTN_WARPS][8][33], sm[ATTN_WARPS][8], sl[ATTN_WARPS][8];
    __shared__ int64_t warp_sums[ATTN_WARPS], first_row, first_pre;
    const AttnArgs &a = d.a;
    constexpr int HD = NB * 32;
    using F = KvFormat<KV>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int cg = blockIdx.y % d.col_groups, h0 = blockIdx.y / d.col_groups * d.hc, hc = min(d.hc, a.n_kv - h0);
    const int unit = warp % d.hc, group = warp / d.hc;
    const bool active = unit < hc && group < d.groups;
    const int G = a.n_q / a.n_kv, kvh = h0 + unit;
    const int cols = min(8, G - cg * 8);

    // ---- this CTA's run of tiles
    RowCursor cur;
    int left;
    if (d.parts == 0) {
        cur.row = blockIdx.x;
        cur.n = attn_row(a, cur.row, &cur.off);
        cur.j = 0;
        left = (int)(((int64_t)cur.n + d.tt - 1) / d.tt);
        if (left == 0 && active) {  // a row that sees nothing
            T *o = static_cast<T *>(a.out) + (cur.row * a.n_q + kvh * G + cg * 8) * HD;
            if (group == 0)
                for (int i = lane; i < cols * HD; i += 32) ActVec<T>::store1(o, i, 0.0f);
        }
    } else {
        int64_t r0, r1, pre, total;
        scan_rows(a, d.tt, warp_sums, &r0, &r1, &pre, &total);
        const int64_t w0 = total * blockIdx.x / d.parts, w1 = total * (blockIdx.x + 1) / d.parts;
        for (int64_t t = r0; t < r1; t++) {
            const int64_t n = attn_tiles(a, t, d.tt);
            if (w0 >= pre && w0 < pre + n) { first_row = t; first_pre = pre; }
            pre += n;
        }
        __syncthreads();
        left = (int)(w1 - w0);
        if (left > 0) {
            cur.row = first_row;
            cur.n = attn_row(a, cur.row, &cur.off);
            cur.j = (int)(w0 - first_pre) * d.tt;
        }
    }
    if (left <= 0) return;

    // ---- tiles into the ring
    const int cpr = hc * NB * F::BYTES / d.granule, tile_chunks = cpr * d.tt, side = d.tt * d.row_stride, stage_bytes = 2 * side;
    const uint32_t smem0 = agn_smem_u32(smem);
    const int tok0 = tid / cpr, rem0 = tid % cpr, step_tok = ATTN_THREADS / cpr, step_rem = ATTN_THREADS % cpr;
    const int src0 = tok0 * a.bytes_per_token + rem0 * d.granule, dst0 = tok0 * d.row_stride + rem0 * d.granule;
    const int src_step = step_tok * a.bytes_per_token + step_rem * d.granule, dst_step = step_tok * d.row_stride + step_rem * d.granule;
    const int src_wrap = a.bytes_per_token - cpr * d.granule, dst_wrap = d.row_stride - cpr * d.granule;
    auto issue = [&](const RowCursor &c, uint32_t stage_at) {
        const int64_t base = c.off + (int64_t)c.j * a.bytes_per_token + (int64_t)h0 * NB * F::BYTES;
        const unsigned char *ks = a.k_cache + base, *vs = a.v_cache + base;
        const int valid = min(d.tt, c.n - c.j);
        uint32_t dst = smem0 + stage_at + dst0;
        int tok = tok0, rem = rem0, src = src0;
        for (int i = tid; i < tile_chunks; i += ATTN_THREADS) {
            const bool in = tok < valid;  // slots that the row does not see are zeros, not what the cache holds there
            const int from = in ? src : 0;
            if (d.granule == 16) {
                cp_async<16>(dst, ks + from, in);
                cp_async<16>(dst + side, vs + from, in);
            } else if (d.granule == 8) {
                cp_async<8>(dst, ks + from, in);
                cp_async<8>(dst + side, vs + from, in);
            } else if (d.granule == 4) {
                cp_async<4>(dst, ks + from, in);
                cp_async<4>(dst + side, vs + from, in);
            } else {
                const uint16_t kx = in ? *reinterpret_cast<const uint16_t *>(ks + from) : (uint16_t)0;
                const uint16_t vx = in ? *reinterpret_cast<const uint16_t *>(vs + from) : (uint16_t)0;
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst), "h"(kx) : "memory");
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + side), "h"(vx) : "memory");
            }
            tok += step_tok;
            rem += step_rem;
            src += src_step;
            dst += dst_step;
            if (rem >= cpr) {
                rem -= cpr;
                tok++;
                src += src_wrap;
                dst += dst_wrap;
            }
        }
    };
    auto advance = [&](RowCursor &c) {
        c.j += d.tt;
        while (c.j >= c.n) {  // the next row with anything to see; there is one while tiles are left
            c.row++;
            c.n = attn_row(a, c.row, &c.off);
            c.j = 0;
        }
    };
    RowCursor ahead = cur;
    int to_issue = left;
    for (int s = 0; s < d.stages - 1; s++) {
        if (to_issue > 0) {
            issue(ahead, s * stage_bytes);
            if (--to_issue > 0) advance(ahead);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // ---- per row: the query heads as two f16 parts, softmax state, output accumulators
    uint32_t q[2 * NB][4];
    float o[2 * NB][4], m = -INFINITY, l = 0.0f, coef = 0.0f;
    bool fresh = true, first_segment = true;
    int seg_start = cur.j, stage_at = 0, fill_at = (d.stages - 1) * stage_bytes;  // bytes of the stage that is read, of the one that is filled
    const int ring = d.stages * stage_bytes;
    for (; left > 0; left--) {
        if (fresh) {
            fresh = false;
            seg_start = cur.j;
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            const bool there = active && g < cols;
            const T *qr = static_cast<const T *>(a.q) + (cur.row * a.n_q + (there ? kvh * G + cg * 8 + g : 0)) * HD;
            float amax = 0.0f;
            float4 x[2 * NB];
#pragma unroll
            for (int b = 0; b < 2 * NB; b++) {
                x[b] = there ? ActVec<T>::load(qr, (b >> 1) * 8 + 2 * t4 + (b & 1)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x[b].x), fabsf(x[b].y))), fmaxf(fabsf(x[b].z), fabsf(x[b].w)));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int e = min(max((int)(__float_as_uint(amax) >> 23), 1), 253);  // 2^(e-127) <= amax < 2^(e-126)
            const float down = __uint_as_float((uint32_t)(254 - e) << 23);         // 2^(127-e)
            coef = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)e << 23);
#pragma unroll
            for (int b = 0; b < 2 * NB; b++) {
                const float v[4] = {x[b].x * down, x[b].y * down, x[b].z * down, x[b].w * down};
                const __half2 h01 = __floats2half2_rn(v[0], v[1]), h23 = __floats2half2_rn(v[2], v[3]);
                const float2 f01 = __half22float2(h01), f23 = __half22float2(h23);
                const __half2 l01 = __floats2half2_rn(v[0] - f01.x, v[1] - f01.y), l23 = __floats2half2_rn(v[2] - f23.x, v[3] - f23.y);
                q[b][0] = *reinterpret_cast<const uint32_t *>(&h01);
                q[b][1] = *reinterpret_cast<const uint32_t *>(&l01);
                q[b][2] = *reinterpret_cast<const uint32_t *>(&h23);
                q[b][3] = *reinterpret_cast<const uint32_t *>(&l23);
            }
        }
        if (d.stages == 1) {  // plain loads: nothing runs ahead
            issue(cur, 0);
        } else if (d.stages == 2) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        }
        __syncthreads();
        if (d.stages > 1) {  // the stage that every warp has left
            if (to_issue > 0) {
                issue(ahead, fill_at);
                if (--to_issue > 0) advance(ahead);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        if (active) {
            const unsigned char *kt = smem + stage_at + unit * NB * F::BYTES, *vt = kt + side;
            const int per = d.tt / d.groups;
            for (int s0 = group * per; s0 < (group + 1) * per; s0 += 8 * U) {
                if (cur.j + s0 >= cur.n) break;
                float sc[U][2];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const unsigned char *krow = kt + (s0 + 8 * u + (g >> 1) + (g & 1) * 4) * d.row_stride;
                    const unsigned char *k0 = kt + (s0 + 8 * u + t4) * d.row_stride, *k1 = k0 + 4 * d.row_stride;
                    sc[u][0] = sc[u][1] = 0.0f;
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        if (KV == KV_F16) {
                            const uint4 w = *reinterpret_cast<const uint4 *>(krow + b * 64 + t4 * 16);
                            mma_f16(acc, q[2 * b], w.x, w.y);
                            mma_f16(acc, q[2 * b + 1], w.z, w.w);
                        } else {
                            float blk[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            uint32_t x0, x1;
                            load8_at(krow + b * F::BYTES + F::DATA + t4 * 8, KV == KV_Q8 && ((NB & 1 ? unit * NB + b : b) & 1) == 0, x0, x1);
                            x0 = offset_bytes<KV>(x0);
                            x1 = offset_bytes<KV>(x1);
                            mma_f16(blk, q[2 * b], bytes_to_half2(x0, 0x4140), bytes_to_half2(x0, 0x4342));
                            mma_f16(blk, q[2 * b + 1], bytes_to_half2(x1, 0x4140), bytes_to_half2(x1, 0x4342));
                            sc[u][0] = __fmaf_rn(blk[0] + blk[2], block_scale<KV>(k0 + b * F::BYTES), sc[u][0]);
                            sc[u][1] = __fmaf_rn(blk[1] + blk[3], block_scale<KV>(k1 + b * F::BYTES), sc[u][1]);
                        }
                    }
                    if (KV == KV_F16) { sc[u][0] = acc[0] + acc[2]; sc[u][1] = acc[1] + acc[3]; }
                }
                float mt = m;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int j = cur.j + s0 + 8 * u + t4;
                    sc[u][0] = j < cur.n ? sc[u][0] * coef : -INFINITY;
                    sc[u][1] = j + 4 < cur.n ? sc[u][1] * coef : -INFINITY;
                    mt = fmaxf(mt, fmaxf(sc[u][0], sc[u][1]));
                }
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
                if (__any_sync(0xffffffffu, mt > m)) {
                    const float c = ex2(m - (mt == -INFINITY ? 0.0f : mt));  // 0 at the first slots
                    l *= c;
                    const float c0 = __shfl_sync(0xffffffffu, c, t4 * 8), c1 = __shfl_sync(0xffffffffu, c, t4 * 8 + 4);
#pragma unroll
                    for (int i = 0; i < 2 * NB; i++) { o[i][0] *= c0; o[i][1] *= c1; o[i][2] *= c0; o[i][3] *= c1; }
                    m = mt;
                }
                const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    sc[u][0] = ex2(sc[u][0] - mu);
                    sc[u][1] = ex2(sc[u][1] - mu);
                    l += sc[u][0] + sc[u][1];
                }
                // The matrix unit's adder cuts what it shifts out: products of a few slots are summed there and the running sums are kept
                // by rounded additions (over thousands of slots the cuts would add up to 5e-6 of the result).
                const unsigned char *v0 = vt + (s0 + t4) * d.row_stride;
                float ph[U][2], pl[U][2];
                if (KV == KV_F16) {
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        split_tf32<KV>(sc[u][0], ph[u][0], pl[u][0]);
                        split_tf32<KV>(sc[u][1], ph[u][1], pl[u][1]);
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    float acc0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, acc1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        float f[2][4];
#pragma unroll
                        for (int i = 0; i < 2; i++) {  // slots t4 and t4 + 4 of the eight
                            const unsigned char *blk = v0 + (8 * u + 4 * i) * d.row_stride + b * F::BYTES;
                            if (KV == KV_F16) {
                                const uint2 w = *reinterpret_cast<const uint2 *>(blk + g * 8);
                                const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&w.x));
                                const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
                                f[i][0] = x.x; f[i][1] = x.y; f[i][2] = y.x; f[i][3] = y.y;
                            } else {
                                const bool odd = KV == KV_Q8 && ((NB & 1 ? unit * NB + b : b) & 1) == 0;
                                const uint32_t w = offset_bytes<KV>(load4_at(blk + F::DATA + g * 4, odd));
#pragma unroll
                                for (int c = 0; c < 4; c++) f[i][c] = byte_to_float(w, c);
                                split_tf32<KV>(sc[u][i] * block_scale<KV>(blk), ph[u][i], pl[u][i]);
                            }
                        }
                        mma_tf32(acc0, f[0][0], f[0][1], f[1][0], f[1][1], ph[u][0], ph[u][1]);
                        mma_tf32(acc1, f[0][2], f[0][3], f[1][2], f[1][3], ph[u][0], ph[u][1]);
                        mma_tf32(acc0, f[0][0], f[0][1], f[1][0], f[1][1], pl[u][0], pl[u][1]);
                        mma_tf32(acc1, f[0][2], f[0][3], f[1][2], f[1][3], pl[u][0], pl[u][1]);
                    }
                    add4(o[2 * b], acc0);
                    add4(o[2 * b + 1], acc1);
                }
            }
        }
        if (d.stages == 1) __syncthreads();
        const bool row_done = cur.j + d.tt >= cur.n;
        if (row_done || left == 1) {  // the end of a row, or of this CTA's part of one
            const bool whole = row_done && seg_start == 0;
            float lt = l + __shfl_xor_sync(0xffffffffu, l, 1);
            lt += __shfl_xor_sync(0xffffffffu, lt, 2);
            float M = m, L = lt;
            if (d.groups > 1) {  // join the shares of a head's warps
                __syncthreads();
                if (t4 == 0) { sm[warp][g] = m; sl[warp][g] = lt; }
                __syncthreads();
                for (int k = 0; k < d.groups; k++) M = fmaxf(M, sm[unit + k * d.hc][g]);
                L = 0.0f;
                for (int k = 0; k < d.groups; k++) L += sl[unit + k * d.hc][g] * ex2(sm[unit + k * d.hc][g] - (M == -INFINITY ? 0.0f : M));
                const float c = ex2(m - (M == -INFINITY ? 0.0f : M));
                const float c0 = __shfl_sync(0xffffffffu, c, t4 * 8), c1 = __shfl_sync(0xffffffffu, c, t4 * 8 + 4);
#pragma unroll
                for (int b = 0; b < NB; b++) {
#pragma unroll
                    for (int i = 2 * b; i < 2 * b + 2; i++) {
                        o[i][0] *= c0; o[i][1] *= c1; o[i][2] *= c0; o[i][3] *= c1;
                        xch[warp][2 * t4][4 * g + 2 * (i & 1)] = o[i][0];
                        xch[warp][2 * t4 + 1][4 * g + 2 * (i & 1)] = o[i][1];
                        xch[warp][2 * t4][4 * g + 2 * (i & 1) + 1] = o[i][2];
                        xch[warp][2 * t4 + 1][4 * g + 2 * (i & 1) + 1] = o[i][3];
                    }
                    __syncthreads();
                    if (group == 0)
                        for (int k = 1; k < d.groups; k++)
#pragma unroll
                            for (int i = 2 * b; i < 2 * b + 2; i++) {
                                const float(*x)[33] = xch[unit + k * d.hc];
                                o[i][0] += x[2 * t4][4 * g + 2 * (i & 1)];
                                o[i][1] += x[2 * t4 + 1][4 * g + 2 * (i & 1)];
                                o[i][2] += x[2 * t4][4 * g + 2 * (i & 1) + 1];
                                o[i][3] += x[2 * t4 + 1][4 * g + 2 * (i & 1) + 1];
                            }
                    __syncthreads();
                }
            }
            if (active && group == 0) {
                const float L0 = __shfl_sync(0xffffffffu, L, t4 * 8), L1 = __shfl_sync(0xffffffffu, L, t4 * 8 + 4);
                const int head = kvh * G + cg * 8;
                if (whole) {
                    T *out = static_cast<T *>(a.out) + (cur.row * a.n_q + head) * HD;
                    const float i0 = 1.0f / L0, i1 = 1.0f / L1;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const float4 y0 = make_float4(o[2 * b][0] * i0, o[2 * b][2] * i0, o[2 * b + 1][0] * i0, o[2 * b + 1][2] * i0);
                        const float4 y1 = make_float4(o[2 * b][1] * i1, o[2 * b][3] * i1, o[2 * b + 1][1] * i1, o[2 * b + 1][3] * i1);
                        if (2 * t4 < cols) ActVec<T>::store(out + 2 * t4 * HD, b * 8 + g, y0);
                        if (2 * t4 + 1 < cols) ActVec<T>::store(out + (2 * t4 + 1) * HD, b * 8 + g, y1);
                    }
                } else {
                    float *p = d.part + ((int64_t)2 * blockIdx.x + (first_segment ? 0 : 1)) * d.slot_floats + (int64_t)head * (HD + 4);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        if (2 * t4 < cols)
                            *reinterpret_cast<float4 *>(p + 2 * t4 * (HD + 4) + b * 32 + 4 * g) =
                                make_float4(o[2 * b][0], o[2 * b][2], o[2 * b + 1][0], o[2 * b + 1][2]);
                        if (2 * t4 + 1 < cols)
                            *reinterpret_cast<float4 *>(p + (2 * t4 + 1) * (HD + 4) + b * 32 + 4 * g) =
                                make_float4(o[2 * b][1], o[2 * b][3], o[2 * b + 1][1], o[2 * b + 1][3]);
                    }
                    if (t4 == 0 && g < cols) {
                        p[g * (HD + 4) + HD] = M;
                        p[g * (HD + 4) + HD + 1] = L;
                    }
                }
            }
            first_segment = false;
            fresh = true;
        }
        if (left > 1) advance(cur);
        stage_at = stage_at + stage_bytes == ring ? 0 : stage_at + stage_bytes;
        fill_at = fill_at + stage_bytes == ring ? 0 : fill_at + stage_bytes;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Joins the parts of the rows that attn_decode_kernel shared out over several CTAs, and writes the rows that see nothing: a CTA
// per (row, query head); the parts' weights first, one part per thread, then blockDim.x / (32 NB) shares of the parts are summed
// side by side, a value per thread.
constexpr int JOIN_THREADS = 512;
template <typename T> __global__ void __launch_bounds__(JOIN_THREADS) attn_join_kernel(DecodeArgs d) {
    agn_pdl_prologue();
    __shared__ int64_t warp_sums[JOIN_THREADS / 32], mine[2], all;
    __shared__ float weight[2 * ATTN_MAX_SMS], sums[JOIN_THREADS], red[2][JOIN_THREADS / 32];
    __shared__ int slot[2 * ATTN_MAX_SMS];
    const AttnArgs &a = d.a;
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, tid = threadIdx.x, hd = a.hd;
    T *out = static_cast<T *>(a.out) + (t * a.n_q + h) * hd;
    int64_t r0, r1, pre, total;
    scan_rows(a, d.tt, warp_sums, &r0, &r1, &pre, &total);
    if (r0 <= t && t < r1) {
        for (int64_t r = r0; r < t; r++) pre += attn_tiles(a, r, d.tt);
        mine[0] = pre;
        mine[1] = attn_tiles(a, t, d.tt);
        all = total;
    }
    __syncthreads();
    const int64_t w = mine[0], n = mine[1];
    if (n == 0) {
        if (tid < hd) ActVec<T>::store1(out, tid, 0.0f);
        return;
    }
    // CTA x had tiles floor(x W / parts) .. floor((x + 1) W / parts) - 1
    const int x0 = (int)(((w + 1) * d.parts - 1) / all), x1 = (int)(((w + n) * d.parts - 1) / all), nx = x1 - x0 + 1;
    if (nx == 1) return;
    const float *part = d.part + (int64_t)h * (hd + 4);
    float m = -INFINITY, l = 0.0f;
    if (tid < nx) {  // at most 2 * 148 parts
        const int64_t begin = all * (x0 + tid) / d.parts, end = all * (x0 + tid + 1) / d.parts;
        // its first run of tiles is this row's unless the CTA began in an earlier row; a CTA without tiles left nothing
        const int s = begin < end ? 2 * (x0 + tid) + (begin < w ? 1 : 0) : -1;
        slot[tid] = s;
        if (s >= 0) {
            m = part[(int64_t)s * d.slot_floats + hd];
            l = part[(int64_t)s * d.slot_floats + hd + 1];
        }
    }
    float M = agn_warp_max(m);
    if ((tid & 31) == 0) red[0][tid >> 5] = M;
    __syncthreads();
    for (int i = 0; i < JOIN_THREADS / 32; i++) M = fmaxf(M, red[0][i]);
    const float c = ex2(m - (M == -INFINITY ? 0.0f : M));
    if (tid < nx) {
        weight[tid] = slot[tid] >= 0 ? c : 0.0f;
    }
    float L = agn_warp_sum(tid < nx ? l * c : 0.0f);
    if ((tid & 31) == 0) red[1][tid >> 5] = L;
    __syncthreads();
    L = 0.0f;
    for (int i = 0; i < JOIN_THREADS / 32; i++) L += red[1][i];
    const int shares = JOIN_THREADS / hd, share = tid / hd, i = tid % hd;
    float o = 0.0f;
    if (share < shares) {
#pragma unroll 8
        for (int x = share; x < nx; x += shares) {
            const float f = weight[x];
            const float v = f != 0.0f ? part[(int64_t)slot[x] * d.slot_floats + i] : 0.0f;
            o = __fmaf_rn(f, v, o);
        }
    }
    sums[tid] = o;
    __syncthreads();
    if (tid < hd) {
        for (int k = 1; k < shares; k++) o += sums[tid + k * hd];
        ActVec<T>::store1(out, tid, o / L);
    }
}

// The decode kernel's shape for a call: tiles, stages, how the warps share them.
struct DecodePlan {
    int tt, stages, hc, groups, row_stride, seg_bytes, col_groups, chunks, parts, slot_floats;
    size_t smem;
};
constexpr int ATTN_SMEM = 106500;  // of the stages: two CTAs per SM beside their 9 KB of joining buffers

DecodePlan decode_plan(int64_t T, int n_q, int n_kv, int hd, int64_t max_seq, int block_bytes, int sms) {
    DecodePlan p;
    p.hc = n_kv < 8 ? n_kv : 8;
    p.chunks = (n_kv + p.hc - 1) / p.hc;
    p.col_groups = (n_q / n_kv + 7) / 8;
    p.seg_bytes = p.hc * (hd / 32) * block_bytes;
    p.row_stride = (p.seg_bytes - 32 + 127) / 128 * 128 + 32;  // rows 8 banks apart: the four slots a warp reads together do not collide
    const int per_head = 8 / p.hc;  // warps of a head
    p.tt = 128;
    while (p.tt > 8 && 2 * p.tt * p.row_stride > ATTN_SMEM / 3) p.tt /= 2;
    while (p.tt > 16 && p.tt > 8 * per_head && T * ((max_seq + p.tt - 1) / p.tt) < 2 * sms) p.tt /= 2;  // short caches: more CTAs
    p.groups = per_head < p.tt / 8 ? per_head : p.tt / 8;
    while (p.tt / 8 % p.groups) p.groups--;
    p.stages = 3;
    if (2 * p.tt * p.row_stride * 3 > 200 * 1024) p.stages = 2;
    p.smem = (size_t)p.stages * 2 * p.tt * p.row_stride + 16;
    p.slot_floats = n_q * (hd + 4);
    p.parts = 0;
    if (T <= ATTN_MAX_SPLIT_ROWS) {
        const int64_t most = T * ((max_seq + p.tt - 1) / p.tt), fill = 2 * sms / (p.chunks * p.col_groups) > 0 ? 2 * sms / (p.chunks * p.col_groups) : 1;
        p.parts = (int)(most < fill ? most : fill);
    }
    return p;
}

template <typename T, int KV, int NB, int U> int32_t launch_decode_u(agn_ctx *ctx, const DecodePlan &p, const DecodeArgs &d) {
    if (agn_ring_ctas_per_sm(ctx, attn_decode_kernel<T, KV, NB, U>, ATTN_THREADS, p.smem) < 1)
        return agn_fail(ctx, AGN_EINVAL, "attention_kv: a slot of %d bytes needs more shared memory than the device has", d.a.bytes_per_token);
    const dim3 grid((unsigned)(p.parts ? p.parts : d.a.T), (unsigned)(p.chunks * p.col_groups));
    agn_launch(ctx, attn_decode_kernel<T, KV, NB, U>, grid, dim3(ATTN_THREADS), p.smem, d);
    AGN_LAUNCHED(ctx, "attention_kv_decode");
    if (p.parts) {
        agn_launch(ctx, attn_join_kernel<T>, dim3((unsigned)d.a.T, (unsigned)d.a.n_q), dim3(JOIN_THREADS), 0, d);
        AGN_LAUNCHED(ctx, "attention_kv_decode");
    }
    return AGN_OK;
}

template <typename T, int KV, int NB> int32_t launch_decode(agn_ctx *ctx, const DecodePlan &p, const DecodeArgs &d) {
    return p.tt / p.groups % 16 == 0 ? launch_decode_u<T, KV, NB, 2>(ctx, p, d) : launch_decode_u<T, KV, NB, 1>(ctx, p, d);
}

template <typename T, int KV> int32_t launch_decode_kv(agn_ctx *ctx, const DecodePlan &p, const DecodeArgs &d) {
    switch (d.a.hd / 32) {
    case 1: return launch_decode<T, KV, 1>(ctx, p, d);
    case 2: return launch_decode<T, KV, 2>(ctx, p, d);
    case 3: return launch_decode<T, KV, 3>(ctx, p, d);
    case 4: return launch_decode<T, KV, 4>(ctx, p, d);
    case 5: return launch_decode<T, KV, 5>(ctx, p, d);
    case 6: return launch_decode<T, KV, 6>(ctx, p, d);
    case 7: return launch_decode<T, KV, 7>(ctx, p, d);
    default: return launch_decode<T, KV, 8>(ctx, p, d);
    }
}

bool attn_shape_ok(int64_t T, int n_q, int n_kv, int hd, int64_t max_seq) {
    return T >= 0 && T <= 0x7fffffffLL && n_q > 0 && n_kv > 0 && n_q % n_kv == 0 && n_q <= 65535 && hd > 0 && hd <= 256 && hd % 32 == 0 &&
           max_seq > 0 && max_seq <= 0x7fffff00LL;
}

// Two parts per CTA of the decode kernel; the CTAs are as many as the largest part of this architecture holds two of per SM.
int64_t attn_workspace(int64_t T, int n_q, int hd) {
    return T > 0 && T <= ATTN_MAX_SPLIT_ROWS ? (int64_t)2 * 2 * ATTN_MAX_SMS * n_q * (hd + 4) * 4 : 0;
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
    const bool prompt = !pos && sizeof(T) == 2 && agn_attention_prompt_fits(rows, n_q, n_kv, hd);
    const int64_t need = prompt ? agn_attention_prompt_workspace(pos_start + rows, n_kv, hd) : attn_workspace(rows, n_q, hd);
    if (need > 0 && (!workspace || (int64_t)workspace_bytes < need || !agn_aligned16(workspace)))
        return agn_fail(ctx, AGN_EINVAL, "attention_kv: needs %lld bytes of 16-byte aligned workspace", (long long)need);
    AGN_CUDA(ctx, cudaSetDevice(ctx->device));
    AttnArgs a;
    a.q = q; a.out = out; a.k_cache = static_cast<const unsigned char *>(k_cache); a.v_cache = static_cast<const unsigned char *>(v_cache);
    a.pos = pos; a.seq = seq; a.T = rows; a.n_seqs = n_seqs; a.max_seq = max_seq; a.n_q = n_q; a.n_kv = n_kv; a.hd = hd; a.pos_start = pos_start;
    a.bytes_per_token = (int)agn_kv_bytes_per_token(kv_dtype, (int64_t)n_kv * hd); a.scale = scale; a.flags = ctx->d_flags;
    ctx->flags_dirty = true;
    if (prompt) return agn_attention_prompt_f16(ctx, a, kv_dtype, workspace);
    const int block_bytes = kv_dtype == AGN_F16 ? 64 : kv_dtype == AGN_Q8_0 ? 34 : 36;
    const DecodePlan p = decode_plan(rows, n_q, n_kv, hd, max_seq, block_bytes, ctx->sm_count < ATTN_MAX_SMS ? ctx->sm_count : ATTN_MAX_SMS);
    DecodeArgs d;
    d.a = a; d.part = static_cast<float *>(workspace); d.parts = p.parts; d.tt = p.tt; d.stages = p.stages; d.hc = p.hc; d.groups = p.groups;
    d.row_stride = p.row_stride; d.col_groups = p.col_groups; d.slot_floats = p.slot_floats;
    // the widest copy that the caches' address, the row's and the heads' share of it allow
    const int last = (n_kv - (p.chunks - 1) * p.hc) * (hd / 32) * block_bytes;
    const uint64_t bits = (uint64_t)reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | (uint64_t)a.bytes_per_token |
                          (uint64_t)p.seg_bytes | (uint64_t)last | 16;
    d.granule = (int)(bits & (0 - bits));
    DecodePlan use = p;
    if (d.granule < 4) { d.stages = use.stages = 1; use.smem = (size_t)2 * p.tt * p.row_stride + 16; }
    if (kv_dtype == AGN_F16) return launch_decode_kv<T, KV_F16>(ctx, use, d);
    if (kv_dtype == AGN_Q8_0) return launch_decode_kv<T, KV_Q8>(ctx, use, d);
    return launch_decode_kv<T, KV_WORDS>(ctx, use, d);
}

}  // namespace

extern "C" int64_t agn_attention_kv_workspace_bytes(int64_t T, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int64_t max_seq_len,
                                                    int32_t has_pos) {
    if (!attn_shape_ok(T, n_q_heads, n_kv_heads, head_dim, max_seq_len)) return 0;
    const int64_t decode = attn_workspace(T, n_q_heads, head_dim);
    if (has_pos || !agn_attention_prompt_fits(T, n_q_heads, n_kv_heads, head_dim)) return decode;
    const int64_t prompt = agn_attention_prompt_workspace(max_seq_len, n_kv_heads, head_dim);
    return prompt > decode ? prompt : decode;
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
