// Attention of single rows (any position of any sequence) over the KV cache: the decode step.  One .cu per cache layout instantiates the kernel.
//
// A slot's 2 * bytes_per_token bytes are read once for all query heads, which bounds it by HBM in principle; what holds it is the issue of instructions (57 % of the
// slots of 16 warps an SM, 368 instructions per 8 slots and head): 64 rows of up to 32768 slots, 28/4 heads of 128, q8_0 in words, 1.24 GB in 323-328 us, 3.8 TB/s;
// 8 rows of 5000 to 8192 f16 slots, 32/8 heads of 128, 59.7 us, 3.8 TB/s.  What a CTA works on is a run of tiles of TT slots: all
// rows' tiles are numbered one after the other and shared out evenly (a batch of very different lengths, or one long row, fills the GPU alike);
// a row that falls into several CTAs is joined by attn_join_kernel.  Tiles arrive by cp.async in a ring of stages, all KV heads of a slot
// together, and each warp takes one KV head (and a share of the tile's slots where there are fewer than 8).
//
// Per 8 slots and head, on the matrix units so that the instructions per cached byte stay below what the stream allows:
//   S = Q K^T as m16n8k16 f16: rows 0-7 hold the upper halves of the (up to 8) query heads, rows 8-15 the lower halves (q = hi + lo, each 11 bits,
//     after a power of two has brought the row's largest value to [2^14, 2^15)), the columns are slots; the cached bytes are exact in f16, so a score
//     keeps 22 bits; block scales are applied to the f32 products of 32 dims.
//   O^T += V^T P^T as m16n8k8 tf32, twice: p * scale split into two tf32 parts (22 bits, any range), V's bytes exact in tf32.
//     The accumulators of S are P^T's operand layout as they are (columns 2t, 2t + 1 stand for slots t, t + 4).  f16 rows take both parts too: the upper one alone
//     saves 5 % over words and nothing over an f16 cache, and is off by 2.8e-4 instead of the 2.1e-4 that rounding the result costs.
// The running maximum is a reference that is moved only when a row has outgrown it by 2^8, so that the accumulators are rarely rescaled.
#pragma once
#include <math.h>

#include "agn_attention.cuh"

constexpr int ATTN_THREADS = 256, ATTN_WARPS = 8, ATTN_MAX_SPLIT_ROWS = 512;

struct DecodeArgs {
    AttnArgs a;
    float *part;  // [2 * parts][n_q][hd + 4]: sums of weighted values, maximum (log2), sum of weights
    int parts;    // CTAs along x; 0: one CTA per row, no joining
    int act16;
    int tt, stages, hc, groups, row_stride, granule, col_groups, slot_floats;
};

// A row of hc heads in shared memory: 8 banks off a multiple of 32, so that the four slots that a warp's lanes read together do not collide.
__host__ __device__ constexpr int attn_row_stride(int seg_bytes) { return (seg_bytes - 32 + 127) / 128 * 128 + 32; }
// Slots that a warp takes from a tile: as many as 8 warps' tiles of K and V stay near 35 KB, a third of what two CTAs per SM have each.
__host__ __device__ constexpr int attn_slots_per_warp(bool f16) { return f16 ? 8 : 16; }

// Tile w of W is in part x where start(x) <= w < start(x + 1).
struct AttnShares {
    int64_t share, extra;
    __device__ AttnShares(int64_t total, int parts) {
        if (total < 0x7fffffffLL) {
            share = (uint32_t)total / (uint32_t)parts;
            extra = (uint32_t)total % (uint32_t)parts;
        } else {
            share = total / parts;
            extra = total % parts;
        }
    }
    __device__ int64_t start(int x) const { return x * share + (x < extra ? x : extra); }
    __device__ int part(int64_t w) const {
        const int64_t big = extra * (share + 1);
        if (w < big) return (int)(w < 0x7fffffffLL ? (uint32_t)w / (uint32_t)(share + 1) : w / (share + 1));
        return (int)(extra + (w - big < 0x7fffffffLL && share < 0x7fffffffLL ? (uint32_t)(w - big) / (uint32_t)share : (w - big) / share));
    }
};

#ifdef __CUDACC__

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
// The power of two that brings a query row's largest value to [2^14, 2^15), where the two f16 parts keep 22 bits of all values down to 2^-17 of it and lose what is
// below 2^-39 of it; returns what its scores then have to be multiplied by for the softmax in base 2 (not 0: -inf times that is -inf).
__device__ __forceinline__ float query_scale(float amax, float scale, float &up) {
    const int e = min(max((int)(__float_as_uint(amax) >> 23), 15), 254);  // 2^(e-127) <= amax < 2^(e-126)
    up = __uint_as_float((uint32_t)(268 - e) << 23);                        // 2^(141-e)
    return fmaxf(scale * 1.4426950408889634f * __uint_as_float((uint32_t)(e - 14) << 23), 1.17549435e-38f);
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

struct agn_true { static constexpr bool value = true; };
struct agn_false { static constexpr bool value = false; };
// queries and output, f32 or f16
__device__ __forceinline__ float4 load_act4(const DecodeArgs &d, int64_t at, int vec) {
    return d.act16 ? ActVec<__half>::load(static_cast<const __half *>(d.a.q) + at, vec) : ActVec<float>::load(static_cast<const float *>(d.a.q) + at, vec);
}
__device__ __forceinline__ void store_act4(const DecodeArgs &d, int64_t at, int vec, float4 v) {
    if (d.act16) ActVec<__half>::store(static_cast<__half *>(d.a.out) + at, vec, v);
    else ActVec<float>::store(static_cast<float *>(d.a.out) + at, vec, v);
}
__device__ __forceinline__ void store_act(const DecodeArgs &d, int64_t at, float v) {
    if (d.act16) static_cast<__half *>(d.a.out)[at] = __float2half_rn(v);
    else static_cast<float *>(d.a.out)[at] = v;
}

struct RowCursor {
    int64_t row, off;
    int n, j;  // visible slots, next slot
};

__device__ __forceinline__ int64_t attn_tiles(const AttnArgs &a, int64_t t, int tt) {
    int64_t off;
    return ((uint32_t)attn_row(a, t, &off) + (uint32_t)tt - 1) / (uint32_t)tt;
}

// Tiles of all rows before each thread's share of the rows (at most ATTN_MAX_SPLIT_ROWS), and of all rows.
__device__ __forceinline__ void scan_rows(const AttnArgs &a, int tt, int64_t *warp_sums, int64_t *r0, int64_t *r1, int64_t *before, int64_t *total) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    const int rows = (int)a.T, per = (rows + (int)blockDim.x - 1) / (int)blockDim.x;
    *r0 = min(tid * per, rows);
    *r1 = min((tid + 1) * per, rows);
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

// HC: the KV heads of a slot that a CTA takes (1, 2, 4, 8), which fixes tile and row layout at compile time; 0: any number, from the arguments.
template <int KV, int NB, int HC> __global__ void __launch_bounds__(ATTN_THREADS, NB <= 4 ? 2 : 1) attn_decode_kernel(const __grid_constant__ DecodeArgs d) {
    agn_pdl_prologue();
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float xch[ATTN_WARPS][8][33], sm[ATTN_WARPS][8], sl[ATTN_WARPS][8];
    __shared__ int64_t warp_sums[ATTN_WARPS], first_row, first_pre;
    const AttnArgs &a = d.a;
    using F = KvFormat<KV>;
    constexpr int HD = NB * 32, PER = attn_slots_per_warp(KV == KV_F16), U = PER / 8;
    const int HCV = HC ? HC : d.hc, GROUPS = HC ? 8 / (HC ? HC : 1) : d.groups, TT = PER * GROUPS;
    const int RS = HC ? attn_row_stride(HC * NB * F::BYTES) : d.row_stride;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int cg = blockIdx.y % d.col_groups, h0 = blockIdx.y / d.col_groups * HCV, hc = HC ? HC : min(HCV, a.n_kv - h0);
    const int unit = warp % HCV, group = warp / HCV;
    const bool active = HC ? true : unit < hc && group < GROUPS;
    const int G = a.n_q / a.n_kv, kvh = h0 + unit, cols = min(8, G - cg * 8), head = kvh * G + cg * 8;

    // ---- this CTA's run of tiles
    RowCursor cur;
    int left;
    if (d.parts == 0) {
        cur.row = blockIdx.x;
        cur.n = attn_row(a, cur.row, &cur.off);
        cur.j = 0;
        left = ((uint32_t)cur.n + (uint32_t)TT - 1) / (uint32_t)TT;
        if (left == 0 && active && group == 0)  // a row that sees nothing
            for (int i = lane; i < cols * HD; i += 32) store_act(d, (cur.row * a.n_q + head) * HD + i, 0.0f);
    } else {
        cur.row = 0;
        cur.n = attn_row(a, 0, &cur.off);  // of a single row, or one that the scan below moves on from
        int64_t w0, w1, pre0 = 0;
        if (a.T == 1) {
            const AttnShares shares(((uint32_t)cur.n + (uint32_t)TT - 1) / (uint32_t)TT, d.parts);
            w0 = shares.start(blockIdx.x);
            w1 = shares.start(blockIdx.x + 1);
        } else {
            int64_t r0, r1, pre, total;
            scan_rows(a, TT, warp_sums, &r0, &r1, &pre, &total);
            const AttnShares shares(total, d.parts);
            w0 = shares.start(blockIdx.x);
            w1 = shares.start(blockIdx.x + 1);
            for (int64_t t = r0; t < r1; t++) {
                const int64_t n = attn_tiles(a, t, TT);
                if (w0 >= pre && w0 < pre + n) { first_row = t; first_pre = pre; }
                pre += n;
            }
            __syncthreads();
            if (w1 > w0) {
                cur.row = first_row;
                pre0 = first_pre;
                cur.n = attn_row(a, cur.row, &cur.off);
            }
        }
        left = (int)(w1 - w0);
        cur.j = (int)(w0 - pre0) * TT;
    }
    if (left <= 0) return;

    // ---- tiles into the ring
    const int bpt = a.bytes_per_token, side = TT * RS, stage_bytes = 2 * side, ring = d.stages * stage_bytes;
    const uint32_t smem0 = agn_smem_u32(smem);
    auto copy_tile = [&](const RowCursor &c, uint32_t stage_at, auto wide) {  // wide: pieces of 16 bytes
        constexpr bool W = decltype(wide)::value;
        const int granule = W ? 16 : d.granule, cpr = hc * NB * F::BYTES / granule;
        const int step_tok = ATTN_THREADS / cpr, step_rem = ATTN_THREADS % cpr;
        const int64_t base = c.off + (int64_t)c.j * bpt + (int64_t)h0 * NB * F::BYTES;
        const unsigned char *ks = a.k_cache + base, *vs = a.v_cache + base;
        const int valid = min(TT, c.n - c.j);
        int tok = tid / cpr, rem = tid % cpr;
        for (int i = tid; i < cpr * TT; i += ATTN_THREADS) {
            const bool in = tok < valid;  // slots that the row does not see are zeros, not what the cache holds there
            const uint32_t from = in ? tok * bpt + rem * granule : 0, dst = smem0 + stage_at + tok * RS + rem * granule;
            if (W) {
                cp_async<16>(dst, ks + from, in);
                cp_async<16>(dst + side, vs + from, in);
            } else if (granule == 8) {
                cp_async<8>(dst, ks + from, in);
                cp_async<8>(dst + side, vs + from, in);
            } else if (granule == 4) {
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
            if (rem >= cpr) {
                rem -= cpr;
                tok++;
            }
        }
    };
    // Whole tiles in pieces of 16 bytes where the layout is fixed: this thread's pieces as running pointers.
    constexpr int CPR = HC * NB * F::BYTES / 16, STEP_T = CPR ? ATTN_THREADS / (CPR ? CPR : 1) : 0, STEP_R = CPR ? ATTN_THREADS % (CPR ? CPR : 1) : 0;
    const int tok0 = HC ? tid / (CPR ? CPR : 1) : 0, rem0 = HC ? tid % (CPR ? CPR : 1) : 0;
    const int src0 = tok0 * bpt + rem0 * 16, dst0 = tok0 * RS + rem0 * 16;
    auto issue = [&](const RowCursor &c, uint32_t stage_at) {
        if (d.granule != 16) {
            copy_tile(c, stage_at, agn_false());
        } else if (HC && c.n - c.j >= TT) {
            const int64_t base = c.off + (int64_t)c.j * bpt + (int64_t)h0 * NB * F::BYTES + src0;
            const unsigned char *ks = a.k_cache + base, *vs = a.v_cache + base;
            uint32_t dst = smem0 + stage_at + dst0;
            int rem = rem0;
#pragma unroll
            for (int i = 0; i < (CPR * PER * (HC ? 8 / (HC ? HC : 1) : 1) + ATTN_THREADS - 1) / ATTN_THREADS; i++) {
                if (tid + i * ATTN_THREADS < CPR * TT) {
                    cp_async<16>(dst, ks, true);
                    cp_async<16>(dst + side, vs, true);
                }
                rem += STEP_R;
                const bool wrap = rem >= CPR;
                const int src_step = STEP_T * bpt + STEP_R * 16 + (wrap ? bpt - CPR * 16 : 0);
                dst += STEP_T * RS + STEP_R * 16 + (wrap ? RS - CPR * 16 : 0);
                ks += src_step;
                vs += src_step;
                if (wrap) rem -= CPR;
            }
        } else {
            copy_tile(c, stage_at, agn_true());
        }
    };
    auto advance = [&](RowCursor &c) {
        c.j += TT;
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
    const int lane_k = unit * NB * F::BYTES + (group * PER + (g >> 1) + (g & 1) * 4) * RS;  // the slot whose key this lane reads
    const int lane_s = unit * NB * F::BYTES + (group * PER + t4) * RS;                      // the first slot whose score and value it holds

    // Slots cur.j + group * PER + 8 u + t4 (+ 4); EDGE: some of them are behind the row's end.
    auto slots = [&](auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        const unsigned char *kb = smem + stage_at + lane_k, *sb = smem + stage_at + lane_s, *vb = sb + side;
        float sc[U][2];
#pragma unroll
        for (int u = 0; u < U; u++) {
            sc[u][0] = sc[u][1] = 0.0f;
            const unsigned char *krow = kb + 8 * u * RS, *k0 = sb + 8 * u * RS, *k1 = k0 + 4 * RS;
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (KV == KV_F16) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(krow + b * 64 + t4 * 16);
                    mma_f16(acc, q[2 * b], w.x, w.y);
                    mma_f16(acc, q[2 * b + 1], w.z, w.w);
                    // blocks of dims are added up by rounded additions, too (the matrix unit's cuts over all dims reach 6e-6 of a result)
                    sc[u][0] += acc[0] + acc[2];
                    sc[u][1] += acc[1] + acc[3];
                    acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
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
        }
        float mt = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (EDGE) {
                const int j = cur.j + group * PER + 8 * u + t4;
                if (j >= cur.n) sc[u][0] = -INFINITY;
                if (j + 4 >= cur.n) sc[u][1] = -INFINITY;
            }
            mt = fmaxf(mt, fmaxf(sc[u][0], sc[u][1]));
        }
        mt *= coef;  // coef > 0
        if (__any_sync(0xffffffffu, mt > m + 8.0f)) {  // true at a row's first slots
            mt = fmaxf(m, mt);
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
            const float c = ex2(m - (mt == -INFINITY ? 0.0f : mt));
            l *= c;
            const float c0 = __shfl_sync(0xffffffffu, c, t4 * 8), c1 = __shfl_sync(0xffffffffu, c, t4 * 8 + 4);
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) { o[i][0] *= c0; o[i][1] *= c1; o[i][2] *= c0; o[i][3] *= c1; }
            m = mt;
        }
        const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int u = 0; u < U; u++) {
            sc[u][0] = ex2(__fmaf_rn(sc[u][0], coef, -mu));
            sc[u][1] = ex2(__fmaf_rn(sc[u][1], coef, -mu));
            l += sc[u][0] + sc[u][1];
        }
        // The matrix unit's adder cuts what it shifts out: products of a few slots are summed there and the running sums are kept by rounded
        // additions (over thousands of slots the cuts would add up to 5e-6 of the result).
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
                    const unsigned char *blk = vb + (8 * u + 4 * i) * RS + b * F::BYTES;
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
    };

    for (; left > 0; left--) {
        if (fresh) {
            fresh = false;
            seg_start = cur.j;
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            const bool there = active && g < cols;
            const int64_t at = (cur.row * a.n_q + (there ? head + g : 0)) * HD;
            float amax = 0.0f;
            float4 x[2 * NB];
#pragma unroll
            for (int b = 0; b < 2 * NB; b++) {
                x[b] = there ? load_act4(d, at, (b >> 1) * 8 + 2 * t4 + (b & 1)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x[b].x), fabsf(x[b].y))), fmaxf(fabsf(x[b].z), fabsf(x[b].w)));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            float up;
            coef = query_scale(amax, a.scale, up);
#pragma unroll
            for (int b = 0; b < 2 * NB; b++) {
                const float v[4] = {x[b].x * up, x[b].y * up, x[b].z * up, x[b].w * up};
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
            if (cur.j + TT <= cur.n) slots(agn_false());
            else if (cur.j + group * PER < cur.n) slots(agn_true());
        }
        if (d.stages == 1) __syncthreads();
        const bool row_done = cur.j + TT >= cur.n;
        if (row_done || left == 1) {  // the end of a row, or of this CTA's part of one
            const bool whole = row_done && seg_start == 0;
            float lt = l + __shfl_xor_sync(0xffffffffu, l, 1);
            lt += __shfl_xor_sync(0xffffffffu, lt, 2);
            float M = m, L = lt;
            if (GROUPS > 1) {  // join the shares of a head's warps
                __syncthreads();
                if (t4 == 0) { sm[warp][g] = m; sl[warp][g] = lt; }
                __syncthreads();
                for (int k = 0; k < GROUPS; k++) M = fmaxf(M, sm[unit + k * HCV][g]);
                L = 0.0f;
                for (int k = 0; k < GROUPS; k++) L += sl[unit + k * HCV][g] * ex2(sm[unit + k * HCV][g] - (M == -INFINITY ? 0.0f : M));
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
                        for (int k = 1; k < GROUPS; k++)
#pragma unroll
                            for (int i = 2 * b; i < 2 * b + 2; i++) {
                                const float(*x)[33] = xch[unit + k * HCV];
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
                if (whole) {
                    const int64_t at = (cur.row * a.n_q + head) * HD;
                    const float i0 = 1.0f / L0, i1 = 1.0f / L1;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const float4 y0 = make_float4(o[2 * b][0] * i0, o[2 * b][2] * i0, o[2 * b + 1][0] * i0, o[2 * b + 1][2] * i0);
                        const float4 y1 = make_float4(o[2 * b][1] * i1, o[2 * b][3] * i1, o[2 * b + 1][1] * i1, o[2 * b + 1][3] * i1);
                        if (2 * t4 < cols) store_act4(d, at + 2 * t4 * HD, b * 8 + g, y0);
                        if (2 * t4 + 1 < cols) store_act4(d, at + (2 * t4 + 1) * HD, b * 8 + g, y1);
                    }
                } else {
                    float *p = d.part + ((int64_t)2 * blockIdx.x + (first_segment ? 0 : 1)) * d.slot_floats + (int64_t)head * (HD + 4);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        if (2 * t4 < cols)
                            *reinterpret_cast<float4 *>(p + 2 * t4 * (HD + 4) + b * 32 + 4 * g) = make_float4(o[2 * b][0], o[2 * b][2], o[2 * b + 1][0], o[2 * b + 1][2]);
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

template <int KV, int NB, int HC> int32_t launch_decode_as(agn_ctx *ctx, const DecodeArgs &d, dim3 grid, size_t smem) {
    if (agn_ring_ctas_per_sm(ctx, attn_decode_kernel<KV, NB, HC>, ATTN_THREADS, smem) < 1)
        return agn_fail(ctx, AGN_EINVAL, "attention_kv: a slot of %d bytes needs more shared memory than the device has", d.a.bytes_per_token);
    agn_launch(ctx, attn_decode_kernel<KV, NB, HC>, grid, dim3(ATTN_THREADS), smem, d);
    AGN_LAUNCHED(ctx, "attention_kv_decode");
    return AGN_OK;
}

// Fixed layouts for the head sizes 64 and 128 with 1, 2, 4 or 8 heads to a CTA: 16 rows of 32768 slots, 28/4 heads of 128, q8_0 in words, 164 us against 187
// with the layout from the arguments; 8 rows of 8192, 32/8 heads, f16 cache, 64 against 72.
template <int KV, int NB> int32_t launch_decode_nb(agn_ctx *ctx, const DecodeArgs &d, dim3 grid, size_t smem) {
    if (NB == 2 || NB == 4) {
        if (d.granule == 16 && d.stages > 1) {
            if (d.hc == 1) return launch_decode_as<KV, NB, NB == 2 || NB == 4 ? 1 : 0>(ctx, d, grid, smem);
            if (d.hc == 2) return launch_decode_as<KV, NB, NB == 2 || NB == 4 ? 2 : 0>(ctx, d, grid, smem);
            if (d.hc == 4) return launch_decode_as<KV, NB, NB == 2 || NB == 4 ? 4 : 0>(ctx, d, grid, smem);
            if (d.hc == 8 && d.a.n_kv % 8 == 0) return launch_decode_as<KV, NB, NB == 2 || NB == 4 ? 8 : 0>(ctx, d, grid, smem);
        }
    }
    return launch_decode_as<KV, NB, 0>(ctx, d, grid, smem);
}

template <int KV> int32_t launch_decode(agn_ctx *ctx, const DecodeArgs &d, dim3 grid, size_t smem) {
    switch (d.a.hd / 32) {
    case 1: return launch_decode_nb<KV, 1>(ctx, d, grid, smem);
    case 2: return launch_decode_nb<KV, 2>(ctx, d, grid, smem);
    case 3: return launch_decode_nb<KV, 3>(ctx, d, grid, smem);
    case 4: return launch_decode_nb<KV, 4>(ctx, d, grid, smem);
    case 5: return launch_decode_nb<KV, 5>(ctx, d, grid, smem);
    case 6: return launch_decode_nb<KV, 6>(ctx, d, grid, smem);
    case 7: return launch_decode_nb<KV, 7>(ctx, d, grid, smem);
    default: return launch_decode_nb<KV, 8>(ctx, d, grid, smem);
    }
}

#endif  // __CUDACC__

int32_t agn_attention_decode_f16(agn_ctx *ctx, const DecodeArgs &d, dim3 grid, size_t smem);
int32_t agn_attention_decode_q8(agn_ctx *ctx, const DecodeArgs &d, dim3 grid, size_t smem);
int32_t agn_attention_decode_words(agn_ctx *ctx, const DecodeArgs &d, dim3 grid, size_t smem);
