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
// between the four warps.  64 sequences of one row, 16/32 heads of 128: 49 us, 5.5 TB/s.
constexpr int TB = 8;  // tokens whose q, k, v are staged at a time
template <int DK> __global__ void __launch_bounds__(128, 6) delta_recurrent_kernel(const __grid_constant__ DeltaArgs a) {
    agn_pdl_prologue();
    constexpr int R = DK / 16;
    __shared__ __align__(16) float sq[TB][DK], sk[TB][DK], sv[TB][32];
    __shared__ float sa[TB], sb[TB], sqk[TB];
    __shared__ __align__(16) float red[2][4][2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = blockIdx.x * 32, h = blockIdx.y, hk = h / (a.n_v / a.n_k);
    const int64_t s = blockIdx.z;
    const int rg = warp * 4 + (lane >> 3), c4 = (lane & 7) * 4;
    const int64_t soff = ((s * a.n_v + h) * DK + rg) * a.dv + c0 + c4;
    float4 S[R];  // on its way before anything else: the longest wait of a short call
#pragma unroll
    for (int i = 0; i < R; i++)
        S[i] = a.state_in ? __ldcs(reinterpret_cast<const float4 *>(a.state_in + soff + (int64_t)16 * i * a.dv)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    int64_t b, e;
    delta_rows(a, s, &b, &e);
    for (int64_t t0 = b; t0 < e; t0 += TB) {
        const int cnt = (int)(e - t0 < TB ? e - t0 : TB);
        __syncthreads();
        for (int i = warp; i < cnt; i += 4) {
            const int64_t t = t0 + i;
            constexpr int V = DK / 32;
            float qv[V], kv[V], qq = 0.0f, kk = 0.0f, qk = 0.0f;
            const float vv = a.v[t * a.v_stride + h * a.dv + c0 + lane], gv = a.g[t * a.n_v + h], bv = a.beta[t * a.n_v + h];
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
            sv[i][lane] = vv;
            if (lane == 0) {
                sa[i] = expf(gv);
                sb[i] = bv;
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
    for (int i = 0; i < R; i++) __stcs(reinterpret_cast<float4 *>(a.state_out + soff + (int64_t)16 * i * a.dv), S[i]);
}

// ---- Chunked form, for prompts -----------------------------------------------------------------------------------------
//
// Inside a chunk of C = 64 rows, with c_i = a_1 ... a_i and r_ij = a_(j+1) ... a_i (products, so a decay of 0 needs no care):
//   A_ij = beta_i r_ij k_i.k_j (i > j),   N = (I + A)^-1 diag(beta),   P_ij = r_ij q_i.k_j (i >= j)
//   D = N (V - diag(c) K S),   O = diag(c) Q S + P D,   S' = c_C S + K^T diag(r_Cj) D
// delta_prepare_kernel computes N, P, c, r_C and the normalised q and k of every chunk side by side; delta_chunk_kernel carries 32
// columns of one head's state from chunk to chunk (the columns are independent: 128 CTAs for one sequence of 32 heads of 128).
//
// Bound by the matrix units (59 % busy on the SMs at work: 1.05 M multiply-adds per chunk and 32 columns, three times over, at tf32's rate) and by the waits between
// dependent products; a chunk takes 6 us.  4096 rows of 16/32 heads of 128: 92 us of preparation and 388 us of chunks.  Every product is taken in two parts of 11
// bits each, x = hi + lo, as hi hi + hi lo + lo hi, summed in f32.  K, Q, N and P are f16 parts in the workspace, every row brought to UP by a power of two of its own
// (its largest entry; a row of one product is a row of the result, which takes the factor back), so that a small key, query or write strength keeps its bits;
// f16 is exact in tf32.  S, V - c K S, D and r D stay f32 in shared memory and are split into tf32 parts, which have f32's range, as they are read: columns do not share a
// scale, so that one of another size, a large row later in the chunk or a state that has decayed takes no bits from the rest.  (f16 parts under one power of two per 32
// columns and chunk, at m16n8k16's double rate: 239 us of chunks, but a column 2^-20 of its neighbour had ten bits left.  bf16 for the two mixed products: 367 us, twice the
// error.  Sixteen workers of eight columns each: 430 us.)  Errors do not grow from row to row where 0 <= beta <= 2, g <= 0 and |k| <= 1; products neither
// overflow nor lose their lower parts where the largest state or value lies between 2^-90 and 2^112.  A chunk that is not so is computed row by row in f32 instead.
constexpr int CH = 64, CHUNK_THREADS = 256, CARRY_THREADS = CHUNK_THREADS + 128;
constexpr float UP = 1024.0f, DOWN = 1.0f / UP;  // rows' largest entries lie in [UP, 2 UP); what is kept of the others is 2^-35 of that or better

// A row whose largest entry is m times `up` has it in [UP, 2 UP); times `down`, it is what it was.
__device__ __forceinline__ void row_scale(float m, float &up, float &down) {
    const int e = min(max((int)(__float_as_uint(m) >> 23), 11), 254);  // from 2^-116 on
    up = __uint_as_float((uint32_t)(264 - e) << 23);
    down = __uint_as_float((uint32_t)(e - 10) << 23);
}
// Per chunk and value head, for its rows' results: RF_X: c_i times K's factor (of K S), RF_QS: c_i times Q's, RF_D: N's, RF_R: r_Ci times K's (of r D, in front of K^T),
// RF_PD: P's; then c_C.  Factors of products with an operand that has been brought down (by DOWN) include UP.
constexpr int RF_X = 0, RF_QS = 64, RF_D = 128, RF_R = 192, RF_PD = 256, RF_C = 320, ROW_FACTORS = 324;

// The workspace holds the operands as they stand in shared memory, rows 16 bytes off a multiple of 128 (so that the eight rows of a fragment do not collide):
// a chunk's K, Q, N or P is one bulk copy.
__host__ __device__ constexpr int kq_row(int dk) { return dk + 8; }
constexpr int NP_ROW = CH + 8;

struct ChunkArgs {
    DeltaArgs d;
    __half *kq;      // [slots][n_k][k hi, k lo, q hi, q lo][64][kq_row]
    __half *np;      // [slots][n_v][N hi, N lo, P hi, P lo][64][NP_ROW]
    float *factors;  // [slots][n_v][ROW_FACTORS]
    int *odd;        // [slots][n_v]: the chunk breaks the bounds
    int spin;
};

// A sequence's chunks have slots of their own: sequence s from slot b_s / 64 + s on.
__device__ __forceinline__ int64_t delta_slot(int64_t begin, int64_t s) { return begin / CH + s; }

__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(agn_smem_u32(p)) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(agn_smem_u32(p)) : "memory");
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&d)[4], const float *a, float b0, float b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// A 16 x 16 fragment of f16 operands (four registers as ldmatrix gives them) as the operands of two products of eight: slots t4 and t4 + 4 of the first one stand
// for columns 2 t4 and 2 t4 + 1, those of the second one for columns 2 t4 + 8 and 2 t4 + 9.  f16 is exact in tf32.
__device__ __forceinline__ void half_to_tf32(const uint32_t (&r)[4], float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&r[i]));
        f[(i >> 1) * 4 + (i & 1)] = x.x;
        f[(i >> 1) * 4 + (i & 1) + 2] = x.y;
    }
}
// The other operand, 16 rows from b on (this lane's column), split into two tf32 parts on its way: hi rounded to 11 bits, lo the rest.
struct Split16 {
    float hi[4], lo[4];
    __device__ __forceinline__ Split16(const float *b, int row) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = b[((i >> 1) * 8 + (i & 1)) * row];
            hi[i] = __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
            lo[i] = x - hi[i];
        }
    }
};
// big += hi hi, small += hi lo + lo hi: apart, because the matrix unit's adder cuts what is below the sum's last bit
__device__ __forceinline__ void mma_split(float (&big)[4], float (&small)[4], const float (&ah)[8], const float (&al)[8], const Split16 &b) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        mma8(big, ah + 4 * i, b.hi[2 * i], b.hi[2 * i + 1]);
        mma8(small, ah + 4 * i, b.lo[2 * i], b.lo[2 * i + 1]);
        mma8(small, al + 4 * i, b.hi[2 * i], b.hi[2 * i + 1]);
    }
}
__device__ __forceinline__ void cp16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(agn_smem_u32(dst)), "l"(src) : "memory");
}

// One CTA per (chunk slot, key head); the value heads of the key head share its two products.
constexpr int TROW = CH + 4;  // floats: four of them at a multiple of 16 bytes
template <int DK> struct PrepSmem {
    static constexpr int ROW = kq_row(DK);
    union {
        __half op[4][CH * ROW];  // k hi, k lo, q hi, q lo
        struct {
            float kk[CH][TROW], qk[CH][TROW], A[CH][TROW], N[CH][TROW];
        } t;
    };
    float down[2][CH];  // factors of the rows of k, of q
    float a[CH], beta[CH], whole[8], tail[CH];  // products of a over eight rows, over the rows behind a column up to the end of its eight
    int odd_kq, odd;
};

// The blocks N_21 = -N_22 (A_21 N_11) of size B below the diagonal blocks of size B, four values side by side per thread; A_21's place takes the inner product.
template <int B> __device__ __forceinline__ void lower_block(float (&A)[CH][TROW], float (&N)[CH][TROW], int tid) {
    constexpr int TPB = B * B / 4;  // threads of a block
    const int base = tid / TPB * 2 * B, row = tid % TPB / (B / 4), col = tid % (B / 4) * 4;
    const bool on = tid < CH / (2 * B) * TPB;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (on) {
            const float *u = half ? &N[base + B + row][base + B] : &A[base + B + row][base];
#pragma unroll
            for (int l = 0; l < B; l += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(u + l);
                const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float4 w = *reinterpret_cast<const float4 *>(half ? &A[base + B + l + k][base + col] : &N[base + l + k][base + col]);
                    y.x = __fmaf_rn(fs[k], w.x, y.x); y.y = __fmaf_rn(fs[k], w.y, y.y);
                    y.z = __fmaf_rn(fs[k], w.z, y.z); y.w = __fmaf_rn(fs[k], w.w, y.w);
                }
            }
        }
        __syncthreads();
        if (on) {
            if (half) *reinterpret_cast<float4 *>(&N[base + B + row][base + col]) = make_float4(-y.x, -y.y, -y.z, -y.w);
            else *reinterpret_cast<float4 *>(&A[base + B + row][base + col]) = y;
        }
        __syncthreads();
    }
}

template <int DK> __global__ void __launch_bounds__(CHUNK_THREADS, 3) delta_prepare_kernel(const __grid_constant__ ChunkArgs x) {
    agn_pdl_prologue();
    extern __shared__ __align__(128) unsigned char raw[];
    PrepSmem<DK> &sm = *reinterpret_cast<PrepSmem<DK> *>(raw);
    constexpr int ROW = PrepSmem<DK>::ROW;
    const DeltaArgs &d = x.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hk = blockIdx.y;
    const int64_t slot = blockIdx.x;
    // the sequence: the last one that begins at or before this slot
    int64_t lo = 0, hi = d.n_seqs - 1, b, e;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) / 2;
        delta_rows(d, mid, &b, &e);
        if (delta_slot(b, mid) <= slot) lo = mid;
        else hi = mid - 1;
    }
    delta_rows(d, lo, &b, &e);
    const int64_t first = b + (slot - delta_slot(b, lo)) * CH;
    if (first < b || first >= e) return;
    const int rows = (int)(e - first < CH ? e - first : CH);
    if (tid == 0) sm.odd_kq = 0;
    __syncthreads();

    // q and k, eight rows per warp, all loads ahead of the first use
    constexpr int V = DK / 32;
    float v[8][2][V];
#pragma unroll
    for (int n = 0; n < 8; n++) {
        const int i = warp * 8 + n;
#pragma unroll
        for (int w = 0; w < 2; w++) {
            const float *src = w == 0 ? d.k + (first + i) * d.k_stride + hk * DK : d.q + (first + i) * d.q_stride + hk * DK;
#pragma unroll
            for (int j = 0; j < V / 2; j++) {
                const float2 y = i < rows ? *reinterpret_cast<const float2 *>(src + 2 * (lane + 32 * j)) : make_float2(0.0f, 0.0f);
                v[n][w][2 * j] = y.x;
                v[n][w][2 * j + 1] = y.y;
            }
        }
    }
#pragma unroll
    for (int n = 0; n < 8; n++) {
        const int i = warp * 8 + n;
#pragma unroll
        for (int w = 0; w < 2; w++) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < V; j++) ss = __fmaf_rn(v[n][w][j], v[n][w][j], ss);
            ss = agn_warp_sum(ss);
            const float f = i >= rows ? 0.0f : d.eps >= 0.0f ? rsqrtf(ss + d.eps) : 1.0f;
            // the normalised row's norm is at most 1 unless a sum of squares overflowed or was not a number; a query may have any
            if (lane == 0 && !(d.eps >= 0.0f ? ss < INFINITY && (ss + d.eps > 0.0f || i >= rows) : ss < (w == 0 ? 1.01f : INFINITY))) sm.odd_kq = 1;
            float most = 0.0f, up, down;
#pragma unroll
            for (int j = 0; j < V; j++) {
                v[n][w][j] *= f;
                most = fmaxf(most, fabsf(v[n][w][j]));
            }
            row_scale(agn_warp_max(most), up, down);
            if (lane == 0) sm.down[w][i] = down;
            __half *g = x.kq + (((slot * d.n_k + hk) * 4 + 2 * w) * CH + i) * ROW;
#pragma unroll
            for (int j = 0; j < V / 2; j++) {
                uint32_t h2, l2;
                split2(v[n][w][2 * j] * up, v[n][w][2 * j + 1] * up, h2, l2);
                const int at = 2 * (lane + 32 * j);
                *reinterpret_cast<uint32_t *>(&sm.op[2 * w][i * ROW + at]) = h2;
                *reinterpret_cast<uint32_t *>(&sm.op[2 * w + 1][i * ROW + at]) = l2;
                *reinterpret_cast<uint32_t *>(g + at) = h2;
                *reinterpret_cast<uint32_t *>(g + CH * ROW + at) = l2;
            }
        }
    }
    __syncthreads();

    // k k^T (warps 0-3) and q k^T (warps 4-7), 16 rows per warp, up to the diagonal
    const int wm = warp & 3, which = warp >> 2, g = lane >> 2, t4 = lane & 3;
    float acc[8][4];
#pragma unroll
    for (int n = 0; n < 8; n++) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
    for (int ks = 0; ks < DK / 16; ks++) {
        uint32_t ah[4], al[4];
        const int arow = (wm * 16 + (lane & 15)) * ROW + ks * 16 + (lane >> 4) * 8;
        ldsm4(ah, &sm.op[2 * which][arow]);
        ldsm4(al, &sm.op[2 * which + 1][arow]);
#pragma unroll
        for (int n = 0; n < 8; n += 2) {
            if (n > 2 * wm + 1) break;
            // k as the second operand: its rows are the columns of the product; two tiles of eight
            uint32_t bh[4], bl[4];
            const int brow = (n * 8 + (lane & 7) + (lane >> 4) * 8) * ROW + ks * 16 + ((lane >> 3) & 1) * 8;
            ldsm4(bh, &sm.op[0][brow]);
            ldsm4(bl, &sm.op[1][brow]);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                mma16(acc[n + h], ah, bh[2 * h], bh[2 * h + 1]);
                mma16(acc[n + h], ah, bl[2 * h], bl[2 * h + 1]);
                mma16(acc[n + h], al, bh[2 * h], bh[2 * h + 1]);
            }
        }
    }
    __syncthreads();  // the operands are done with: the tables take their place
    {
        float(*to)[TROW] = which ? sm.t.qk : sm.t.kk;
        const float f0 = sm.down[which][wm * 16 + g], f1 = sm.down[which][wm * 16 + g + 8];
#pragma unroll
        for (int n = 0; n < 8; n++) {
            const int col = n * 8 + 2 * t4;
            const float c0 = sm.down[0][col], c1 = sm.down[0][col + 1];
            to[wm * 16 + g][col] = acc[n][0] * f0 * c0;
            to[wm * 16 + g][col + 1] = acc[n][1] * f0 * c1;
            to[wm * 16 + g + 8][col] = acc[n][2] * f1 * c0;
            to[wm * 16 + g + 8][col + 1] = acc[n][3] * f1 * c1;
        }
    }

    const int ratio = d.n_v / d.n_k;
    for (int hv = hk * ratio; hv < (hk + 1) * ratio; hv++) {
        if (tid == 0) sm.odd = 0;
        __syncthreads();
        if (tid < CH) {
            const int64_t at = (first + tid) * d.n_v + hv;
            const float a = tid < rows ? expf(d.g[at]) : 1.0f, be = tid < rows ? d.beta[at] : 0.0f;
            sm.a[tid] = a;
            sm.beta[tid] = be;
            if (!(a <= 1.0f) || !(be >= 0.0f && be <= 2.0f)) sm.odd = 1;
        }
        __syncthreads();
        const int seg = tid >> 5, col = 2 * (tid & 31), own = col >> 3;  // eight rows and two columns per thread
        if (tid < CH) {
            float r = 1.0f;
            for (int i = tid + 1; i < (tid | 7) + 1; i++) r *= sm.a[i];
            sm.tail[tid] = r;
            if ((tid & 7) == 0) sm.whole[tid >> 3] = r * sm.a[tid];
        }
        __syncthreads();
        __half *np = x.np + (slot * d.n_v + hv) * 4 * CH * NP_ROW;
        float *factors = x.factors + (slot * d.n_v + hv) * ROW_FACTORS;
        {
            // r_ij down the eight rows, beginning with the product up to the row above them
            float r[2] = {1.0f, 1.0f}, between = 1.0f, c = 1.0f;
            for (int k = own + 1; k < seg; k++) between *= sm.whole[k];
            if (seg > own) {
                r[0] = sm.tail[col] * between;
                r[1] = sm.tail[col + 1] * between;
            }
            for (int k = 0; k < seg; k++) c *= sm.whole[k];  // c_i, by the first columns' threads
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int i = 8 * seg + k;
                const float ai = sm.a[i], be = sm.beta[i];
                const float2 kk = *reinterpret_cast<const float2 *>(&sm.t.kk[i][col]), qk = *reinterpret_cast<const float2 *>(&sm.t.qk[i][col]);
                if (i > col) r[0] *= ai;
                if (i > col + 1) r[1] *= ai;
                *reinterpret_cast<float2 *>(&sm.t.A[i][col]) = make_float2(i > col ? be * r[0] * kk.x : 0.0f, i > col + 1 ? be * r[1] * kk.y : 0.0f);
                *reinterpret_cast<float2 *>(&sm.t.N[i][col]) = make_float2(0.0f, 0.0f);
                const float p0 = i >= col ? r[0] * qk.x : 0.0f, p1 = i >= col + 1 ? r[1] * qk.y : 0.0f;
                float up, down;
                row_scale(agn_warp_max(fmaxf(fabsf(p0), fabsf(p1))), up, down);  // a warp has whole rows
                uint32_t h2, l2;
                split2(p0 * up, p1 * up, h2, l2);
                *reinterpret_cast<uint32_t *>(np + (2 * CH + i) * NP_ROW + col) = h2;
                *reinterpret_cast<uint32_t *>(np + (3 * CH + i) * NP_ROW + col) = l2;
                c *= ai;
                if (col == 0) {
                    factors[RF_X + i] = c * sm.down[0][i] * UP;
                    factors[RF_QS + i] = c * sm.down[1][i] * UP;
                    factors[RF_PD + i] = down * UP;
                    if (i == CH - 1) factors[RF_C] = c;
                }
                if (i == CH - 1) *reinterpret_cast<float2 *>(factors + RF_R + col) = make_float2(r[0] * sm.down[0][col], r[1] * sm.down[0][col + 1]);
            }
        }
        __syncthreads();
        // (I + A)^-1: the eight 8 x 8 blocks of the diagonal by substitution, a column per thread
        if (tid < CH) {
            const int o = tid & ~7, cc = tid & 7;
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float sum = i == cc ? 1.0f : 0.0f;
#pragma unroll
                for (int l = 0; l < i; l++) sum = __fmaf_rn(-sm.t.A[o + i][o + l], y[l], sum);
                y[i] = sum;
                sm.t.N[o + i][o + cc] = sum;
            }
        }
        __syncthreads();
        // then the blocks below it, twice the size each time
        lower_block<8>(sm.t.A, sm.t.N, tid);
        lower_block<16>(sm.t.A, sm.t.N, tid);
        lower_block<32>(sm.t.A, sm.t.N, tid);
        for (int i = tid; i < CH * CH / 2; i += CHUNK_THREADS) {
            const int row = i >> 5, col = 2 * (i & 31);
            uint32_t h2, l2;
            const float n0 = sm.t.N[row][col] * sm.beta[col], n1 = sm.t.N[row][col + 1] * sm.beta[col + 1];
            float up, down;
            row_scale(agn_warp_max(fmaxf(fabsf(n0), fabsf(n1))), up, down);  // a row per warp
            split2(n0 * up, n1 * up, h2, l2);
            *reinterpret_cast<uint32_t *>(np + row * NP_ROW + col) = h2;
            *reinterpret_cast<uint32_t *>(np + (CH + row) * NP_ROW + col) = l2;
            if (col == 0) factors[RF_D + row] = down * UP;
        }
        if (tid == 0) x.odd[slot * d.n_v + hv] = sm.odd | sm.odd_kq;
        __syncthreads();
    }
}

template <int DK> struct ChunkSmem {
    static constexpr int KROW = kq_row(DK), NROW = NP_ROW, BROW = 36, VROW = 40;  // elements; rows whose fragments do not collide
    __half k[2][2][CH * KROW], q[2][CH * KROW], n[2][CH * NROW], p[2][CH * NROW];
    float s[DK * BROW], xx[CH * BROW], dd[CH * BROW], dr[CH * BROW];  // S and V - c K S and D, times DOWN; r D times K's factors
    float v[2][CH * VROW], factors[2][ROW_FACTORS];
    uint32_t most[9];  // the largest magnitude in the state's columns of each worker, in the chunk's values
    uint64_t kq_full, v_full, n_full, p_full, kq_free, n_free, p_free;
    int gave_up;
};

// Warps 0-7 work, warps 8-11 fetch values, K and Q, N, P (a bulk copy takes its thread about 300 ns to start, whatever its size, so that one thread for all of
// them would be behind).  The workers' own barrier (1) never waits for the fetching warps; the two sides tell each other through mbarriers: *_full, the data
// of a chunk is there; *_free, its place may be filled again.
__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool workers_sync_or(bool x) {
    uint32_t r;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.or.pred q, 1, 256, p;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(r) : "r"((uint32_t)x) : "memory");
    return r != 0;
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(agn_smem_u32(bar)) : "memory"); }

// Rows of an odd chunk one by one in f32: the 32 columns of the state are in shared memory as [DK][33] floats.
template <int DK> __device__ __noinline__ void delta_rows_by_one(const DeltaArgs &d, float *S, float *tmp, int64_t first, int rows, int hk, int hv, int c0) {
    const int tid = threadIdx.x, col = tid & 31, part = tid >> 5;
    constexpr int PER = DK / 8;
    for (int i = 0; i < rows; i++) {
        const int64_t t = first + i;
        const float *kr = d.k + t * d.k_stride + hk * DK, *qr = d.q + t * d.q_stride + hk * DK;
        float qq = 0.0f, kk = 0.0f, qk = 0.0f;
        for (int j = col; j < DK; j += 32) {
            qq = __fmaf_rn(qr[j], qr[j], qq);
            kk = __fmaf_rn(kr[j], kr[j], kk);
            qk = __fmaf_rn(qr[j], kr[j], qk);
        }
        const float fq = d.scale * (d.eps >= 0.0f ? rsqrtf(agn_warp_sum(qq) + d.eps) : 1.0f), fk = d.eps >= 0.0f ? rsqrtf(agn_warp_sum(kk) + d.eps) : 1.0f;
        qk = agn_warp_sum(qk) * fq * fk;
        float dk = 0.0f, dq = 0.0f;
        for (int j = part * PER; j < (part + 1) * PER; j++) {
            dk = __fmaf_rn(kr[j] * fk, S[j * 33 + col], dk);
            dq = __fmaf_rn(qr[j] * fq, S[j * 33 + col], dq);
        }
        tmp[part * 64 + col] = dk;
        tmp[part * 64 + 32 + col] = dq;
        workers_sync();
        dk = dq = 0.0f;
        for (int w = 0; w < 8; w++) {
            dk += tmp[w * 64 + col];
            dq += tmp[w * 64 + 32 + col];
        }
        const float al = expf(d.g[t * d.n_v + hv]), be = d.beta[t * d.n_v + hv];
        const float dl = be * __fmaf_rn(-al, dk, d.v[t * d.v_stride + hv * d.dv + c0 + col]);
        if (part == 0) d.out[(t * d.n_v + hv) * d.dv + c0 + col] = __fmaf_rn(qk, dl, al * dq);
        for (int j = part * PER; j < (part + 1) * PER; j++) S[j * 33 + col] = __fmaf_rn(kr[j] * fk, dl, al * S[j * 33 + col]);
        workers_sync();
    }
}

template <int DK> __global__ void __launch_bounds__(CARRY_THREADS) delta_chunk_kernel(const __grid_constant__ ChunkArgs x) {
    agn_pdl_prologue();
    extern __shared__ __align__(128) unsigned char raw[];
    using SM = ChunkSmem<DK>;
    SM &sm = *reinterpret_cast<SM *>(raw);
    constexpr int KROW = SM::KROW, NROW = SM::NROW, BROW = SM::BROW, VROW = SM::VROW;
    constexpr int MT = DK / 16, NU = MT / 2;  // the state's 16 x 8 tiles: MT x 4, NU to a warp
    const DeltaArgs &d = x.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int c0 = blockIdx.x * 32, hv = blockIdx.y, hk = hv / (d.n_v / d.n_k);
    const int64_t s = blockIdx.z;
    int64_t b, e;
    delta_rows(d, s, &b, &e);
    const int64_t slot0 = delta_slot(b, s), chunks = (e - b + CH - 1) / CH;
    const bool fetches = warp >= 8;
    const int mt = warp % MT, n0 = (warp & 7) / MT * NU;  // this warp's tiles of the state: rows 16 mt .., columns 8 (n0 + n) ..

    float S[NU][4];
    const int64_t soff = ((s * d.n_v + hv) * DK + 16 * mt + g) * d.dv + c0 + 2 * t4;
#pragma unroll
    for (int n = 0; n < NU; n++) {
        float2 u = make_float2(0.0f, 0.0f), w = u;
        if (d.state_in && !fetches) {
            u = *reinterpret_cast<const float2 *>(d.state_in + soff + 8 * (n0 + n));
            w = *reinterpret_cast<const float2 *>(d.state_in + soff + 8 * (n0 + n) + (int64_t)8 * d.dv);
        }
        S[n][0] = u.x; S[n][1] = u.y; S[n][2] = w.x; S[n][3] = w.y;
    }

    // One thread's bulk copies: K and Q of a chunk, N, P.
    constexpr uint32_t KQ_BYTES = 2 * CH * KROW * 2, NP_BYTES = 2 * CH * NROW * 2;
    auto load_kq = [&](int64_t c) {
        const __half *src = x.kq + ((slot0 + c) * d.n_k + hk) * 4 * CH * KROW;
        agn_mbar_expect_tx(&sm.kq_full, 2 * KQ_BYTES);
        agn_bulk_g2s(sm.k[c & 1], src, KQ_BYTES, &sm.kq_full);
        agn_bulk_g2s(sm.q, src + 2 * CH * KROW, KQ_BYTES, &sm.kq_full);
    };
    auto load_np = [&](int64_t c, int w, void *dst, uint64_t *bar) {
        agn_mbar_expect_tx(bar, NP_BYTES);
        agn_bulk_g2s(dst, x.np + (((slot0 + c) * d.n_v + hv) * 4 + w) * CH * NROW, NP_BYTES, bar);
    };
    auto load_v = [&](int64_t c) {
        const int64_t first = b + c * CH;
        float *dst = sm.v[c & 1];
        const float *src = d.v + first * d.v_stride + (int64_t)hv * d.dv + c0;
#pragma unroll
        for (int i = 0; i < CH * 8 / 32; i++) {
            const int row = (lane >> 3) + 4 * i, at = (lane & 7) * 4;
            if (first + row < e) cp16(dst + row * VROW + at, src + row * d.v_stride + at);
            else *reinterpret_cast<float4 *>(dst + row * VROW + at) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        const float *f = x.factors + ((slot0 + c) * d.n_v + hv) * ROW_FACTORS;
        for (int i = 4 * lane; i < ROW_FACTORS; i += 128) cp16(sm.factors[c & 1] + i, f + i);
    };
    auto tell_largest = [&](uint32_t most) {  // magnitudes as bits: NaN above infinity above the numbers
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) sm.most[warp] = most;
    };
    auto bits = [](float x) { return __float_as_uint(x) & 0x7fffffffu; };
    // a bounded wait; once one has run out the CTA's other waits give up after their next poll
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        for (int left = x.spin; left > 0; left -= 1024) {
            if (agn_mbar_wait(bar, parity, left < 1024 ? left : 1024)) return true;
            if (*(volatile int *)&sm.gave_up) return false;
        }
        *(volatile int *)&sm.gave_up = 1;
        return false;
    };
    if (tid == 0) {
        agn_mbar_init(&sm.kq_full, 1);
        agn_mbar_init(&sm.v_full, 1);
        agn_mbar_init(&sm.n_full, 1);
        agn_mbar_init(&sm.p_full, 1);
        agn_mbar_init(&sm.kq_free, 8);
        agn_mbar_init(&sm.n_free, 8);
        agn_mbar_init(&sm.p_free, 8);
        agn_mbar_init_fence();
        sm.gave_up = 0;
    }
    __syncthreads();

    if (fetches) {
        uint64_t *const full[4] = {&sm.v_full, &sm.kq_full, &sm.n_full, &sm.p_full}, *const free[4] = {&sm.kq_free, &sm.kq_free, &sm.n_free, &sm.p_free};
        const int what = warp - 8;
        int64_t c = 0;
        for (; c < chunks; c++) {
            if (c > 0 && !__all_sync(0xffffffffu, wait(free[what], (c - 1) & 1))) break;  // the turn in which the place was last used
            if (what == 0) {
                load_v(c);
                asm volatile("cp.async.wait_all;" ::: "memory");
                const float *v = sm.v[c & 1];
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < CH * 8 / 32; i++) {
                    const float4 y = *reinterpret_cast<const float4 *>(v + ((lane >> 3) + 4 * i) * VROW + (lane & 7) * 4);
                    most = max(most, max(max(bits(y.x), bits(y.y)), max(bits(y.z), bits(y.w))));
                }
                tell_largest(most);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.v_full);
            } else if (lane == 0) {
                if (what == 1) load_kq(c);
                else if (what == 2) load_np(c, 0, sm.n, &sm.n_full);
                else load_np(c, 2, sm.p, &sm.p_full);
            }
            __syncwarp();
        }
        // no copy may be in flight when the CTA ends
        if (lane == 0 && what > 0 && c > 0) (void)agn_mbar_wait(full[what], (c - 1) & 1, AGN_MBAR_SPIN_LIMIT_DEFAULT);  // not cut short by the option
        if (lane == 0 && sm.gave_up) atomicOr(d.flags, AGN_FLAG_TIMEOUT);
        return;
    }

    int odd = chunks > 0 ? x.odd[slot0 * d.n_v + hv] : 0;
    bool gave_up = false;  // a wait ran out, for all workers alike
    auto freed = [&](uint64_t *bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    auto tell_state = [&] {
        uint32_t most = 0;
#pragma unroll
        for (int n = 0; n < NU; n++) most = max(most, max(max(bits(S[n][0]), bits(S[n][1])), max(bits(S[n][2]), bits(S[n][3]))));
        tell_largest(most);
    };
    tell_state();
    for (int64_t c = 0; c < chunks; c++) {
        const int64_t first = b + c * CH;
        const int rows = (int)(e - first < CH ? e - first : CH);
        const uint32_t turn = c & 1;
        if ((gave_up = workers_sync_or(!(wait(&sm.kq_full, turn) && wait(&sm.v_full, turn))))) break;
        uint32_t most = 0;
#pragma unroll
        for (int w = 0; w < 9; w++) most = max(most, sm.most[w]);
        const bool bad = most >= 0x77800000u || (most > 0 && most < 0x12800000u);  // 2^112 and more, not finite; all below 2^-90
        const int odd_next = c + 1 < chunks ? x.odd[(slot0 + c + 1) * d.n_v + hv] : 0;
        const float *v = sm.v[c & 1];
        if (odd || bad) {
            // nobody's copies into these buffers may be on their way any more
            if ((gave_up = workers_sync_or(!(wait(&sm.n_full, turn) && wait(&sm.p_full, turn))))) break;
            float *Sf = reinterpret_cast<float *>(sm.q), *tmp = reinterpret_cast<float *>(sm.n);  // q, N are not needed
#pragma unroll
            for (int n = 0; n < NU; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) Sf[(16 * mt + g + (i >> 1) * 8) * 33 + 8 * (n0 + n) + 2 * t4 + (i & 1)] = S[n][i];
            workers_sync();
            delta_rows_by_one<DK>(d, Sf, tmp, first, rows, hk, hv, c0);
#pragma unroll
            for (int n = 0; n < NU; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) S[n][i] = Sf[(16 * mt + g + (i >> 1) * 8) * 33 + 8 * (n0 + n) + 2 * t4 + (i & 1)];
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // these writes come before the next copies' ones
            freed(&sm.kq_free);
            freed(&sm.n_free);
            freed(&sm.p_free);
            workers_sync();  // sm.most has been read
            tell_state();
            odd = odd_next;
            continue;
        }
        odd = odd_next;
#pragma unroll
        for (int n = 0; n < NU; n++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                *reinterpret_cast<float2 *>(&sm.s[(16 * mt + g + 8 * i) * BROW + 8 * (n0 + n) + 2 * t4]) = make_float2(S[n][2 * i] * DOWN, S[n][2 * i + 1] * DOWN);
        workers_sync();

        // ---- K S and Q S: 16 rows and 16 columns per warp
        const int wm = warp & 3, wn = (warp >> 2) * 16, bat = 2 * t4 * BROW + g;  // this lane's first element of a B fragment
        const __half *kh = sm.k[c & 1][0], *kl = sm.k[c & 1][1];
        float ks[2][4] = {}, qs[2][4] = {}, ks_low[2][4] = {}, qs_low[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < DK / 16; kk++) {
            uint32_t r0[4], r1[4];
            float kfh[8], kfl[8], qfh[8], qfl[8];
            const int arow = (wm * 16 + (lane & 15)) * KROW + kk * 16 + (lane >> 4) * 8;
            ldsm4(r0, kh + arow);
            ldsm4(r1, kl + arow);
            half_to_tf32(r0, kfh);
            half_to_tf32(r1, kfl);
            ldsm4(r0, sm.q[0] + arow);
            ldsm4(r1, sm.q[1] + arow);
            half_to_tf32(r0, qfh);
            half_to_tf32(r1, qfl);
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const Split16 f(sm.s + kk * 16 * BROW + wn + 8 * n + bat, BROW);
                mma_split(ks[n], ks_low[n], kfh, kfl, f);
                mma_split(qs[n], qs_low[n], qfh, qfl, f);
            }
        }
        const int r0 = wm * 16 + g;
        const float *rf = sm.factors[c & 1] + r0;
        const float of_x[2] = {rf[RF_X], rf[RF_X + 8]}, of_qs[2] = {rf[RF_QS], rf[RF_QS + 8]};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int col = wn + 8 * n + 2 * t4;
                const float2 vv = *reinterpret_cast<const float2 *>(v + (r0 + 8 * i) * VROW + col);
                const float x0 = __fmaf_rn(-of_x[i], ks[n][2 * i] + ks_low[n][2 * i], vv.x), x1 = __fmaf_rn(-of_x[i], ks[n][2 * i + 1] + ks_low[n][2 * i + 1], vv.y);
                *reinterpret_cast<float2 *>(&sm.xx[(r0 + 8 * i) * BROW + col]) = make_float2(x0 * DOWN, x1 * DOWN);
                qs[n][2 * i] = of_qs[i] * (qs[n][2 * i] + qs_low[n][2 * i]);
                qs[n][2 * i + 1] = of_qs[i] * (qs[n][2 * i + 1] + qs_low[n][2 * i + 1]);
            }
        freed(&sm.kq_free);  // q has been read; the other buffers of k and v were last chunk's
        if ((gave_up = workers_sync_or(!wait(&sm.n_full, turn)))) break;

        // ---- D = N X.  (N is a lower triangle, but leaving its empty blocks out would only make the warps uneven: the slowest one does them all.)
        float dd[2][4] = {}, po[2][4] = {};
        {
            float low[2][4] = {};
#pragma unroll
            for (int kk = 0; kk < CH / 16; kk++) {
                if (kk > wm) break;
                uint32_t r0[4], r1[4];
                float fh[8], fl[8];
                const int arow = (wm * 16 + (lane & 15)) * NROW + kk * 16 + (lane >> 4) * 8;
                ldsm4(r0, sm.n[0] + arow);
                ldsm4(r1, sm.n[1] + arow);
                half_to_tf32(r0, fh);
                half_to_tf32(r1, fl);
#pragma unroll
                for (int n = 0; n < 2; n++) mma_split(dd[n], low[n], fh, fl, Split16(sm.xx + kk * 16 * BROW + wn + 8 * n + bat, BROW));
            }
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) dd[n][i] += low[n][i];
        }
        const float of_d[2] = {rf[RF_D], rf[RF_D + 8]}, of_r[2] = {rf[RF_R], rf[RF_R + 8]};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int at = (r0 + 8 * i) * BROW + wn + 8 * n + 2 * t4;
                const float d0 = dd[n][2 * i] * of_d[i], d1 = dd[n][2 * i + 1] * of_d[i];
                *reinterpret_cast<float2 *>(&sm.dd[at]) = make_float2(d0 * DOWN, d1 * DOWN);
                *reinterpret_cast<float2 *>(&sm.dr[at]) = make_float2(d0 * of_r[i], d1 * of_r[i]);
            }
        freed(&sm.n_free);
        if ((gave_up = workers_sync_or(!wait(&sm.p_full, turn)))) break;

        // ---- S' = c_C S + K^T (r D)
        {
            float sum[NU][4] = {}, low[NU][4] = {};
#pragma unroll
            for (int kk = 0; kk < CH / 16; kk++) {
                uint32_t r0[4], r1[4];
                float fh[8], fl[8];
                const int arow = (kk * 16 + (lane & 7) + (lane >> 4) * 8) * KROW + mt * 16 + ((lane >> 3) & 1) * 8;
                ldsm4t(r0, kh + arow);
                ldsm4t(r1, kl + arow);
                half_to_tf32(r0, fh);
                half_to_tf32(r1, fl);
#pragma unroll
                for (int n = 0; n < NU; n++) mma_split(sum[n], low[n], fh, fl, Split16(sm.dr + kk * 16 * BROW + 8 * (n0 + n) + bat, BROW));
            }
            const float cc = sm.factors[c & 1][RF_C];
#pragma unroll
            for (int n = 0; n < NU; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) S[n][i] = __fmaf_rn(cc, S[n][i], sum[n][i] + low[n][i]);
        }

        // ---- O = c Q S + P D
        {
            float low[2][4] = {};
#pragma unroll
            for (int kk = 0; kk < CH / 16; kk++) {
                if (kk > wm) break;
                uint32_t r0[4], r1[4];
                float fh[8], fl[8];
                const int arow = (wm * 16 + (lane & 15)) * NROW + kk * 16 + (lane >> 4) * 8;
                ldsm4(r0, sm.p[0] + arow);
                ldsm4(r1, sm.p[1] + arow);
                half_to_tf32(r0, fh);
                half_to_tf32(r1, fl);
#pragma unroll
                for (int n = 0; n < 2; n++) mma_split(po[n], low[n], fh, fl, Split16(sm.dd + kk * 16 * BROW + wn + 8 * n + bat, BROW));
            }
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) po[n][i] += low[n][i];
        }
        const float of_pd[2] = {rf[RF_PD], rf[RF_PD + 8]};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (r0 + 8 * i < rows)
                    *reinterpret_cast<float2 *>(d.out + ((first + r0 + 8 * i) * d.n_v + hv) * d.dv + c0 + wn + 8 * n + 2 * t4) =
                        make_float2(__fmaf_rn(po[n][2 * i], of_pd[i], qs[n][2 * i]) * d.scale, __fmaf_rn(po[n][2 * i + 1], of_pd[i], qs[n][2 * i + 1]) * d.scale);
        freed(&sm.p_free);
        tell_state();
    }
    if (gave_up) {  // by the workers themselves: the fetching warps may have looked at sm.gave_up before one of these waits ran out
        if (tid == 0) atomicOr(d.flags, AGN_FLAG_TIMEOUT);
        return;
    }
#pragma unroll
    for (int n = 0; n < NU; n++) {
        *reinterpret_cast<float2 *>(d.state_out + soff + 8 * (n0 + n)) = make_float2(S[n][0], S[n][1]);
        *reinterpret_cast<float2 *>(d.state_out + soff + 8 * (n0 + n) + (int64_t)8 * d.dv) = make_float2(S[n][2], S[n][3]);
    }
}

// The chunked form pays from about this many rows a sequence on, on average.  16/32 heads of 128, recurrent / chunked, us: one sequence of 32 rows 27 / 28, of 40
// 34 / 28, of 128 102 / 46; 32 sequences of 32 rows 227 / 298, of 40 280 / 299, of 48 335 / 304, of 128 870 / 519.
constexpr int CHUNK_MIN_ROWS = 40;
bool delta_chunked(int64_t T, int64_t n_seqs) { return T >= CHUNK_MIN_ROWS * n_seqs; }

struct ChunkLayout {
    int64_t slots, kq, np, factors, odd, bytes;  // byte offsets
};
ChunkLayout chunk_layout(int64_t T, int64_t n_seqs, int n_k, int n_v, int dk) {
    ChunkLayout l;
    l.slots = T / CH + n_seqs;
    l.kq = 0;
    l.np = l.kq + l.slots * n_k * 4 * CH * kq_row(dk) * 2;
    l.factors = l.np + l.slots * n_v * 4 * CH * NP_ROW * 2;
    l.odd = l.factors + l.slots * n_v * ROW_FACTORS * 4;
    l.bytes = (l.odd + l.slots * n_v * 4 + 15) / 16 * 16;
    return l;
}

template <int DK> int32_t launch_chunked(agn_ctx *ctx, const DeltaArgs &d, void *workspace, int n_seqs) {
    const ChunkLayout l = chunk_layout(d.T, d.n_seqs, d.n_k, d.n_v, DK);
    ChunkArgs x;
    unsigned char *w = static_cast<unsigned char *>(workspace);
    x.d = d;
    x.kq = reinterpret_cast<__half *>(w + l.kq);
    x.np = reinterpret_cast<__half *>(w + l.np);
    x.factors = reinterpret_cast<float *>(w + l.factors);
    x.odd = reinterpret_cast<int *>(w + l.odd);
    x.spin = ctx->mbar_spin_limit;
    if (agn_ring_ctas_per_sm(ctx, delta_prepare_kernel<DK>, CHUNK_THREADS, sizeof(PrepSmem<DK>)) < 1 ||
        agn_ring_ctas_per_sm(ctx, delta_chunk_kernel<DK>, CARRY_THREADS, sizeof(ChunkSmem<DK>)) < 1)
        return agn_fail(ctx, AGN_ECUDA, "gated_delta_rule: the chunk kernels do not fit the device's shared memory");
    ctx->flags_dirty = true;
    agn_launch(ctx, delta_prepare_kernel<DK>, dim3((unsigned)l.slots, (unsigned)d.n_k), dim3(CHUNK_THREADS), sizeof(PrepSmem<DK>), x);
    AGN_LAUNCHED(ctx, "gated_delta_chunk");
    agn_launch(ctx, delta_chunk_kernel<DK>, dim3((unsigned)(d.dv / 32), (unsigned)d.n_v, (unsigned)n_seqs), dim3(CARRY_THREADS), sizeof(ChunkSmem<DK>), x);
    AGN_LAUNCHED(ctx, "gated_delta_chunk");
    return AGN_OK;
}

bool delta_shape_ok(int64_t T, int64_t n_seqs, int n_k, int n_v, int dk, int dv) {
    return T >= 0 && T <= 0x7fffffffLL && n_seqs > 0 && n_seqs <= 65535 && n_k > 0 && n_v > 0 && n_v % n_k == 0 && n_v <= 65535 && (dk == 64 || dk == 128) &&
           dv > 0 && dv % 32 == 0 && dv <= 256;
}

}  // namespace

extern "C" int64_t agn_gated_delta_rule_workspace_bytes(int64_t T, int64_t n_seqs, int32_t n_k_heads, int32_t n_v_heads, int32_t head_k,
                                                        int32_t head_v) {
    if (!delta_shape_ok(T, n_seqs, n_k_heads, n_v_heads, head_k, head_v) || !delta_chunked(T, n_seqs)) return 0;
    return chunk_layout(T, n_seqs, n_k_heads, n_v_heads, head_k).bytes;
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
    if (!agn_aligned(g, 4) || !agn_aligned(beta, 4) || !agn_aligned(cu_seqlens, 4))
        return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: g, beta and cu_seqlens must be aligned to their element type");
    if (out && (out == q || out == k || out == v)) return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: out must not alias q, k or v");
    AGN_CUDA(ctx, cudaSetDevice(ctx->device));
    DeltaArgs a;
    a.q = q; a.k = k; a.v = v; a.g = g; a.beta = beta; a.state_in = state_in; a.state_out = state_out; a.out = out; a.cu = cu_seqlens;
    a.T = T; a.n_seqs = n_seqs; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.n_k = n_k_heads; a.n_v = n_v_heads; a.dv = head_v; a.scale = scale; a.eps = l2norm_eps; a.flags = ctx->d_flags;
    if (cu_seqlens) ctx->flags_dirty = true;
    if (delta_chunked(T, n_seqs)) {
        const int64_t need = chunk_layout(T, n_seqs, n_k_heads, n_v_heads, head_k).bytes;
        if (!workspace || (int64_t)workspace_bytes < need || !agn_aligned16(workspace))
            return agn_fail(ctx, AGN_EINVAL, "gated_delta_rule: needs %lld bytes of 16-byte aligned workspace", (long long)need);
        return head_k == 64 ? launch_chunked<64>(ctx, a, workspace, (int)n_seqs) : launch_chunked<128>(ctx, a, workspace, (int)n_seqs);
    }
    const dim3 grid((unsigned)(head_v / 32), (unsigned)n_v_heads, (unsigned)n_seqs);
    if (head_k == 64) agn_launch(ctx, delta_recurrent_kernel<64>, grid, dim3(128), 0, a);
    else agn_launch(ctx, delta_recurrent_kernel<128>, grid, dim3(128), 0, a);
    AGN_LAUNCHED(ctx, "gated_delta_recurrent");
    return AGN_OK;
}
