// Attention of a prompt's rows (consecutive positions of one sequence) over the KV cache, to f32's precision: f32 rows, and f16 rows of head sizes
// that the tensor-memory form (agn_attention_prompt.cu) does not cover.
//
// Bound by the matrix units: per 16 rows, 16 slots and 32 dims 8 products m16n8k16 (f16) for the scores and 12 (bf16) for the output, which caps the kernel near 220
// TFLOP/s; what holds it is shared memory, where each warp's 16 rows read every tile again, and the splitting of the weights.  Precision comes from operands in parts:
// queries as hi + lo f16 against the cached bytes (exact in f16), weights times the block scale as three bf16 parts against the cached bytes (exact in bf16), and against an
// f16 cache as two tf32 parts.  A CTA takes 16 rows per warp of one KV head - row r is (token r / G, head r % G) - and 64 slots at a time, which it brings from the
// cache's blocks to 16-bit rows in shared memory once for all warps, the next 64 while these are worked on.  512 tokens of 32/8 heads of 64, q8_0: 34 us (128 CTAs, eight
// tiles one after the other); 2048 tokens of 28/4 heads of 128: 351 us, 86 TFLOP/s (f16 cache 324 us).  Blocks of four warps, two to an SM, convert every tile twice as
// often: 256 rows behind 8000 slots 440 -> 847 us (with the weights as two tf32 parts throughout).
#include <math.h>

#include "agn_attention_decode.cuh"

namespace {

constexpr int SL = 64;  // slots of a tile

template <int NB> struct ChunkShape {
    static constexpr int HD = NB * 32, WARPS = NB <= 4 ? 8 : 4, THREADS = 32 * WARPS, ROWS = 16 * WARPS, ROW = HD + 8;  // f16 elements of a row in shared memory
    static constexpr int BLOCKS = (2 * SL * NB + THREADS - 1) / THREADS;  // cache blocks that a thread converts per tile
};

template <int NB> struct ChunkTiles {
    using C = ChunkShape<NB>;
    __half q[2][C::ROWS * C::ROW];  // hi, lo
    __half k[2][SL * C::ROW], v[2][SL * C::ROW];
    __align__(16) float ks[2][NB][SL + 8], vs[2][NB][SL + 8], coef[C::ROWS];  // scales of neighbouring slots side by side
    int odd;
};

// One block of 32 values on its way from the cache: 16 words of f16, or 8 words of bytes and a scale.  q8_0 as the words lie in memory: a block that begins at a
// multiple of 4 is 8 words (scale and bytes) and the last two bytes, one that does not is the scale and 8 words.  Taking them apart is left to place_block, since a
// use of a loaded word here would wait for it (2048 rows of 28/4 heads of 128, with the weights as tf32 parts: 397 us, so 374).
template <int KV> struct Block {
    uint32_t w[KV == KV_F16 ? 16 : 8];
    uint32_t more;  // q8_0: the two bytes outside the words; words: the scale
};

template <int KV> __device__ __forceinline__ void fetch_block(Block<KV> &x, const unsigned char *p, bool there) {
#pragma unroll
    for (int i = 0; i < (KV == KV_F16 ? 16 : 8); i++) x.w[i] = KV == KV_WORDS ? 0x80808080u : 0u;
    x.more = 0;
    if (!there) return;
    const uint32_t *w = reinterpret_cast<const uint32_t *>(p);
    if (KV == KV_WORDS) {
        x.more = w[0];
#pragma unroll
        for (int i = 0; i < 8; i++) x.w[i] = w[i + 1];
    } else if (KV == KV_Q8) {
        const int off = (int)(reinterpret_cast<uintptr_t>(p) & 2);
        const uint32_t *d = reinterpret_cast<const uint32_t *>(p + off);
#pragma unroll
        for (int i = 0; i < 8; i++) x.w[i] = d[i];
        x.more = *reinterpret_cast<const uint16_t *>(p + (off ? 0 : 32));
    } else if (!(reinterpret_cast<uintptr_t>(p) & 15)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 y = reinterpret_cast<const uint4 *>(p)[i];
            x.w[4 * i] = y.x; x.w[4 * i + 1] = y.y; x.w[4 * i + 2] = y.z; x.w[4 * i + 3] = y.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) x.w[i] = reinterpret_cast<const uint16_t *>(p)[2 * i] | (uint32_t)reinterpret_cast<const uint16_t *>(p)[2 * i + 1] << 16;
    }
}

// Two of four bytes (as byte + 128) as exact bf16: 128 + the lower seven bits, less 128 or 256 by the upper one (0x4380 is 256, 0x4300 128).
__device__ __forceinline__ uint32_t bytes_to_bf162(uint32_t u, uint32_t sel) {
    const uint32_t a = __byte_perm(u & 0x7f7f7f7fu, 0x43434343u, sel), b = __byte_perm(~u & 0x80808080u, 0x43434343u, sel);
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// To 32 values of 16 bits and the block's scale: f16, but bf16 for the bytes of V (is_v), whose weights are bf16 parts.  from: what was fetched (its address, of a q8_0
// block).  Returns whether one of V's f16 values is not finite (it becomes 0).
template <int KV> __device__ __forceinline__ bool place_block(const Block<KV> &x, const unsigned char *from, __half *to, float *scale, bool is_v) {
    bool odd = false;
    uint32_t bytes[8];
    if (KV == KV_WORDS) {
        *scale = __uint_as_float(x.more);
#pragma unroll
        for (int i = 0; i < 8; i++) bytes[i] = x.w[i];
    } else if (KV == KV_Q8) {
        const bool apart = reinterpret_cast<uintptr_t>(from) & 2;  // the scale lies before the words, not in the first one
        *scale = __half2float(__ushort_as_half((unsigned short)(apart ? x.more : x.w[0])));
#pragma unroll
        for (int i = 0; i < 8; i++) bytes[i] = apart ? x.w[i] : __funnelshift_r(x.w[i], i < 7 ? x.w[i < 7 ? i + 1 : 7] : x.more, 16);
    }
    uint4 *dst = reinterpret_cast<uint4 *>(to);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t h[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (KV == KV_F16) {
                h[c] = x.w[4 * i + c];
                if (is_v) {
                    const bool o0 = (h[c] & 0x7c00u) == 0x7c00u, o1 = (h[c] & 0x7c000000u) == 0x7c000000u;
                    odd |= o0 || o1;
                    if (o0) h[c] &= 0xffff0000u;
                    if (o1) h[c] &= 0x0000ffffu;
                }
            } else {
                const uint32_t u = offset_bytes<KV>(bytes[2 * i + (c >> 1)]);
                h[c] = is_v ? bytes_to_bf162(u, c & 1 ? 0x4342 : 0x4140) : bytes_to_half2(u, c & 1 ? 0x4342 : 0x4140);
            }
        }
        dst[i] = make_uint4(h[0], h[1], h[2], h[3]);
    }
    return odd;
}

// Weights have f32's range: a weight however small may meet a value that outweighs it.  Times the scale of a block of bytes they are three bf16 parts (8 bits each; the
// bytes are exact in bf16), against an f16 cache two tf32 parts (11 bits each; f16 is exact in tf32).  (Two f16 parts under the tile's largest scale, 287 us for 2048 rows
// of 28/4 heads of 128, lost weights under 2^-25 to 2^-31 of the row's largest.)
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
    const auto pair = [](float a, float b) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&r);
    };
    hi = pair(x, y);
    x = fminf(x - __uint_as_float(hi << 16), 1e35f);  // with an infinite scale not inf - inf
    y = fminf(y - __uint_as_float(hi & 0xffff0000u), 1e35f);
    mid = pair(x, y);
    lo = pair(x - __uint_as_float(mid << 16), y - __uint_as_float(mid & 0xffff0000u));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(agn_smem_u32(p)) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(agn_smem_u32(p)) : "memory");
}

template <int KV, int NB> __global__ void __launch_bounds__(ChunkShape<NB>::THREADS, 1) attn_chunk_kernel(const __grid_constant__ DecodeArgs d, AttnSplit split, int row_tiles, int *odd_flags) {
    agn_pdl_prologue();
    using C = ChunkShape<NB>;
    using F = KvFormat<KV>;
    extern __shared__ __align__(128) unsigned char raw[];
    ChunkTiles<NB> &sm = *reinterpret_cast<ChunkTiles<NB> *>(raw);
    const AttnArgs &a = d.a;
    constexpr int HD = C::HD, ROW = C::ROW;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3, G = a.n_q / a.n_kv, kvh = blockIdx.x % a.n_kv;
    const int share = blockIdx.x / a.n_kv % split.splits;
    const int rows = (int)a.T * G, r0 = (row_tiles - 1 - (int)(blockIdx.x / a.n_kv / split.splits)) * C::ROWS;  // the rows that see most first
    const int last_row = min(r0 + C::ROWS, rows) - 1, end = a.pos_start + last_row / G + 1, seen_tiles = (end + SL - 1) / SL;
    const int per_share = (seen_tiles + split.splits - 1) / split.splits, tile0 = min(share * per_share, seen_tiles), tiles = min(seen_tiles, tile0 + per_share);  // tile0 .. tiles - 1
    if (tid == 0) sm.odd = 0;

    auto block_at = [&](int n, int tile) {
        return (n < SL * NB ? a.k_cache : a.v_cache) + (int64_t)(tile * SL + n / NB % SL) * a.bytes_per_token + (kvh * NB + n % NB) * F::BYTES;
    };
    auto fetch = [&](Block<KV> &x, int i, int tile) {
        const int n = tid + i * C::THREADS;
        fetch_block<KV>(x, block_at(n, tile), n < 2 * SL * NB && tile * SL + n / NB % SL < end);
    };
    auto place = [&](const Block<KV> &x, int i, int tile) {
        const int n = tid + i * C::THREADS, b = n % NB, slot = n / NB % SL;
        const bool is_k = n < SL * NB;
        if (n >= 2 * SL * NB) return;
        const bool odd = place_block<KV>(x, block_at(n, tile), (is_k ? sm.k : sm.v)[tile & 1] + slot * ROW + b * 32, &(is_k ? sm.ks : sm.vs)[tile & 1][b][slot], !is_k);
        if (KV == KV_F16 && odd) sm.odd = 1;
    };
    constexpr int HELD = NB <= 4 ? C::BLOCKS : 1;  // blocks that wait in registers while a tile is worked on; larger heads have none left for them
    Block<KV> next[HELD];
    auto fetch_tile = [&](int tile) {
#pragma unroll
        for (int i = 0; i < C::BLOCKS; i++) {
            fetch(next[i % HELD], i, tile);
            if (NB > 4) place(next[0], i, tile);
        }
    };
    auto place_tile = [&](int tile) {
        if (NB <= 4) {
#pragma unroll
            for (int i = 0; i < C::BLOCKS; i++) place(next[i % HELD], i, tile);
        }
    };
    __syncthreads();
    if (tile0 < tiles) fetch_tile(tile0);

    // ---- Q, a warp's 16 rows: largest value to [2^14, 2^15), two f16 parts
    constexpr int QB = NB <= 4 ? 8 : 4;  // rows whose loads are on their way together (one after the other: 24 us more for 2048 rows of 28/4 heads of 128)
    for (int i0 = 0; i0 < 16; i0 += QB) {
        float x[QB][NB];
#pragma unroll
        for (int i = 0; i < QB; i++) {
            const int r = r0 + warp * 16 + i0 + i;
            const int64_t at = ((int64_t)(r / G) * a.n_q + kvh * G + r % G) * HD + lane;
#pragma unroll
            for (int c = 0; c < NB; c++)
                x[i][c] = r >= rows ? 0.0f : d.act16 ? __half2float(static_cast<const __half *>(a.q)[at + c * 32]) : static_cast<const float *>(a.q)[at + c * 32];
        }
#pragma unroll
        for (int i = 0; i < QB; i++) {
            const int row = warp * 16 + i0 + i;
            float amax = 0.0f;
#pragma unroll
            for (int c = 0; c < NB; c++) amax = fmaxf(amax, fabsf(x[i][c]));
            amax = agn_warp_max(amax);
            float up;
            const float coef = query_scale(amax, a.scale, up);
            if (lane == 0) sm.coef[row] = coef;
#pragma unroll
            for (int c = 0; c < NB; c++) {
                const float v = x[i][c] * up;
                const __half h = __float2half_rn(v);
                sm.q[0][row * ROW + c * 32 + lane] = h;
                sm.q[1][row * ROW + c * 32 + lane] = __float2half_rn(v - __half2float(h));
            }
        }
    }
    if (tile0 < tiles) place_tile(tile0);
    __syncthreads();

    const int ra = r0 + warp * 16 + g;  // this lane's rows: ra and ra + 8
    const float coef[2] = {sm.coef[warp * 16 + g], sm.coef[warp * 16 + g + 8]};
    const int lim[2] = {a.pos_start + min(ra, rows - 1) / G, a.pos_start + min(ra + 8, rows - 1) / G}, warp_first = a.pos_start + min(r0 + warp * 16, rows - 1) / G;
    const int warp_last = a.pos_start + min(r0 + warp * 16 + 15, rows - 1) / G;
    float o[4 * NB][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4 * NB; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

    for (int tile = tile0; tile < tiles; tile++) {
        if (tile + 1 < tiles) fetch_tile(tile + 1);
        const bool sees = tile * SL <= warp_last;  // a warp whose rows see none of it waits for the others
        const int buf = tile & 1;
        const bool edge = tile * SL + SL - 1 > warp_first;
        float s[SL / 8][4];
        if (sees) {
#pragma unroll
            for (int n = 0; n < SL / 8; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float blk[SL / 8][4];
#pragma unroll
                for (int n = 0; n < SL / 8; n++) blk[n][0] = blk[n][1] = blk[n][2] = blk[n][3] = 0.0f;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    uint32_t hi[4], lo[4];
                    const int qa = (warp * 16 + (lane & 15)) * ROW + b * 32 + k * 16 + (lane >> 4) * 8;
                    ldsm4(hi, sm.q[0] + qa);
                    ldsm4(lo, sm.q[1] + qa);
#pragma unroll
                    for (int n = 0; n < SL / 8; n += 2) {
                        uint32_t kf[4];  // two groups of eight slots
                        ldsm4(kf, sm.k[buf] + (n * 8 + (lane & 7) + (lane >> 4) * 8) * ROW + b * 32 + k * 16 + ((lane >> 3) & 1) * 8);
                        mma_f16(blk[n], hi, kf[0], kf[1]);
                        mma_f16(blk[n + 1], hi, kf[2], kf[3]);
                        mma_f16(blk[n], lo, kf[0], kf[1]);
                        mma_f16(blk[n + 1], lo, kf[2], kf[3]);
                    }
                }
                if (KV == KV_F16) {  // blocks of dims are added up by rounded additions, too: over all dims the matrix unit's cuts would add up to 6e-6 of a result
#pragma unroll
                    for (int n = 0; n < SL / 8; n++) add4(s[n], blk[n]);
                } else {
#pragma unroll
                    for (int n = 0; n < SL / 8; n++) {
                        const float2 f = *reinterpret_cast<const float2 *>(&sm.ks[buf][b][8 * n + 2 * t4]);
                        s[n][0] = __fmaf_rn(blk[n][0], f.x, s[n][0]);
                        s[n][1] = __fmaf_rn(blk[n][1], f.y, s[n][1]);
                        s[n][2] = __fmaf_rn(blk[n][2], f.x, s[n][2]);
                        s[n][3] = __fmaf_rn(blk[n][3], f.y, s[n][3]);
                    }
                }
            }
            float mt[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < SL / 8; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (edge && tile * SL + 8 * n + 2 * t4 + (i & 1) > lim[i >> 1]) s[n][i] = -INFINITY;
                    mt[i >> 1] = fmaxf(mt[i >> 1], s[n][i]);
                }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                mt[i] = fmaxf(mt[i], __shfl_xor_sync(0xffffffffu, mt[i], 1));
                mt[i] = fmaxf(mt[i], __shfl_xor_sync(0xffffffffu, mt[i], 2)) * coef[i];
            }
            if (__any_sync(0xffffffffu, mt[0] > m[0] + 8.0f || mt[1] > m[1] + 8.0f)) {  // true at the first tile
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    mt[i] = fmaxf(mt[i], m[i]);
                    const float c = ex2(m[i] - (mt[i] == -INFINITY ? 0.0f : mt[i]));
                    l[i] *= c;
                    m[i] = mt[i];
#pragma unroll
                    for (int n = 0; n < 4 * NB; n++) { o[n][2 * i] *= c; o[n][2 * i + 1] *= c; }
                }
            }
            const float mu[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
            for (int n = 0; n < SL / 8; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[n][i] = ex2(__fmaf_rn(s[n][i], coef[i >> 1], -mu[i >> 1]));
                    l[i >> 1] += s[n][i];
                }
        }
        if (tile + 1 < tiles) place_tile(tile + 1);
        if (sees) {
            // ---- O += P V; the sums of a tile in the matrix unit (whose adder cuts), the running ones by rounded additions.  Dims 8 c + 2 t4 (+ 1) of the block in o[4 b + c].
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float acc[4][4];
#pragma unroll
                for (int c = 0; c < 4; c++) acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.0f;
#pragma unroll
                for (int n = 0; n < SL / 8; n += 2) {
                    if (KV == KV_F16) {
                        float hi[2][4], lo[2][4];
#pragma unroll
                        for (int u = 0; u < 2; u++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                hi[u][i] = __uint_as_float((__float_as_uint(s[n + u][i]) + 0x1000u) & 0xffffe000u);
                                lo[u][i] = s[n + u][i] - hi[u][i];
                            }
#pragma unroll
                        for (int c = 0; c < 4; c += 2) {
                            uint32_t v[4];  // two groups of eight dims, of eight slots each
                            ldsm4t(v, sm.v[buf] + (8 * n + (lane & 15)) * ROW + b * 32 + c * 8 + (lane >> 4) * 8);
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&v[k]));
                                const int u = k & 1, to = c + (k >> 1);
                                mma_tf32(acc[to], hi[u][0], hi[u][2], hi[u][1], hi[u][3], f.x, f.y);
                                mma_tf32(acc[to], lo[u][0], lo[u][2], lo[u][1], lo[u][3], f.x, f.y);
                            }
                        }
                    } else {
                        uint32_t hi[4], mid[4], lo[4];
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const float2 f = *reinterpret_cast<const float2 *>(&sm.vs[buf][b][8 * (n + u) + 2 * t4]);
                            float w[4] = {s[n + u][0] * f.x, s[n + u][1] * f.y, s[n + u][2] * f.x, s[n + u][3] * f.y};
                            if (edge) {  // a scale that is not finite, in a slot that the row does not see
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    if (tile * SL + 8 * (n + u) + 2 * t4 + (i & 1) > lim[i >> 1]) w[i] = 0.0f;
                            }
                            split_bf16(w[0], w[1], hi[2 * u], mid[2 * u], lo[2 * u]);
                            split_bf16(w[2], w[3], hi[2 * u + 1], mid[2 * u + 1], lo[2 * u + 1]);
                        }
#pragma unroll
                        for (int c = 0; c < 4; c += 2) {
                            uint32_t v[4];
                            ldsm4t(v, sm.v[buf] + (8 * n + (lane & 15)) * ROW + b * 32 + c * 8 + (lane >> 4) * 8);
                            mma_bf16(acc[c], hi, v[0], v[1]);
                            mma_bf16(acc[c + 1], hi, v[2], v[3]);
                            mma_bf16(acc[c], mid, v[0], v[1]);
                            mma_bf16(acc[c + 1], mid, v[2], v[3]);
                            mma_bf16(acc[c], lo, v[0], v[1]);
                            mma_bf16(acc[c + 1], lo, v[2], v[3]);
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; c++) add4(o[4 * b + c], acc[c]);
            }
        }
        __syncthreads();
    }

#pragma unroll
    for (int i = 0; i < 2; i++) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const int r = ra + 8 * i;
        if (r >= rows) continue;
        const int64_t at = ((int64_t)(r / G) * a.n_q + kvh * G + r % G) * HD;
        if (split.splits > 1) {  // a share: what agn_attention_join needs
            float *to = split.part + ((int64_t)share * a.T * a.n_q + at / HD) * (HD + 4);
            if (t4 == 0) *reinterpret_cast<float2 *>(to + HD) = make_float2(m[i], l[i]);
#pragma unroll
            for (int b = 0; b < NB; b++) {
#pragma unroll
                for (int c = 0; c < 4; c++) *reinterpret_cast<float2 *>(to + b * 32 + 8 * c + 2 * t4) = make_float2(o[4 * b + c][2 * i], o[4 * b + c][2 * i + 1]);
            }
            continue;
        }
        const float inv = m[i] == -INFINITY ? NAN : 1.0f / l[i];  // all scores -inf: 0 / 0
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float2 y = make_float2(o[4 * b + c][2 * i] * inv, o[4 * b + c][2 * i + 1] * inv);
                const int64_t x = at + b * 32 + 8 * c + 2 * t4;
                if (d.act16) *reinterpret_cast<__half2 *>(static_cast<__half *>(a.out) + x) = __floats2half2_rn(y.x, y.y);
                else *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + x) = y;
            }
    }
    if (KV == KV_F16) {  // rare: V held values that are not finite
        __syncthreads();
        if (!sm.odd) return;
        if (split.splits > 1) {
            if (tid == 0) odd_flags[kvh] = 1;  // by agn_attention_join
            return;
        }
        for (int x = tid; x < C::ROWS * HD; x += C::THREADS) {
            const int r = r0 + x / HD, dim = x % HD;
            if (r >= rows) break;
            const float bad = odd_value(a, AGN_F16, kvh * HD + dim, a.pos_start + r / G, [](int) { return true; }, 1);
            if (bad == 0.0f) continue;
            const int64_t at = ((int64_t)(r / G) * a.n_q + kvh * G + r % G) * HD + dim;
            store_act(d, at, bad + (d.act16 ? __half2float(static_cast<const __half *>(a.out)[at]) : static_cast<const float *>(a.out)[at]));
        }
    }
}

__global__ void attn_clear_kernel(int *p, int n) {
    agn_pdl_prologue();
    for (int i = threadIdx.x; i < n; i += blockDim.x) p[i] = 0;
}

int chunk_rows(int hd) { return hd <= 128 ? 128 : 64; }
struct ChunkLayout {
    int row_tiles, splits;
    int64_t odd, bytes;
};
ChunkLayout chunk_layout(int64_t slots, int64_t T, int n_q, int n_kv, int hd, int sms, bool anywhere = false) {
    ChunkLayout l;
    l.row_tiles = (int)((T * (n_q / n_kv) + chunk_rows(hd) - 1) / chunk_rows(hd));
    l.splits = (anywhere ? attn_splits_most : attn_splits)((int64_t)l.row_tiles * n_kv, (slots + SL - 1) / SL, 1.0 + 0.041 * hd, T * n_q, hd, sms);
    l.odd = attn_part_bytes(l.splits, T, n_q, hd);
    l.bytes = l.splits > 1 ? l.odd + (n_kv * 4 + 15) / 16 * 16 : 0;
    return l;
}

template <int KV, int NB> int32_t launch_chunk(agn_ctx *ctx, const DecodeArgs &d, const ChunkLayout &l, void *workspace) {
    static_assert(ChunkShape<NB>::ROWS == (NB <= 4 ? 128 : 64), "chunk_rows");
    using C = ChunkShape<NB>;
    if (agn_ring_ctas_per_sm(ctx, attn_chunk_kernel<KV, NB>, C::THREADS, sizeof(ChunkTiles<NB>)) < 1)
        return agn_fail(ctx, AGN_ECUDA, "attention_kv: the chunk kernel does not fit the device's shared memory");
    AttnSplit split = {static_cast<float *>(workspace), l.splits};
    int *odd = l.splits > 1 && KV == KV_F16 ? reinterpret_cast<int *>(static_cast<unsigned char *>(workspace) + l.odd) : nullptr;
    if (odd) {
        agn_launch(ctx, attn_clear_kernel, dim3(1), dim3(256), 0, odd, d.a.n_kv);
        AGN_LAUNCHED(ctx, "attention_kv_chunk");
    }
    agn_launch(ctx, attn_chunk_kernel<KV, NB>, dim3((unsigned)((int64_t)l.row_tiles * d.a.n_kv * l.splits)), dim3(C::THREADS), sizeof(ChunkTiles<NB>), d, split, l.row_tiles, odd);
    AGN_LAUNCHED(ctx, "attention_kv_chunk");
    // one flag per KV head: a group of all slots
    return l.splits > 1 ? agn_attention_join(ctx, d.a, AGN_F16, d.act16, split, odd, 1, 0x7fffffff) : AGN_OK;
}

template <int KV> int32_t launch_chunk_kv(agn_ctx *ctx, const DecodeArgs &d, const ChunkLayout &l, void *workspace) {
    switch (d.a.hd / 32) {
    case 1: return launch_chunk<KV, 1>(ctx, d, l, workspace);
    case 2: return launch_chunk<KV, 2>(ctx, d, l, workspace);
    case 3: return launch_chunk<KV, 3>(ctx, d, l, workspace);
    case 4: return launch_chunk<KV, 4>(ctx, d, l, workspace);
    case 5: return launch_chunk<KV, 5>(ctx, d, l, workspace);
    case 6: return launch_chunk<KV, 6>(ctx, d, l, workspace);
    case 7: return launch_chunk<KV, 7>(ctx, d, l, workspace);
    default: return launch_chunk<KV, 8>(ctx, d, l, workspace);
    }
}

}  // namespace

int64_t agn_attention_chunk_workspace(int64_t slots, int64_t T, int n_q, int n_kv, int hd, int sms, bool anywhere) {
    return chunk_layout(slots, T, n_q, n_kv, hd, sms, anywhere).bytes;
}

int32_t agn_attention_chunk(agn_ctx *ctx, const AttnArgs &a, int kv_dtype, int act16, void *workspace) {
    const ChunkLayout l = chunk_layout((int64_t)a.pos_start + a.T, a.T, a.n_q, a.n_kv, a.hd, ctx->sm_count < ATTN_MAX_SMS ? ctx->sm_count : ATTN_MAX_SMS);
    DecodeArgs d = {};
    d.a = a;
    d.act16 = act16;
    if (kv_dtype == AGN_F16) return launch_chunk_kv<KV_F16>(ctx, d, l, workspace);
    if (kv_dtype == AGN_Q8_0) return launch_chunk_kv<KV_Q8>(ctx, d, l, workspace);
    return launch_chunk_kv<KV_WORDS>(ctx, d, l, workspace);
}
