// Attention of a prompt's rows (consecutive positions of one sequence, f16) over the KV cache, on the 5th-generation tensor cores.
//
// Bound by the tensor cores (4 * head_dim flop per row, head and slot) and, equally, by the exponentials (16 a clock and SM
// against 128 x 128 products of 128 in 1024 clocks); what holds it is the way from scores to weights to the next scores.  4096 tokens of 28/4 heads of 128, q8_0:
// 154-159 us with the unpacking (8), 760-780 TFLOP/s; 1001 tokens behind 7001 slots, 32/8 heads of 128: 172 us.  Keys, values and weights are rounded to f16, for
// one product each instead of two and three: rows are off by 4.7e-4 to 5.4e-4 of their norm, where rounding the result alone costs 2.1e-4.  Two kernels:
//
//   attn_unpack_kernel writes the sequence's K and V as f16 tiles of 128 slots of one head, each the very bytes that the matrix
//   instruction wants in shared memory (rows of 128 bytes, 16-byte pieces exchanged by row: the 128-byte swizzle), so that a tile is
//   one bulk copy and no CTA dequantises what another one needs too (every tile is read by T * G / 256 CTAs).
//
//   attn_prompt_kernel: a CTA takes 256 query rows of one KV head - row r is (token r / G, head r % G of the group), so a tile
//   serves the whole group - as two tiles of 128, so that the tensor cores work on one tile while the softmax of the other
//   runs.  Warps 0-3 and 4-7: softmax of the two tiles, a row per thread; warp 8 fetches tiles; warp 9 issues the products.
//   TMEM: S0, S1, O0, O1 (128 columns each); the weights overwrite their scores as f16 and are the A operand of the second
//   product from there.  The output is rescaled only when a row's maximum has grown by more than 2^8 (weights stay in f16's
//   range; sums and accumulators are f32).
#include <math.h>

#include "agn_attention.cuh"

namespace {

// The reference is W_UP powers of two below a row's maximum, so that weights reach 2^W_UP and, with the 2^8 that a row may outgrow it by, stay below 2^15: f16 then keeps
// its 11 bits down to 2^-21 of a row's largest weight (light slots may have the larger values) and something down to 2^-32.
constexpr float W_UP = 7.0f;
constexpr int TILE = 128, PROMPT_THREADS = 320, SLOTS = 5, DRAIN_POLLS = AGN_MBAR_SPIN_LIMIT_DEFAULT;  // the last waits are not cut short by the option

struct PromptArgs {
    AttnArgs a;
    __half *k, *v;   // [n_kv][tiles] images of TILE x hd
    int *odd;        // [n_kv][tiles]: the V tile has a value that is not finite
    int *range;      // [K, V][n_kv][tiles]: RANGE_* of what the tile holds
    int kv_dtype;
    int64_t tiles, rows;  // tiles of the sequence; rows T * G of a KV head
    int spin, row_tiles;
    AttnSplit split;
};

// Whether f16 holds a tile: something of 65520 or more, which f16 turns into infinity; keys from f16's smallest normal number on; keys other than 0.  Keys that all
// lie below it would lose their bits (a large `scale` may still make scores of them); small values are as exact as the f16 result.
constexpr int RANGE_OVER = 1, RANGE_NORMAL = 2, RANGE_SOME = 4;

// One CTA per (tile, KV head, K or V).  Values that are not finite are 0 in V's image and noted: a weight of 0 for a slot that a
// row does not see must not meet them in the product.
template <int KV> __global__ void __launch_bounds__(1024) attn_unpack_kernel(const __grid_constant__ PromptArgs p) {
    agn_pdl_prologue();
    const AttnArgs &a = p.a;
    const int64_t tile = blockIdx.x;
    const int head = blockIdx.y, hd = a.hd, chunks = hd / 8;
    bool odd = false;
    float most = 0.0f;
    const bool is_v = blockIdx.z;
    const int end = a.pos_start + (int)a.T;
    const unsigned char *src = is_v ? a.v_cache : a.k_cache;
    unsigned char *dst = reinterpret_cast<unsigned char *>(is_v ? p.v : p.k) + (head * p.tiles + tile) * TILE * hd * 2;
    for (int i = threadIdx.x; i < TILE * chunks; i += blockDim.x) {
        const int r = i / chunks, c = i % chunks;
        const int64_t slot = tile * TILE + r;
        float v[8];
        if (slot < end) {
            const unsigned char *row = src + slot * a.bytes_per_token;
            const int d = head * hd + c * 8;
            if (KV == KV_F16) {
                const uint16_t *w = reinterpret_cast<const uint16_t *>(row) + d;
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = __half2float(__ushort_as_half(w[k]));
            } else {
                const unsigned char *blk = row + (d >> 5) * KvFormat<KV>::BYTES;
                const float s = block_scale<KV>(blk);
                const uint16_t *w = reinterpret_cast<const uint16_t *>(blk + KvFormat<KV>::DATA + (d & 31));
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t u = KV == KV_Q8 ? w[k] ^ 0x8080u : w[k];
                    v[2 * k] = (float)((int)(u & 0xff) - 128) * s;
                    v[2 * k + 1] = (float)((int)(u >> 8) - 128) * s;
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = 0.0f;
        }
        if (KV != KV_F16) {
#pragma unroll
            for (int k = 0; k < 8; k++) most = fmaxf(most, fabsf(v[k]));  // NaN is ignored
        }
        if (is_v) {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (!half_finite(v[k])) {
                    odd |= !(fabsf(v[k]) < INFINITY);
                    v[k] = 0.0f;
                }
        }
        __half2 h[4];
#pragma unroll
        for (int k = 0; k < 4; k++) h[k] = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
        *reinterpret_cast<uint4 *>(dst + (c >> 3) * TILE * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = *reinterpret_cast<const uint4 *>(h);
    }
    odd = __syncthreads_or(odd);
    if (is_v && threadIdx.x == 0) p.odd[head * p.tiles + tile] = odd;
    if (KV != KV_F16) {  // f16 tiles are what the cache holds
        __shared__ float warp_most[32];
        most = agn_warp_max(most);
        if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = most;
        __syncthreads();
        if (threadIdx.x < 32) {
            most = agn_warp_max(warp_most[threadIdx.x]);
            int bits = most >= 65520.0f ? RANGE_OVER : 0;
            if (!is_v) bits |= (most >= 6.103515625e-5f ? RANGE_NORMAL : 0) | (most > 0.0f ? RANGE_SOME : 0);
            if (threadIdx.x == 0) p.range[((is_v ? a.n_kv : 0) + head) * p.tiles + tile] = bits;
        }
    }
}

// Rows whose tiles f16 does not hold, straight from the cache in f32: the CTA's rows r0 .. r0 + 2 TILE - 1 over its share's tiles, written as the kernel below writes
// them (values that are not finite as 0).  A warp per row, four slots at a time; rare, and slow (2048 rows of 28/4 heads of 128 over 2048 slots: 23 ms, where the tensor
// cores take 55 us).
template <int HD, int KV> __device__ __noinline__ void prompt_rows_f32(const PromptArgs &p, int head, int share, int64_t r0, int tile0, int tiles) {
    const AttnArgs &a = p.a;
    const int lane = threadIdx.x & 31, G = a.n_q / a.n_kv;
    constexpr int V = HD / 32;
    const float coef = a.scale * 1.4426950408889634f;
    for (int i = threadIdx.x >> 5; i < 2 * TILE && r0 + i < p.rows; i += PROMPT_THREADS / 32) {
        const int64_t r = r0 + i, row = r / G * a.n_q + head * G + r % G;
        const int end = min(a.pos_start + (int)(r / G) + 1, (tile0 + tiles) * TILE);
        float q[V], o[V], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int c = 0; c < V; c++) {
            q[c] = __half2float(static_cast<const __half *>(a.q)[row * HD + lane + 32 * c]);
            o[c] = 0.0f;
        }
        for (int j = tile0 * TILE; j < end; j += 4) {
            float s[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const unsigned char *key = a.k_cache + (int64_t)min(j + k, end - 1) * a.bytes_per_token;
                float x = 0.0f;
#pragma unroll
                for (int c = 0; c < V; c++) x = __fmaf_rn(q[c], cache_value<KV>(key, head * HD + lane + 32 * c), x);
                s[k] = agn_warp_sum(x) * coef;
                if (j + k >= end) s[k] = -INFINITY;
            }
            const float mt = fmaxf(fmaxf(m, fmaxf(s[0], s[1])), fmaxf(s[2], s[3])), mu = mt == -INFINITY ? 0.0f : mt, down = ex2(m - mu);
            m = mt;
            l *= down;
#pragma unroll
            for (int c = 0; c < V; c++) o[c] *= down;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (j + k >= end) break;
                const unsigned char *value = a.v_cache + (int64_t)(j + k) * a.bytes_per_token;
                const float w = ex2(s[k] - mu);
                l += w;
#pragma unroll
                for (int c = 0; c < V; c++) {
                    const float v = cache_value<KV>(value, head * HD + lane + 32 * c);
                    o[c] = __fmaf_rn(w, fabsf(v) < INFINITY ? v : 0.0f, o[c]);
                }
            }
        }
        if (p.split.splits > 1) {
            float *to = p.split.part + ((int64_t)share * a.T * a.n_q + row) * (HD + 4);
#pragma unroll
            for (int c = 0; c < V; c++) to[lane + 32 * c] = o[c];
            if (lane == 0) {
                to[HD] = m;
                to[HD + 1] = l;
            }
        } else {
            const float inv = m == -INFINITY ? NAN : 1.0f / l;
#pragma unroll
            for (int c = 0; c < V; c++) static_cast<__half *>(a.out)[row * HD + lane + 32 * c] = __float2half_rn(o[c] * inv);
        }
    }
}

// ---- tensor-core instructions
// Operand in shared memory: rows of 128 bytes, swizzled in groups of eight rows (1024 bytes).  lead: bytes to the next 64 elements of the
// row dimension where that is the contiguous one.
__device__ __forceinline__ uint64_t smem_operand(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// f16 x f16 -> f32, M = 128; b_rows_contiguous: the second operand's N is its contiguous dimension
__device__ __forceinline__ constexpr uint32_t mma_shape(int n, bool b_rows_contiguous) {
    return 1u << 4 | (b_rows_contiguous ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b),
                 "r"(shape), "r"((int)add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b),
                 "r"(shape), "r"((int)add)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(agn_smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(agn_smem_u32(bar)) : "memory");
}
#define TMEM_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define TMEM_W4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
                 "%28,%29,%30,%31}, [%32];"
                 : TMEM_R4(r, 0), TMEM_R4(r, 4), TMEM_R4(r, 8), TMEM_R4(r, 12), TMEM_R4(r, 16), TMEM_R4(r, 20), TMEM_R4(r, 24), TMEM_R4(r, 28)
                 : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
                 "%28,%29,%30,%31};" ::TMEM_W4(r, 0), TMEM_W4(r, 4), TMEM_W4(r, 8), TMEM_W4(r, 12), TMEM_W4(r, 16), TMEM_W4(r, 20), TMEM_W4(r, 24), TMEM_W4(r, 28),
                 "r"(at)
                 : "memory");
}
// The registers go through the wait, so that nothing that uses them is scheduled in front of it.
#define TMEM_RW4(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3])
__device__ __forceinline__ void tmem_loaded(uint32_t *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : TMEM_RW4(r, 0), TMEM_RW4(r, 4), TMEM_RW4(r, 8), TMEM_RW4(r, 12), TMEM_RW4(r, 16), TMEM_RW4(r, 20), TMEM_RW4(r, 24), TMEM_RW4(r, 28)::"memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : TMEM_R4(r, 0), TMEM_R4(r, 4), TMEM_R4(r, 8), TMEM_R4(r, 12)
                 : "r"(at));
}
__device__ __forceinline__ void tmem_loaded16(uint32_t *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : TMEM_RW4(r, 0), TMEM_RW4(r, 4), TMEM_RW4(r, 8), TMEM_RW4(r, 12)::"memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::TMEM_W4(r, 0), TMEM_W4(r, 4), TMEM_W4(r, 8),
                 TMEM_W4(r, 12), "r"(at)
                 : "memory");
}

template <int HD> struct PromptSmem {
    unsigned char q[2][TILE * HD * 2], kv[SLOTS][TILE * HD * 2];  // tiles in the order K0 V0 K1 V1 ..
    uint64_t q_full, full[SLOTS], free[SLOTS], s_full[2], p_full[2], o_full[2], drained;
    uint32_t tmem;
    int gave_up, range, odd;
};

template <int HD> __global__ void __launch_bounds__(PROMPT_THREADS, 1) attn_prompt_kernel(const __grid_constant__ PromptArgs p) {
    agn_pdl_prologue();
    extern __shared__ unsigned char raw[];
    PromptSmem<HD> &sm = *reinterpret_cast<PromptSmem<HD> *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const AttnArgs &a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.n_q / a.n_kv, head = blockIdx.x % a.n_kv, share = blockIdx.x / a.n_kv % p.split.splits;
    const int64_t r0 = (int64_t)(p.row_tiles - 1 - (int)(blockIdx.x / a.n_kv / p.split.splits)) * 2 * TILE;  // the rows that see most first, so that the last CTAs are short
    const int64_t last_row = r0 + 2 * TILE - 1 < p.rows ? r0 + 2 * TILE - 1 : p.rows - 1;
    const int seen_tiles = (int)((a.pos_start + last_row / G) / TILE) + 1;  // by the CTA's last row
    const int per_share = (seen_tiles + p.split.splits - 1) / p.split.splits, tile0 = min(share * per_share, seen_tiles);
    const int tiles = min(seen_tiles - tile0, per_share);  // of this CTA's share, from tile0 on
    constexpr uint32_t IMAGE = TILE * HD * 2;

    // ---- warps 0-7: the query row of this thread, and Q on its way (a warp's 32 rows, whole rows side by side)
    const int i = warp >> 2;
    const int64_t r = r0 + i * TILE + (tid & 127);
    const bool there = r < p.rows;
    const uint32_t tok = (uint32_t)(there ? r : p.rows - 1) / (uint32_t)G;
    const int last = a.pos_start + (int)tok;  // the last slot it sees
    const int64_t own = there ? ((int64_t)tok * a.n_q + head * G + (uint32_t)r % (uint32_t)G) * HD : -1;  // its first value in q and out
    constexpr int CPR = HD / 8, RPI = 32 / CPR;  // 16-byte pieces of a row, rows per instruction
    const int piece = lane % CPR;
    if (warp < 8) {
        const uint32_t qs = agn_smem_u32(sm.q[i]) + (piece >> 3) * TILE * 128 + (warp & 3) * 32 * 128;
#pragma unroll
        for (int k = 0; k < 32; k += RPI) {
            const int wr = k + lane / CPR;
            const int64_t at = __shfl_sync(0xffffffffu, own, wr);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(qs + wr * 128 + (((piece & 7) ^ (wr & 7)) << 4)),
                         "l"(static_cast<const __half *>(a.q) + (at >= 0 ? at + piece * 8 : 0)), "r"(at >= 0 ? 16 : 0)
                         : "memory");
        }
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(agn_smem_u32(&sm.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        agn_mbar_init(&sm.q_full, 256);
        for (int i = 0; i < SLOTS; i++) {
            agn_mbar_init(&sm.full[i], 1);
            agn_mbar_init(&sm.free[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            agn_mbar_init(&sm.s_full[i], 1); agn_mbar_init(&sm.p_full[i], 128); agn_mbar_init(&sm.o_full[i], 1);
        }
        agn_mbar_init(&sm.drained, 1);
        agn_mbar_init_fence();
        sm.gave_up = sm.range = sm.odd = 0;
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sm.tmem;
    // a bounded wait; once one has run out the CTA's other waits give up after their next poll
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        for (int left = p.spin; left > 0; left -= 1024) {
            if (agn_mbar_wait(bar, parity, left < 1024 ? left : 1024)) return true;
            if (*(volatile int *)&sm.gave_up) return false;
        }
        *(volatile int *)&sm.gave_up = 1;
        return false;
    };

    // the same for a whole warp: its lanes go on together or not at all
    auto wait_warp = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); };

    if (warp == 8) {
        if (lane == 0) {
            const unsigned char *k = reinterpret_cast<const unsigned char *>(p.k) + (head * p.tiles + tile0) * IMAGE;
            const unsigned char *v = reinterpret_cast<const unsigned char *>(p.v) + (head * p.tiles + tile0) * IMAGE;
            int n = 0;
            for (; n < 2 * tiles; n++) {
                const int at = n % SLOTS;
                if (n >= SLOTS && !wait(&sm.free[at], (n / SLOTS - 1) & 1)) break;
                agn_mbar_expect_tx(&sm.full[at], IMAGE);
                agn_bulk_g2s(sm.kv[at], (n & 1 ? v : k) + (int64_t)(n >> 1) * IMAGE, IMAGE, &sm.full[at]);
            }
            // no copy may be in flight when the CTA ends: the last one of every slot (the products have waited for the earlier ones)
            for (int i = n > SLOTS ? n - SLOTS : 0; i < n; i++) (void)agn_mbar_wait(&sm.full[i % SLOTS], (i / SLOTS) & 1, DRAIN_POLLS);
        }
        __syncwarp();
    } else if (warp == 9) {
        if (lane == 0) {
            const uint32_t qa = agn_smem_u32(sm.q[0]), kva = agn_smem_u32(sm.kv[0]);
            auto scores = [&](int i, uint32_t tile) {  // S_i = Q_i K^T with the K tile there
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks++) {
                    const uint32_t at = (ks >> 2) * TILE * 128 + (ks & 3) * 32;
                    mma_ss(tmem + i * 128, smem_operand(qa + i * IMAGE + at, 16), smem_operand(tile + at, 16), mma_shape(TILE, false), ks > 0);
                }
                mma_commit(&sm.s_full[i]);
            };
            bool ok = tiles > 0 && wait(&sm.q_full, 0) && wait(&sm.full[0], 0);
            if (ok) {
                fence_after();
                scores(0, kva);
                scores(1, kva);
                mma_commit(&sm.free[0]);
            }
            int v = 1, k = 2;  // slots of V_j and K_(j+1), and how often they have been filled before
            uint32_t v_turn = 0, k_turn = 0;
            for (int j = 0; ok && j < tiles; j++) {
                const bool more = j + 1 < tiles;
                const uint32_t vt = kva + v * IMAGE, kt = kva + k * IMAGE;
                if (!wait(&sm.full[v], v_turn & 1)) break;
                for (int i = 0; i < 2; i++) {
                    if (!(ok = wait(&sm.p_full[i], j & 1))) break;
                    fence_after();
#pragma unroll
                    for (int ks = 0; ks < TILE / 16; ks++)  // O_i += P_i V_j, 16 slots at a time
                        mma_ts(tmem + 256 + i * 128, tmem + i * 128 + ks * 8, smem_operand(vt + ks * 2048, TILE * 128), mma_shape(HD, true),
                               j > 0 || ks > 0);
                    if (i == 1) mma_commit(&sm.free[v]);
                    if (!more) mma_commit(&sm.o_full[i]);
                    else if (i == 1 || (ok = wait(&sm.full[k], k_turn & 1))) scores(i, kt);  // behind that product, which reads the weights in S_i's place
                    else break;
                }
                if (ok && more) mma_commit(&sm.free[k]);
                if ((v += 2) >= SLOTS) { v -= SLOTS; v_turn++; }
                if ((k += 2) >= SLOTS) { k -= SLOTS; k_turn++; }
            }
            mma_commit(&sm.drained);  // every product is done before the tensor memory goes back
            (void)agn_mbar_wait(&sm.drained, 0, DRAIN_POLLS);
        }
        __syncwarp();
    } else {
        // ---- a query row per thread
        asm volatile("cp.async.wait_all;\nfence.proxy.async.shared::cta;" ::: "memory");  // this thread's share of Q, for the tensor cores
        bar_arrive(&sm.q_full);

        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // 32 lanes of the tensor memory per warp, lane number in the upper half
        const uint32_t s_at = tmem + i * 128 + lanes, o_at = tmem + 256 + i * 128 + lanes;
        const float coef = a.scale * 1.4426950408889634f;
        const int first_last = a.pos_start + (int)((r0 + i * TILE) / G);  // what the tile's first row sees
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < tiles; j++) {
            if (!(ok = wait_warp(&sm.s_full[i], j & 1))) break;
            fence_after();
            // 32 scores at a time: while the weights of one piece are taken, the next one's maximum is found and the one after it is on its way.
            const int seen = last - (tile0 + j) * TILE;  // slots c <= seen of this tile
            const bool edge = (tile0 + j) * TILE + TILE - 1 > first_last;
            uint32_t s[2][32];
            float2 sum = make_float2(0.0f, 0.0f);
            auto piece_max = [&](uint32_t *x, int c) {
                if (edge) {
#pragma unroll
                    for (int k = 0; k < 32; k++)
                        if (32 * c + k > seen) x[k] = 0xff800000u;
                }
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    asm("max.f32 %0, %0, %1, %2;" : "+f"(x0) : "f"(__uint_as_float(x[k])), "f"(__uint_as_float(x[k + 1])));
                    asm("max.f32 %0, %0, %1, %2;" : "+f"(x1) : "f"(__uint_as_float(x[k + 2])), "f"(__uint_as_float(x[k + 3])));
                }
                return fmaxf(x0, x1) * coef;
            };
            // Where a row's maximum has grown by more than 2^8 (its first piece, and rarely after that), everything taken against the old one is scaled: the sums, the
            // output of earlier tiles, the weights of this tile's first `done` pieces.
            auto grown = [&](float mt, int done) {
                const bool grow = mt > m + (8.0f + W_UP);
                if (!__any_sync(0xffffffffu, grow)) return;
                const float f = grow ? ex2(m - (mt - W_UP)) : 1.0f;
                if (grow) m = mt - W_UP;
                l *= f;
                sum.x *= f;
                sum.y *= f;
                if (j > 0) {
#pragma unroll
                    for (int c = 0; c < HD; c += 16) {
                        uint32_t o[16];
                        tmem_load16(o_at + c, o);
                        tmem_loaded16(o);
#pragma unroll
                        for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                        tmem_store16(o_at + c, o);
                    }
                }
                const __half2 f2 = __floats2half2_rn(f, f);
                for (int c = 0; c < done; c++) {
                    uint32_t w[16];
                    tmem_stored();
                    tmem_load16(s_at + 16 * c, w);
                    tmem_loaded16(w);
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&w[k]), f2);
                        w[k] = *reinterpret_cast<const uint32_t *>(&y);
                    }
                    tmem_store16(s_at + 16 * c, w);
                }
            };
            tmem_load32(s_at, s[0]);
            tmem_loaded(s[0]);
            tmem_load32(s_at + 32, s[1]);
            float mt = piece_max(s[0], 0);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                grown(mt, c);
                if (c < 3) {
                    tmem_loaded(s[(c + 1) & 1]);
                    mt = piece_max(s[(c + 1) & 1], c + 1);
                }
                const float mu = m == -INFINITY ? 0.0f : m;
                uint32_t *x = s[c & 1], w[16];
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float2 e = __ffma2_rn(make_float2(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), make_float2(coef, coef), make_float2(-mu, -mu));
                    const float2 y = make_float2(ex2(e.x), ex2(e.y));
                    sum = __fadd2_rn(sum, y);
                    const __half2 h2 = __floats2half2_rn(y.x, y.y);
                    w[k] = *reinterpret_cast<const uint32_t *>(&h2);
                }
                tmem_store16(s_at + 16 * c, w);  // over scores that have been read
                if (c < 2) tmem_load32(s_at + 32 * (c + 2), s[c & 1]);
            }
            l += sum.x + sum.y;
            tmem_stored();
            fence_before();
            bar_arrive(&sm.p_full[i]);
        }
        if (p.split.splits > 1) {
            // a share: what agn_attention_join needs
            float *to = p.split.part + ((int64_t)share * a.T * a.n_q + (there ? own / HD : 0)) * (HD + 4);
            if (there) *reinterpret_cast<float2 *>(to + HD) = make_float2(m, l);
            if (tiles > 0 && ok && (ok = wait_warp(&sm.o_full[i], 0))) {
                fence_after();
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    tmem_load32(o_at + c, o);
                    tmem_loaded(o);
                    if (there) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4) *reinterpret_cast<uint4 *>(to + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                    }
                }
            }
        } else if (ok && (ok = wait_warp(&sm.o_full[i], 0))) {
            fence_after();
            const float inv = m == -INFINITY ? NAN : 1.0f / l;  // all scores -inf: 0 / 0
            // The output goes out through the queries' place in shared memory (the last product that reads them is done), whole rows side by side.
            unsigned char *stage = sm.q[i] + (warp & 3) * 32 * HD * 2;
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                tmem_load32(o_at + c, o);
                tmem_loaded(o);
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    __half2 h2[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) h2[q] = __floats2half2_rn(__uint_as_float(o[k + 2 * q]) * inv, __uint_as_float(o[k + 2 * q + 1]) * inv);
                    const int pc = (c + k) / 8;
                    *reinterpret_cast<uint4 *>(stage + lane * HD * 2 + ((pc ^ (lane & 7)) << 4)) = *reinterpret_cast<const uint4 *>(h2);
                }
            }
            __syncwarp();
#pragma unroll 8
            for (int k = 0; k < 32; k += RPI) {
                const int wr = k + lane / CPR;
                const int64_t at = __shfl_sync(0xffffffffu, own, wr);
                if (at >= 0)
                    *reinterpret_cast<uint4 *>(static_cast<__half *>(a.out) + at + piece * 8) =
                        *reinterpret_cast<const uint4 *>(stage + wr * HD * 2 + ((piece ^ (wr & 7)) << 4));
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 9) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (tid == 0 && sm.gave_up) atomicOr(a.flags, AGN_FLAG_TIMEOUT);

    // Rare: f16 does not hold the keys or values of these tiles, or V holds values that are not finite (they were 0 in the product).
    const bool may_be_out = p.kv_dtype != AGN_F16;
    int range = 0, odd = 0;
    for (int j = tid; j < tiles; j += PROMPT_THREADS) {
        const int64_t at = head * p.tiles + tile0 + j;
        odd |= p.odd[at];
        if (may_be_out) range |= p.range[at] | p.range[a.n_kv * p.tiles + at];
    }
    if (range) atomicOr(&sm.range, range);
    if (odd) sm.odd = 1;
    __syncthreads();
    range = sm.range;
    if ((range & RANGE_OVER) || (range & (RANGE_NORMAL | RANGE_SOME)) == RANGE_SOME) {
        if (p.kv_dtype == AGN_Q8_0) prompt_rows_f32<HD, KV_Q8>(p, head, share, r0, tile0, tiles);
        else prompt_rows_f32<HD, KV_WORDS>(p, head, share, r0, tile0, tiles);
        __syncthreads();
    }
    if (p.split.splits > 1 || !sm.odd) return;  // shares: by agn_attention_join
    for (int64_t x = tid; x < 2 * TILE * HD; x += PROMPT_THREADS) {
        const int64_t r = r0 + x / HD;
        const int d = (int)(x % HD), last = a.pos_start + (int)(r / G);
        if (r >= p.rows) break;
        const float bad = odd_value(a, p.kv_dtype, head * HD + d, last, [&](int slot) { return p.odd[head * p.tiles + slot / TILE] != 0; }, TILE);
        if (bad != 0.0f) {
            __half *o = static_cast<__half *>(a.out) + ((r / G) * a.n_q + head * G + r % G) * HD + d;
            *o = __float2half_rn(__half2float(*o) + bad);
        }
    }
}

int64_t image_bytes(int64_t slots, int n_kv, int hd) { return (slots + TILE - 1) / TILE * TILE * n_kv * hd * 2; }
int64_t odd_ints(int64_t slots, int n_kv) { return (slots + TILE - 1) / TILE * n_kv; }

template <int HD> int32_t launch_prompt(agn_ctx *ctx, const PromptArgs &p, int kv_dtype) {
    const size_t smem = sizeof(PromptSmem<HD>) + 1024;
    if (agn_ring_ctas_per_sm(ctx, attn_prompt_kernel<HD>, PROMPT_THREADS, smem) < 1)
        return agn_fail(ctx, AGN_ECUDA, "attention_kv: the prompt kernel does not fit the device's shared memory");
    const dim3 tiles((unsigned)p.tiles, (unsigned)p.a.n_kv, 2);
    if (kv_dtype == AGN_F16) agn_launch(ctx, attn_unpack_kernel<KV_F16>, tiles, dim3(1024), 0, p);
    else if (kv_dtype == AGN_Q8_0) agn_launch(ctx, attn_unpack_kernel<KV_Q8>, tiles, dim3(1024), 0, p);
    else agn_launch(ctx, attn_unpack_kernel<KV_WORDS>, tiles, dim3(1024), 0, p);
    AGN_LAUNCHED(ctx, "attention_kv_prompt");
    agn_launch(ctx, attn_prompt_kernel<HD>, dim3((unsigned)((int64_t)p.row_tiles * p.a.n_kv * p.split.splits)), dim3(PROMPT_THREADS), smem, p);
    AGN_LAUNCHED(ctx, "attention_kv_prompt");
    return p.split.splits > 1 ? agn_attention_join(ctx, p.a, kv_dtype, 1, p.split, p.odd, p.tiles, TILE) : AGN_OK;
}

}  // namespace

// From so few tokens on the prompt form is the faster one (28/4 heads of 128, single rows /
// prompt form, us: behind 8000 q8_0 slots 4 rows 34 / 34, 8 rows 38 / 34, 16 rows 54 / 36; behind 1000 slots 8 rows 21 / 19).
constexpr int PROMPT_MIN_TOKENS = 8;
bool agn_attention_prompt_fits(int64_t T, int n_q, int n_kv, int hd) { return (hd == 64 || hd == 128) && T >= PROMPT_MIN_TOKENS && T * (n_q / n_kv) < (1LL << 30); }

namespace {
struct PromptLayout {
    int64_t image, odd, part, bytes;  // bytes of an image set; byte offsets
    int row_tiles, splits;
};
PromptLayout prompt_layout(int64_t slots, int64_t T, int n_q, int n_kv, int hd, int sms, bool anywhere = false) {
    PromptLayout l;
    l.image = image_bytes(slots, n_kv, hd);
    l.odd = 2 * l.image;
    l.part = l.odd + (3 * odd_ints(slots, n_kv) * 4 + 15) / 16 * 16;  // odd, range of K, range of V
    l.row_tiles = (int)((T * (n_q / n_kv) + 2 * TILE - 1) / (2 * TILE));
    l.splits = (anywhere ? attn_splits_most : attn_splits)((int64_t)l.row_tiles * n_kv, (slots + TILE - 1) / TILE, 2.4, T * n_q, hd, sms);
    l.bytes = l.part + attn_part_bytes(l.splits, T, n_q, hd);
    return l;
}
}  // namespace

int64_t agn_attention_prompt_workspace(int64_t slots, int64_t T, int n_q, int n_kv, int hd, int sms, bool anywhere) {
    return prompt_layout(slots, T, n_q, n_kv, hd, sms, anywhere).bytes;
}

int32_t agn_attention_prompt_f16(agn_ctx *ctx, const AttnArgs &a, int kv_dtype, void *workspace) {
    PromptArgs p;
    const int64_t slots = (int64_t)a.pos_start + a.T;
    const PromptLayout l = prompt_layout(slots, a.T, a.n_q, a.n_kv, a.hd, ctx->sm_count < ATTN_MAX_SMS ? ctx->sm_count : ATTN_MAX_SMS);
    unsigned char *w = static_cast<unsigned char *>(workspace);
    p.a = a;
    p.k = reinterpret_cast<__half *>(w);
    p.v = reinterpret_cast<__half *>(w + l.image);
    p.odd = reinterpret_cast<int *>(w + l.odd);
    p.range = p.odd + odd_ints(slots, a.n_kv);
    p.split.part = reinterpret_cast<float *>(w + l.part);
    p.split.splits = l.splits;
    p.row_tiles = l.row_tiles;
    p.tiles = (slots + TILE - 1) / TILE;
    p.rows = a.T * (a.n_q / a.n_kv);
    p.kv_dtype = kv_dtype;
    p.spin = ctx->mbar_spin_limit;
    return a.hd == 64 ? launch_prompt<64>(ctx, p, kv_dtype) : launch_prompt<128>(ctx, p, kv_dtype);
}
