// What the attention kernels share: the call's arguments and the cache's block formats.
#pragma once
#include <math.h>

#include "agn_common.cuh"

struct AttnArgs {
    const void *q;
    void *out;
    const unsigned char *k_cache, *v_cache;
    const int32_t *pos, *seq;
    int64_t T, n_seqs, max_seq;
    int n_q, n_kv, hd, pos_start, bytes_per_token;
    float scale;
    uint32_t *flags;
};

constexpr int ATTN_MAX_SMS = 148;

// A prompt's rows over a long cache are too few CTAs when the rows are few: the slots are then shared out as well.  Split x of a row leaves part[x][row][hd + 4] (row =
// token * n_q + head): the sums of weighted values, the reference maximum (log2) and the sum of weights; agn_attention_join adds them up.
struct AttnSplit {
    float *part;
    int splits;  // 1: rows are written as they are
};
// The number of splits, up to one CTA per SM, that is the quickest by a model of two terms: the tiles that follow one another in a CTA (tile_us each), and,
// where there are splits, 6 us for one more launch and the shares' way through memory at 2.5 TB/s.  (32 rows of 28/4 heads of 128 over 8000 q8_0 slots, f16: one share
// 161 us, 37 shares 40 us; 512 rows over 1000 slots: one share 42 us, two 62 us.)
inline int attn_splits(int64_t ctas, int64_t tiles, double tile_us, int64_t rows, int hd, int sms) {
    int best = 1;
    double least = tiles * tile_us;
    for (int64_t n = 2; n <= sms / (ctas > 0 ? ctas : 1) && n <= tiles; n++) {
        const double us = (double)((tiles + n - 1) / n) * tile_us + 6.0 + (double)(rows * n) * (hd + 4) * 8 / 2.5e6;
        if (us < least) {
            least = us;
            best = (int)n;
        }
    }
    return best;
}
// A bound on that number for rows that end anywhere in `tiles` tiles: splits have to save more than they cost.  (The number itself does not only grow with the tiles:
// 10 tiles may go to 10 CTAs, 12 tiles to 6.)
inline int attn_splits_most(int64_t ctas, int64_t tiles, double tile_us, int64_t rows, int hd, int sms) {
    int64_t n = sms / (ctas > 0 ? ctas : 1);
    const double paid = (tiles * tile_us - 6.0) / ((double)rows * (hd + 4) * 8 / 2.5e6);
    if (n > tiles) n = tiles;
    if ((double)n > paid) n = paid > 1.0 ? (int64_t)paid : 1;
    return n > 1 ? (int)n : 1;
}
inline int64_t attn_part_bytes(int splits, int64_t T, int n_q, int hd) { return splits > 1 ? (int64_t)splits * T * n_q * (hd + 4) * 4 : 0; }
// odd: [n_kv][odd_tiles] flags of groups of `group` slots whose values are not all finite (they were taken as 0), or null: look at every slot.
int32_t agn_attention_join(agn_ctx *ctx, const AttnArgs &a, int kv_dtype, int act16, AttnSplit split, const int *odd, int64_t odd_tiles, int group);

// Rows of a prompt in f16 on the tensor cores (agn_attention_prompt.cu), where that form covers the call.
bool agn_attention_prompt_fits(int64_t T, int n_q, int n_kv, int hd);
// `anywhere`: enough for rows that end at any slot up to that one; otherwise what rows that end there take.
int64_t agn_attention_prompt_workspace(int64_t slots, int64_t T, int n_q, int n_kv, int hd, int sms, bool anywhere);
int32_t agn_attention_prompt_f16(agn_ctx *ctx, const AttnArgs &a, int kv_dtype, void *workspace);

// Rows of a prompt that the form above does not cover: f32 rows, other head sizes (agn_attention_chunk.cu).
int64_t agn_attention_chunk_workspace(int64_t slots, int64_t T, int n_q, int n_kv, int hd, int sms, bool anywhere);
int32_t agn_attention_chunk(agn_ctx *ctx, const AttnArgs &a, int kv_dtype, int act16, void *workspace);

constexpr int KV_F16 = 0, KV_Q8 = 1, KV_WORDS = 2;
template <int KV> struct KvFormat;  // a block of 32 values of one head: BYTES, with the values DATA bytes behind its start
template <> struct KvFormat<KV_F16> { static constexpr int BYTES = 64, DATA = 0; };
template <> struct KvFormat<KV_Q8> { static constexpr int BYTES = 34, DATA = 2; };
template <> struct KvFormat<KV_WORDS> { static constexpr int BYTES = 36, DATA = 4; };

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int KV> __device__ __forceinline__ float block_scale(const unsigned char *blk) {
    if (KV == KV_WORDS) return *reinterpret_cast<const float *>(blk);
    return __half2float(*reinterpret_cast<const __half *>(blk));
}

// What becomes f16 without turning into infinity or NaN.
__device__ __forceinline__ bool half_finite(float v) { return (__half_as_ushort(__float2half_rn(v)) & 0x7c00) != 0x7c00; }
// One value of a cache row (dims of all its heads).
template <int KV> __device__ __forceinline__ float cache_value(const unsigned char *row, int d) {
    if (KV == KV_F16) return __half2float(reinterpret_cast<const __half *>(row)[d]);
    const unsigned char *blk = row + (d >> 5) * KvFormat<KV>::BYTES;
    const int u = blk[KvFormat<KV>::DATA + (d & 31)];
    return (float)(KV == KV_Q8 ? (int)(signed char)u : u - 128) * block_scale<KV>(blk);
}
// Where values that are not finite were taken as 0: what a row that sees slots 0 .. last has to get added for dim d of the cache row.  Infinity of the one sign that it
// sees, NaN for a NaN or for both signs, 0 where there is none.  look(slot): whether the slot's group of `group` slots holds any.
template <typename Look> __device__ __forceinline__ float odd_value(const AttnArgs &a, int kv_dtype, int d, int last, Look look, int group) {
    bool up = false, down = false;
    for (int s = 0; s <= last; s++) {
        if (!look(s)) {
            s += group - 1 - s % group;
            continue;
        }
        const unsigned char *row = a.v_cache + (int64_t)s * a.bytes_per_token;
        const float v = kv_dtype == AGN_F16 ? cache_value<KV_F16>(row, d) : kv_dtype == AGN_Q8_0 ? cache_value<KV_Q8>(row, d) : cache_value<KV_WORDS>(row, d);
        if (fabsf(v) < INFINITY) continue;
        if (v != v) return NAN;
        if (v > 0.0f) up = true;
        else down = true;
    }
    return up && down ? NAN : up ? INFINITY : down ? -INFINITY : 0.0f;
}
