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

// Rows of a prompt in f16 on the tensor cores (agn_attention_prompt.cu), where that form covers the call.
#define AGN_PROMPT_MIN_ROWS 128
#define AGN_PROMPT_MIN_TOKENS 16
bool agn_attention_prompt_fits(int64_t T, int n_q, int n_kv, int hd);
int64_t agn_attention_prompt_workspace(int64_t slots, int n_kv, int hd);
int32_t agn_attention_prompt_f16(agn_ctx *ctx, const AttnArgs &a, int kv_dtype, void *workspace);

// Rows of a prompt that the form above does not cover: f32 rows, other head sizes (agn_attention_chunk.cu).
int32_t agn_attention_chunk(agn_ctx *ctx, const AttnArgs &a, int kv_dtype, int act16);

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
            s |= group - 1;
            continue;
        }
        const unsigned char *row = a.v_cache + (int64_t)s * a.bytes_per_token;
        const float v = kv_dtype == AGN_F16 ? cache_value<KV_F16>(row, d) : kv_dtype == AGN_Q8_0 ? cache_value<KV_Q8>(row, d) : cache_value<KV_WORDS>(row, d);
        if (half_finite(v)) continue;
        if (v != v) return NAN;
        if (v > 0.0f) up = true;
        else down = true;
    }
    return up && down ? NAN : up ? INFINITY : down ? -INFINITY : 0.0f;
}
