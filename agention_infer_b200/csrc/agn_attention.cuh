// What the attention kernels share: the call's arguments and the cache's block formats.
#pragma once
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
