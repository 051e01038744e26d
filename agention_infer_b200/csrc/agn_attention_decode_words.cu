// attn_decode_kernel over a Q8_0 in blocks of nine words cache.
#include "agn_attention_decode.cuh"

int32_t agn_attention_decode_words(agn_ctx *ctx, const DecodeArgs &d, dim3 grid, size_t smem) { return launch_decode<KV_WORDS>(ctx, d, grid, smem); }
