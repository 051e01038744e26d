// attn_decode_kernel over an f16 cache.
#include "agn_attention_decode.cuh"

int32_t agn_attention_decode_f16(agn_ctx *ctx, const DecodeArgs &d, dim3 grid, size_t smem) { return launch_decode<KV_F16>(ctx, d, grid, smem); }
