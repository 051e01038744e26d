// Generated by gen_ffi.py from include/agention_b200.h — do not edit by hand.
// One declaration per AGN_API entry point, same order as the header.
#![allow(dead_code)]
use std::ffi::{c_char, c_int, c_void};

#[repr(C)] pub struct AgnCtx { _private: [u8; 0] }
#[repr(C)] pub struct AgnEvent { _private: [u8; 0] }
#[repr(C)] pub struct AgnGraph { _private: [u8; 0] }
#[repr(C)] pub struct AgnGguf { _private: [u8; 0] }

/// `agn_tensor_info`: `TensorInfo` (src/types.rs:373-403) plus derived sizes.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct AgnTensorInfo {
    pub name: *const c_char,
    pub ggml_type: i32,
    pub n_dims: u32,
    pub dims: [u64; 4],
    pub byte_offset: u64,
    pub file_offset: u64,
    pub n_rows: u64,
    pub row_len: u64,
    pub row_bytes: u64,
    pub n_bytes: u64,
}

pub const AGN_OK: i32 = 0;
pub const AGN_EINVAL: i32 = 1;
pub const AGN_EUNSUPPORTED_DTYPE: i32 = 2;
pub const AGN_ECUDA: i32 = 3;
pub const AGN_EOOB_ID: i32 = 4;
pub const AGN_ENOMEM: i32 = 5;
pub const AGN_ETIMEOUT: i32 = 6;
pub const AGN_EFORMAT: i32 = 7;
pub const AGN_ENOTFOUND: i32 = 8;
pub const AGN_EIO: i32 = 9;

pub const AGN_F32: i32 = 0;
pub const AGN_F16: i32 = 1;
pub const AGN_Q5_0: i32 = 6;
pub const AGN_Q8_0: i32 = 8;
pub const AGN_Q2_K: i32 = 10;
pub const AGN_Q4_K: i32 = 12;
pub const AGN_Q5_K: i32 = 13;
pub const AGN_Q6_K: i32 = 14;
pub const AGN_BF16: i32 = 30;
pub const AGN_KV_Q8_0_WORDS: i32 = 1008;

pub const AGN_ROPE_NEOX: i32 = 0;
pub const AGN_ROPE_NORMAL: i32 = 1;

#[link(name = "agention_b200")]
extern "C" {
    pub fn agn_ctx_create(device: i32, out: *mut *mut AgnCtx) -> i32;
    pub fn agn_ctx_destroy(ctx: *mut AgnCtx) -> i32;
    pub fn agn_backend_name() -> *const c_char;
    pub fn agn_last_error(ctx: *mut AgnCtx) -> *const c_char;
    pub fn agn_status_string(status: i32) -> *const c_char;
    pub fn agn_ctx_set_stream(ctx: *mut AgnCtx, cuda_stream: *mut c_void) -> i32;
    pub fn agn_ctx_get_stream(ctx: *mut AgnCtx, cuda_stream: *mut *mut c_void) -> i32;
    pub fn agn_ctx_set_option(ctx: *mut AgnCtx, name: *const c_char, value: i64) -> i32;
    pub fn agn_launch_noop(ctx: *mut AgnCtx) -> i32;
    pub fn agn_ctx_launch_count(ctx: *mut AgnCtx) -> u64;
    pub fn agn_ctx_last_kernel(ctx: *mut AgnCtx) -> *const c_char;
    pub fn agn_malloc(ctx: *mut AgnCtx, bytes: usize, dptr: *mut *mut c_void) -> i32;
    pub fn agn_free(ctx: *mut AgnCtx, dptr: *mut c_void) -> i32;
    pub fn agn_host_alloc(ctx: *mut AgnCtx, bytes: usize, hptr: *mut *mut c_void) -> i32;
    pub fn agn_host_free(ctx: *mut AgnCtx, hptr: *mut c_void) -> i32;
    pub fn agn_memcpy_h2d(ctx: *mut AgnCtx, dst: *mut c_void, src: *const c_void, bytes: usize) -> i32;
    pub fn agn_memcpy_d2h(ctx: *mut AgnCtx, dst: *mut c_void, src: *const c_void, bytes: usize) -> i32;
    pub fn agn_memset(ctx: *mut AgnCtx, dst: *mut c_void, value: c_int, bytes: usize) -> i32;
    pub fn agn_sync(ctx: *mut AgnCtx) -> i32;
    pub fn agn_event_create(ctx: *mut AgnCtx, ev: *mut *mut AgnEvent) -> i32;
    pub fn agn_event_record(ctx: *mut AgnCtx, ev: *mut AgnEvent) -> i32;
    pub fn agn_event_elapsed_ms(ctx: *mut AgnCtx, start: *mut AgnEvent, stop: *mut AgnEvent, ms: *mut f32) -> i32;
    pub fn agn_event_destroy(ctx: *mut AgnCtx, ev: *mut AgnEvent) -> i32;
    pub fn agn_graph_begin(ctx: *mut AgnCtx) -> i32;
    pub fn agn_graph_end(ctx: *mut AgnCtx, out: *mut *mut AgnGraph) -> i32;
    pub fn agn_graph_launch(ctx: *mut AgnCtx, graph: *mut AgnGraph) -> i32;
    pub fn agn_graph_destroy(ctx: *mut AgnCtx, graph: *mut AgnGraph) -> i32;
    pub fn agn_rms_norm_f32(ctx: *mut AgnCtx, x: *const f32, w: *const f32, out: *mut f32, T: i64, H: i64, eps: f32) -> i32;
    pub fn agn_add_residual_rms_norm_f32(ctx: *mut AgnCtx, x: *const f32, delta: *const f32, w: *const f32, new_x: *mut f32, normed: *mut f32, T: i64, H: i64, eps: f32) -> i32;
    pub fn agn_rope_freq_scale(scaling_type: *const c_char, has_factor: i32, factor: f32, scale: *mut f32) -> i32;
    pub fn agn_rope_f32(ctx: *mut AgnCtx, x: *mut f32, T: i64, n_heads: i32, head_dim: i32, n_rot: i32, pos: *const i32, pos_start: i32, theta: f32, freq_scale: f32, layout: i32) -> i32;
    pub fn agn_rope_qk_f32(ctx: *mut AgnCtx, q: *mut f32, k: *mut f32, T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, n_rot: i32, pos: *const i32, pos_start: i32, theta: f32, freq_scale: f32, layout: i32) -> i32;
    pub fn agn_qk_norm_rope_f32(ctx: *mut AgnCtx, x: *mut f32, w: *const f32, T: i64, n_heads: i32, head_dim: i32, eps: f32, n_rot: i32, pos: *const i32, pos_start: i32, theta: f32, freq_scale: f32, layout: i32) -> i32;
    pub fn agn_qk_norm_rope_qk_f32(ctx: *mut AgnCtx, q: *mut f32, k: *mut f32, wq: *const f32, wk: *const f32, T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, eps: f32, n_rot: i32, pos: *const i32, pos_start: i32, theta: f32, freq_scale: f32, layout: i32) -> i32;
    pub fn agn_silu_mul_f32(ctx: *mut AgnCtx, gate: *const f32, up: *const f32, out: *mut f32, n: i64) -> i32;
    pub fn agn_softmax_rows_f32(ctx: *mut AgnCtx, input: *const f32, out: *mut f32, n_rows: i64, row_len: i64, row_stride: i64, n_valid: *const i32, causal_period: i32, causal_offset: i32) -> i32;
    pub fn agn_softmax_rows_unnorm_f32(ctx: *mut AgnCtx, input: *const f32, weights: *mut f32, sums: *mut f32, n_rows: i64, row_len: i64, row_stride: i64, n_valid: *const i32, causal_period: i32, causal_offset: i32) -> i32;
    pub fn agn_softmax_rows_scaled_f32(ctx: *mut AgnCtx, input: *const f32, out: *mut f32, sums: *mut f32, n_rows: i64, row_len: i64, row_stride: i64, n_valid: *const i32, causal_period: i32, causal_offset: i32, scale: f32) -> i32;
    pub fn agn_softmax_rows_scaled_f32_out16(ctx: *mut AgnCtx, input: *const f32, out: *mut c_void, sums: *mut f32, n_rows: i64, row_len: i64, row_stride: i64, n_valid: *const i32, causal_period: i32, causal_offset: i32, scale: f32, out_dtype: i32) -> i32;
    pub fn agn_softmax_rows_valid_f32(ctx: *mut AgnCtx, input: *const f32, out: *mut c_void, sums: *mut f32, n_rows: i64, row_len: i64, row_stride: i64, n_valid: *const i32, causal_period: i32, causal_offset: i32, scale: f32, out_dtype: i32) -> i32;
    pub fn agn_get_rows_f32(ctx: *mut AgnCtx, dtype: i32, table: *const c_void, table_bytes: usize, n_rows: i64, row_len: i64, ids: *const u32, T: i64, out: *mut f32) -> i32;
    pub fn agn_kv_write_f32(ctx: *mut AgnCtx, kv_dtype: i32, k: *const f32, v: *const f32, k_cache: *mut c_void, v_cache: *mut c_void, T: i64, head_dim_kv: i64, pos: *const i32, pos_start: i32, max_seq_len: i64) -> i32;
    pub fn agn_qk_norm_rope_kv_write_f32(ctx: *mut AgnCtx, q: *mut f32, k: *mut f32, v: *const f32, wq: *const f32, wk: *const f32, T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, eps: f32, n_rot: i32, pos: *const i32, pos_start: i32, theta: f32, freq_scale: f32, layout: i32, kv_dtype: i32, k_cache: *mut c_void, v_cache: *mut c_void, max_seq_len: i64) -> i32;
    pub fn agn_kv_read_f32(ctx: *mut AgnCtx, kv_dtype: i32, k_cache: *const c_void, v_cache: *const c_void, n_pos: i64, head_dim_kv: i64, k_out: *mut f32, v_out: *mut f32) -> i32;
    pub fn agn_kv_bytes_per_token(kv_dtype: i32, head_dim_kv: i64) -> i64;
    pub fn agn_attention_kv_workspace_bytes(T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, max_seq_len: i64, has_pos: i32) -> i64;
    pub fn agn_attention_kv_f32(ctx: *mut AgnCtx, q: *const f32, out: *mut f32, kv_dtype: i32, k_cache: *const c_void, v_cache: *const c_void, T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, pos: *const i32, pos_start: i32, seq: *const i32, n_seqs: i64, max_seq_len: i64, scale: f32, workspace: *mut c_void, workspace_bytes: usize) -> i32;
    pub fn agn_attention_kv_f16(ctx: *mut AgnCtx, q: *const c_void, out: *mut c_void, kv_dtype: i32, k_cache: *const c_void, v_cache: *const c_void, T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, pos: *const i32, pos_start: i32, seq: *const i32, n_seqs: i64, max_seq_len: i64, scale: f32, workspace: *mut c_void, workspace_bytes: usize) -> i32;
    pub fn agn_gated_delta_rule_workspace_bytes(T: i64, n_seqs: i64, n_k_heads: i32, n_v_heads: i32, head_k: i32, head_v: i32) -> i64;
    pub fn agn_gated_delta_rule_f32(ctx: *mut AgnCtx, q: *const f32, k: *const f32, v: *const f32, g: *const f32, beta: *const f32, state_in: *const f32, state_out: *mut f32, out: *mut f32, T: i64, n_seqs: i64, cu_seqlens: *const i32, n_k_heads: i32, n_v_heads: i32, head_k: i32, head_v: i32, q_stride: i64, k_stride: i64, v_stride: i64, scale: f32, l2norm_eps: f32, workspace: *mut c_void, workspace_bytes: usize) -> i32;
    pub fn agn_rms_norm_silu_gate_f32(ctx: *mut AgnCtx, x: *const f32, gate: *const f32, w: *const f32, out: *mut f32, rows: i64, n: i64, eps: f32) -> i32;
    pub fn agn_rms_norm_silu_gate_f32_out16(ctx: *mut AgnCtx, x: *const f32, gate: *const f32, w: *const f32, out: *mut c_void, rows: i64, n: i64, eps: f32, out_dtype: i32) -> i32;
    pub fn agn_router_top2_f32(ctx: *mut AgnCtx, logits: *const f32, T: i64, n_experts: i32, idx: *mut i32, w: *mut f32) -> i32;
    pub fn agn_gather_rows_by_expert_f32(ctx: *mut AgnCtx, x: *const f32, idx: *const i32, T: i64, H: i64, n_experts: i32, out: *mut f32, offsets: *mut i32, src_token: *mut i32, src_slot: *mut i32) -> i32;
    pub fn agn_silu_mul_f16(ctx: *mut AgnCtx, gate: *const c_void, up: *const c_void, out: *mut c_void, n: i64) -> i32;
    pub fn agn_rms_norm_f16(ctx: *mut AgnCtx, x: *const c_void, w: *const f32, out: *mut c_void, T: i64, H: i64, eps: f32) -> i32;
    pub fn agn_add_residual_rms_norm_f16(ctx: *mut AgnCtx, x: *const c_void, delta: *const c_void, w: *const f32, new_x: *mut c_void, normed: *mut c_void, T: i64, H: i64, eps: f32) -> i32;
    pub fn agn_silu_mul_f32_out16(ctx: *mut AgnCtx, gate: *const f32, up: *const f32, out: *mut c_void, n: i64, out_dtype: i32) -> i32;
    pub fn agn_rms_norm_f32_out16(ctx: *mut AgnCtx, x: *const f32, w: *const f32, out: *mut c_void, T: i64, H: i64, eps: f32, out_dtype: i32) -> i32;
    pub fn agn_add_residual_rms_norm_f32_out16(ctx: *mut AgnCtx, x: *const f32, delta: *const f32, w: *const f32, new_x: *mut f32, normed: *mut c_void, T: i64, H: i64, eps: f32, out_dtype: i32) -> i32;
    pub fn agn_q8_k_blocks(n: i64) -> i64;
    pub fn agn_quantize_rows_q8_k_f32(ctx: *mut AgnCtx, x: *const f32, T: i64, n: i64, d: *mut f32, qs: *mut i8, bsums: *mut i16) -> i32;
    pub fn agn_rms_norm_q8_k_f32(ctx: *mut AgnCtx, x: *const f32, w: *const f32, T: i64, H: i64, eps: f32, d: *mut f32, qs: *mut i8, bsums: *mut i16) -> i32;
    pub fn agn_add_residual_rms_norm_q8_k_f32(ctx: *mut AgnCtx, x: *const f32, delta: *const f32, w: *const f32, new_x: *mut f32, T: i64, H: i64, eps: f32, d: *mut f32, qs: *mut i8, bsums: *mut i16) -> i32;
    pub fn agn_silu_mul_q8_k_f32(ctx: *mut AgnCtx, gate: *const f32, up: *const f32, T: i64, I: i64, d: *mut f32, qs: *mut i8, bsums: *mut i16) -> i32;
    pub fn agn_rope_qk_f16(ctx: *mut AgnCtx, q: *mut c_void, k: *mut c_void, T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, n_rot: i32, pos: *const i32, pos_start: i32, theta: f32, freq_scale: f32, layout: i32) -> i32;
    pub fn agn_qk_norm_rope_qk_f16(ctx: *mut AgnCtx, q: *mut c_void, k: *mut c_void, wq: *const f32, wk: *const f32, T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, eps: f32, n_rot: i32, pos: *const i32, pos_start: i32, theta: f32, freq_scale: f32, layout: i32) -> i32;
    pub fn agn_get_rows_f16(ctx: *mut AgnCtx, dtype: i32, table: *const c_void, table_bytes: usize, n_rows: i64, row_len: i64, ids: *const u32, T: i64, out: *mut c_void) -> i32;
    pub fn agn_host_rms_norm_f32(ctx: *mut AgnCtx, x_host: *const f32, w_dev: *const f32, out_host: *mut f32, T: i64, H: i64, eps: f32) -> i32;
    pub fn agn_host_add_residual_rms_norm_f32(ctx: *mut AgnCtx, x_host: *mut f32, delta_host: *const f32, w_dev: *const f32, normed_host: *mut f32, T: i64, H: i64, eps: f32) -> i32;
    pub fn agn_host_silu_mul_f32(ctx: *mut AgnCtx, gate_host: *const f32, up_host: *const f32, out_host: *mut f32, n: i64) -> i32;
    pub fn agn_host_rope_qk_f32(ctx: *mut AgnCtx, q_host: *mut f32, k_host: *mut f32, T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, n_rot: i32, pos_host: *const i32, pos_start: i32, theta: f32, freq_scale: f32, layout: i32) -> i32;
    pub fn agn_host_qk_norm_rope_qk_f32(ctx: *mut AgnCtx, q_host: *mut f32, k_host: *mut f32, wq_dev: *const f32, wk_dev: *const f32, T: i64, n_q_heads: i32, n_kv_heads: i32, head_dim: i32, eps: f32, n_rot: i32, pos_host: *const i32, pos_start: i32, theta: f32, freq_scale: f32, layout: i32) -> i32;
    pub fn agn_host_softmax_rows_f32(ctx: *mut AgnCtx, in_host: *const f32, out_host: *mut f32, n_rows: i64, row_len: i64, n_valid_host: *const i32, causal_period: i32, causal_offset: i32) -> i32;
    pub fn agn_host_get_rows_f32(ctx: *mut AgnCtx, dtype: i32, table_dev: *const c_void, table_bytes: usize, n_rows: i64, row_len: i64, ids_host: *const u32, T: i64, out_host: *mut f32) -> i32;
    pub fn agn_host_quantize_rows_q8_k_f32(ctx: *mut AgnCtx, x_host: *const f32, T: i64, n: i64, d_host: *mut f32, qs_host: *mut i8, bsums_host: *mut i16) -> i32;
    pub fn agn_gather_rows_by_expert_noalloc_f32(cuda_stream: *mut c_void, x: *const f32, idx: *const i32, T: i64, H: i64, n_experts: i32, out: *mut f32, offsets: *mut i32, src_token: *mut i32, src_slot: *mut i32, err: *mut c_char, err_len: usize) -> i32;
    pub fn agn_gguf_parse(data: *const c_void, len: usize, out: *mut *mut AgnGguf, err: *mut c_char, err_len: usize) -> i32;
    pub fn agn_gguf_open(path: *const c_char, out: *mut *mut AgnGguf, err: *mut c_char, err_len: usize) -> i32;
    pub fn agn_gguf_split_index(name: *const c_char, index: *mut u64, total: *mut u64) -> i32;
    pub fn agn_gguf_close(g: *mut AgnGguf) -> i32;
    pub fn agn_gguf_version(g: *const AgnGguf) -> u32;
    pub fn agn_gguf_tensor_count(g: *const AgnGguf) -> u64;
    pub fn agn_gguf_metadata_count(g: *const AgnGguf) -> u64;
    pub fn agn_gguf_data_offset(g: *const AgnGguf) -> u64;
    pub fn agn_gguf_get_u64(g: *const AgnGguf, key: *const c_char, out: *mut u64) -> i32;
    pub fn agn_gguf_get_f32(g: *const AgnGguf, key: *const c_char, out: *mut f32) -> i32;
    pub fn agn_gguf_get_string(g: *const AgnGguf, key: *const c_char, out: *mut *const c_char) -> i32;
    pub fn agn_gguf_get_array_i64(g: *const AgnGguf, key: *const c_char, out: *mut i64, cap: u64, count: *mut u64) -> i32;
    pub fn agn_gguf_get_array_info(g: *const AgnGguf, key: *const c_char, elem_type: *mut u32, count: *mut u64) -> i32;
    pub fn agn_gguf_tensor_at(g: *const AgnGguf, index: u64, out: *mut AgnTensorInfo) -> i32;
    pub fn agn_gguf_find_tensor(g: *const AgnGguf, name: *const c_char, out: *mut AgnTensorInfo) -> i32;
    pub fn agn_gguf_upload_tensor(ctx: *mut AgnCtx, g: *const AgnGguf, name: *const c_char, dptr: *mut *mut c_void, info: *mut AgnTensorInfo) -> i32;
    pub fn agn_gguf_tensor_data(g: *const AgnGguf, name: *const c_char, data: *mut *const c_void, n_bytes: *mut u64) -> i32;
    pub fn agn_gguf_upload_tensors(ctx: *mut AgnCtx, g: *const AgnGguf, names: *const *const c_char, n: u64, dptrs: *mut *mut c_void, infos: *mut AgnTensorInfo, release_pages: i32, released_bytes: *mut u64) -> i32;
    pub fn agn_gguf_release_pages(g: *const AgnGguf, from: u64, to: u64, released_bytes: *mut u64) -> i32;
    pub fn agn_type_size(dtype: i32, n: usize) -> usize;
}
