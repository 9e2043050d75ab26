//! Raw bindings of libhs_attn.so (include/hs_attn.h) and libhs_kv_cache.so (include/hs_kv_cache.h).
//! The `extern "C"` blocks are generated by gen_bindings.py from the headers; do not edit them by hand.
#![allow(non_camel_case_types)]
use std::ffi::{c_char, c_int, c_void};

/// `hipStream_t`; null = the default stream (what tch / libtorch uses), as `bnb_stream_t`.
pub type hs_stream_t = *mut c_void;

pub const HS_ATTN_ABI_VERSION: c_int = 8;
pub const HS_ATTN_ABI_REVISION: c_int = 1;

// enum hs_status
pub const HS_OK: c_int = 0;
pub const HS_ERR_INVALID_ARGUMENT: c_int = 1;
pub const HS_ERR_OVERFLOW: c_int = 2;
pub const HS_ERR_WORKSPACE: c_int = 3;
pub const HS_ERR_LAUNCH: c_int = 4;
pub const HS_ERR_POOL_EXHAUSTED: c_int = 5;
pub const HS_ERR_BUSY: c_int = 6;
// enum hs_dtype
pub const HS_BF16: c_int = 0;
pub const HS_F32: c_int = 1;
pub const HS_F16: c_int = 2;
// enum hs_qk_norm_kind
pub const HS_QKNORM_NONE: c_int = 0;
pub const HS_QKNORM_LLAMA: c_int = 1;
pub const HS_QKNORM_QWEN35: c_int = 2;
// enum hs_kv_quant (storage format of a cache object)
pub const HS_KV_NONE: c_int = 0;
pub const HS_KV_INT8: c_int = 1;
pub const HS_KV_FP8: c_int = 2;
// enum hs_kv_quant_mode (KvQuantMode of the compatibility fingerprint)
pub const HS_KVQ_NONE: c_int = 0;
pub const HS_KVQ_INT8: c_int = 1;
pub const HS_KVQ_NF4: c_int = 2;
pub const HS_KVQ_FP4: c_int = 3;
pub const HS_KVQ_INT8_TOKEN: c_int = 4;
pub const HS_KVQ_FP8_E4M3FN_HEAD: c_int = 5;
// enum hs_cache_reuse
pub const HS_REUSE: c_int = 0;
pub const HS_STAMP_FRESH: c_int = 1;
pub const HS_DISCARD_AND_RECOMPUTE: c_int = 2;

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct hs_kv_layout {
    pub code_stride_seq: i64,
    pub code_stride_head: i64,
    pub scale_stride_seq: i64,
    pub scale_stride_head: i64,
    pub capacity_tokens: i32,
    pub block_table_stride: i32,
    pub k_block_table: *const i32,
    pub v_block_table: *const i32,
    pub total_tokens_hint: i64,
    pub prefill_columns_hint: i32,
    pub prefill_window: i32,
    pub out_gate: *const c_void,
    pub prefill_q_prologue: *const hs_qk_prologue,
    pub prefill_split_workspace: *mut c_void,
    pub prefill_split_workspace_bytes: i64,
    pub prefill_key_splits: i32,
    pub attn_sinks: i32,
    pub prefill_shadow: *mut c_void,
    pub prefill_shadow_bytes: i64,
    pub prefill_shadow_tokens: i32,
    pub decode_window: i32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct hs_qk_prologue {
    pub norm_kind: i32,
    pub norm_eps: f32,
    pub q_norm_weight: *const c_void,
    pub k_norm_weight: *const c_void,
    pub q_norm_head_stride: i32,
    pub k_norm_head_stride: i32,
    pub rope_sin: *const c_void,
    pub rope_cos: *const c_void,
    pub rope_len: i32,
    pub rotary_dim: i32,
}

#[repr(C)] pub struct hs_cache { _private: [u8; 0] }
#[repr(C)] pub struct hs_pool { _private: [u8; 0] }
#[repr(C)] pub struct hs_paged_cache { _private: [u8; 0] }
#[repr(C)] pub struct hs_compat { _private: [u8; 0] }

// ---- include/hs_attn.h -> libhs_attn.so
#[link(name = "hs_attn")]
extern "C" {
    pub fn hs_attn_last_error() -> *const c_char;
    pub fn hs_attn_abi_version() -> c_int;
    pub fn hs_attn_abi_revision() -> c_int;
    pub fn hs_kv_quantize_int8(k_src: *const c_void, v_src: *const c_void, src_dtype: c_int, k_codes: *mut i8, v_codes: *mut i8, k_scales: *mut f32, v_scales: *mut f32, layout: *const hs_kv_layout, positions: *const i32, start_pos: i32, b: i32, s: i32, hkv: i32, d: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_kv_quantize_int8_rope(k_src: *const c_void, v_src: *const c_void, src_dtype: c_int, rope_sin: *const c_void, rope_cos: *const c_void, rope_len: i32, k_codes: *mut i8, v_codes: *mut i8, k_scales: *mut f32, v_scales: *mut f32, layout: *const hs_kv_layout, positions: *const i32, start_pos: i32, b: i32, s: i32, hkv: i32, d: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_rope_apply(x: *const c_void, dtype: c_int, rope_sin: *const c_void, rope_cos: *const c_void, rope_len: i32, positions: *const i32, start_pos: i32, out: *mut c_void, b: i32, s: i32, h: i32, d: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_rope_apply_partial(x: *const c_void, dtype: c_int, rope_sin: *const c_void, rope_cos: *const c_void, rope_len: i32, positions: *const i32, start_pos: i32, out: *mut c_void, b: i32, s: i32, h: i32, d: i32, rotary_dim: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_qk_prologue_apply(q: *const c_void, k: *const c_void, dtype: c_int, prologue: *const hs_qk_prologue, positions: *const i32, start_pos: i32, q_out: *mut c_void, k_out: *mut c_void, b: i32, s: i32, hq: i32, hkv: i32, d: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_kv_quantize_int8_prologue(k_src: *const c_void, v_src: *const c_void, src_dtype: c_int, prologue: *const hs_qk_prologue, k_codes: *mut i8, v_codes: *mut i8, k_scales: *mut f32, v_scales: *mut f32, layout: *const hs_kv_layout, positions: *const i32, start_pos: i32, b: i32, s: i32, hkv: i32, d: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_kv_fp8_calibrate(k_src: *const c_void, v_src: *const c_void, src_dtype: c_int, k_scales: *mut f32, v_scales: *mut f32, b: i32, s: i32, hkv: i32, d: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_kv_quantize_fp8(k_src: *const c_void, v_src: *const c_void, src_dtype: c_int, k_codes: *mut u8, v_codes: *mut u8, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, positions: *const i32, start_pos: i32, b: i32, s: i32, hkv: i32, d: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_kv_dequantize(codes: *const c_void, scales: *const f32, fmt_fp8: c_int, layout: *const hs_kv_layout, which_table: c_int, out: *mut c_void, out_dtype: c_int, b: i32, t: i32, hkv: i32, d: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_attn_workspace_bytes(b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32) -> usize;
    pub fn hs_decode_attn_num_chunks(b: i32, hkv: i32, max_seq_len: i32, total_tokens_hint: i64) -> i32;
    pub fn hs_decode_attn_int8(q: *const c_void, k_codes: *const i8, v_codes: *const i8, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_attn_int8_static(q: *const c_void, k_codes: *const i8, v_codes: *const i8, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_attn_fp8(q: *const c_void, k_codes: *const u8, v_codes: *const u8, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_step_int8(q: *const c_void, k_new: *const c_void, v_new: *const c_void, src_dtype: c_int, k_codes: *mut i8, v_codes: *mut i8, k_scales: *mut f32, v_scales: *mut f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_step_int8_rope(q: *const c_void, k_new: *const c_void, v_new: *const c_void, rope_sin: *const c_void, rope_cos: *const c_void, rope_len: i32, k_codes: *mut i8, v_codes: *mut i8, k_scales: *mut f32, v_scales: *mut f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_step_int8_prologue(q: *const c_void, k_new: *const c_void, v_new: *const c_void, prologue: *const hs_qk_prologue, k_codes: *mut i8, v_codes: *mut i8, k_scales: *mut f32, v_scales: *mut f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_step_fp8(q: *const c_void, k_new: *const c_void, v_new: *const c_void, src_dtype: c_int, k_codes: *mut u8, v_codes: *mut u8, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_step_fp8_prologue(q: *const c_void, k_new: *const c_void, v_new: *const c_void, prologue: *const hs_qk_prologue, k_codes: *mut u8, v_codes: *mut u8, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_attn_phases(fmt_fp8: c_int, phases: c_int, q: *const c_void, k_codes: *const c_void, v_codes: *const c_void, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_decode_weights_workspace_bytes(b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32) -> usize;
    pub fn hs_decode_step_weights(fmt_fp8: c_int, q: *const c_void, k_new: *const c_void, v_new: *const c_void, src_dtype: c_int, k_codes: *mut c_void, v_codes: *mut c_void, k_scales: *mut f32, v_scales: *mut f32, layout: *const hs_kv_layout, seq_lens: *const i32, out: *mut c_void, weights_in: *const f32, weights_out: *mut f32, weights_stride: i64, workspace: *mut c_void, workspace_bytes: usize, b: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_attn_weights_workspace_bytes(b: i32, s: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32) -> usize;
    pub fn hs_attn_weights(fmt_fp8: c_int, q: *const c_void, k_codes: *const c_void, k_scales: *const f32, layout: *const hs_kv_layout, positions: *const i32, start_pos: i32, weights_in: *const f32, weights_out: *mut f32, weights_stride: i64, workspace: *mut c_void, workspace_bytes: usize, b: i32, s: i32, hq: i32, hkv: i32, d: i32, max_seq_len: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_kv_evict_workspace_bytes(b: i32, hkv: i32, budget: i32, max_seq_len: i32) -> usize;
    pub fn hs_kv_evict(fmt_fp8: c_int, k_codes: *const c_void, v_codes: *const c_void, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, seq_lens: *const i32, weights: *const f32, weights_stride: i64, k_codes_out: *mut c_void, v_codes_out: *mut c_void, k_scales_out: *mut f32, v_scales_out: *mut f32, layout_out: *const hs_kv_layout, seq_lens_out: *mut i32, weights_out: *mut f32, weights_out_stride: i64, kept: *mut i32, budget: i32, sinks: i32, recent: i32, workspace: *mut c_void, workspace_bytes: usize, b: i32, hkv: i32, d: i32, max_seq_len: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_prefill_attn_int8(q: *const c_void, k_new: *const c_void, v_new: *const c_void, k_codes: *mut i8, v_codes: *mut i8, k_scales: *mut f32, v_scales: *mut f32, layout: *const hs_kv_layout, hist_len: i32, out: *mut c_void, b: i32, s: i32, hq: i32, hkv: i32, d: i32, softmax_scale: f32, quantize_on_write: c_int, stream: hs_stream_t) -> c_int;
    pub fn hs_prefill_attn_fp8(q: *const c_void, k_new: *const c_void, v_new: *const c_void, k_codes: *mut u8, v_codes: *mut u8, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, hist_len: i32, out: *mut c_void, b: i32, s: i32, hq: i32, hkv: i32, d: i32, softmax_scale: f32, quantize_on_write: c_int, stream: hs_stream_t) -> c_int;
    pub fn hs_prefill_attn_int8_ragged(q: *const c_void, k_new: *const c_void, v_new: *const c_void, k_codes: *mut i8, v_codes: *mut i8, k_scales: *mut f32, v_scales: *mut f32, layout: *const hs_kv_layout, hist_lens: *const i32, max_hist_len: i32, out: *mut c_void, b: i32, s: i32, hq: i32, hkv: i32, d: i32, softmax_scale: f32, quantize_on_write: c_int, stream: hs_stream_t) -> c_int;
    pub fn hs_prefill_attn_fp8_ragged(q: *const c_void, k_new: *const c_void, v_new: *const c_void, k_codes: *mut u8, v_codes: *mut u8, k_scales: *const f32, v_scales: *const f32, layout: *const hs_kv_layout, hist_lens: *const i32, max_hist_len: i32, out: *mut c_void, b: i32, s: i32, hq: i32, hkv: i32, d: i32, softmax_scale: f32, quantize_on_write: c_int, stream: hs_stream_t) -> c_int;
    pub fn hs_prefill_attn_split_workspace_bytes(b: i32, s: i32, hq: i32, hkv: i32, d: i32) -> usize;
    pub fn hs_prefill_attn_split_workspace_init(workspace: *mut c_void, bytes: usize, stream: hs_stream_t) -> c_int;
    pub fn hs_prefill_shadow_bytes(b: i32, hkv: i32, d: i32, max_tokens: i32) -> usize;
    pub fn hs_prefill_shadow_init(shadow: *mut c_void, bytes: usize, stream: hs_stream_t) -> c_int;
    pub fn hs_deltanet_forward(q: *const c_void, k: *const c_void, v: *const c_void, g: *const f32, beta: *const f32, state: *mut f32, out: *mut f32, b: i32, t: i32, nk: i32, nv: i32, dk: i32, dv: i32, q_scale: f32, l2norm: c_int, stream: hs_stream_t) -> c_int;
    pub fn hs_deltanet_chunked_workspace_bytes(b: i32, t: i32, nk: i32, nv: i32) -> usize;
    pub fn hs_deltanet_forward_chunked(q: *const c_void, k: *const c_void, v: *const c_void, g: *const f32, beta: *const f32, state: *mut f32, out: *mut f32, b: i32, t: i32, nk: i32, nv: i32, dk: i32, dv: i32, q_scale: f32, l2norm: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: hs_stream_t) -> c_int;
    pub fn hs_deltanet_chunked_gated_norm_workspace_bytes(b: i32, t: i32, nk: i32, nv: i32) -> usize;
    pub fn hs_deltanet_forward_chunked_gated_norm(q: *const c_void, k: *const c_void, v: *const c_void, g: *const f32, beta: *const f32, state: *mut f32, z: *const c_void, norm_weight: *const f32, norm_eps: f32, out: *mut c_void, b: i32, t: i32, nk: i32, nv: i32, dk: i32, dv: i32, q_scale: f32, l2norm: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: hs_stream_t) -> c_int;
    pub fn hs_deltanet_prepare(mixed_qkv: *const c_void, conv_weight: *const c_void, conv_state_in: *const c_void, conv_state_out: *mut c_void, a_in: *const c_void, b_in: *const c_void, neg_a_exp: *const f32, dt_bias: *const f32, q: *mut c_void, k: *mut c_void, v: *mut c_void, g: *mut f32, beta: *mut f32, b: i32, s: i32, nk: i32, nv: i32, dk: i32, dv: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_deltanet_gated_norm(x: *const f32, z: *const c_void, weight: *const f32, eps: f32, out: *mut c_void, rows: i64, d: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_deltanet_decode_layer(mixed_qkv: *const c_void, conv_weight: *const c_void, conv_state_in: *const c_void, conv_state_out: *mut c_void, a_in: *const c_void, b_in: *const c_void, neg_a_exp: *const f32, dt_bias: *const f32, z: *const c_void, norm_weight: *const f32, norm_eps: f32, state: *mut f32, out: *mut c_void, b: i32, nk: i32, nv: i32, dk: i32, dv: i32, q_scale: f32, l2norm: c_int, stream: hs_stream_t) -> c_int;
    pub fn hs_deltanet_prefill_layer_workspace_bytes(b: i32, s: i32, nk: i32, nv: i32, dk: i32, dv: i32) -> usize;
    pub fn hs_deltanet_prefill_layer(mixed_qkv: *const c_void, conv_weight: *const c_void, conv_state_in: *const c_void, conv_state_out: *mut c_void, a_in: *const c_void, b_in: *const c_void, neg_a_exp: *const f32, dt_bias: *const f32, z: *const c_void, norm_weight: *const f32, norm_eps: f32, state: *mut f32, out: *mut c_void, b: i32, s: i32, nk: i32, nv: i32, dk: i32, dv: i32, q_scale: f32, l2norm: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: hs_stream_t) -> c_int;
}

// ---- include/hs_kv_cache.h -> libhs_kv_cache.so (optional host mirror)
#[cfg(feature = "kv-cache")]
#[link(name = "hs_kv_cache")]
extern "C" {
    pub fn hs_cache_create(max_seq_len: i64, quant_type: c_int) -> *mut hs_cache;
    pub fn hs_cache_destroy(c: *mut hs_cache);
    pub fn hs_cache_last_error(c: *const hs_cache) -> *const c_char;
    pub fn hs_cache_update(c: *mut hs_cache, new_keys: *const c_void, new_values: *const c_void, dtype: c_int, batch: i32, seq_len: i32, num_kv_heads: i32, head_dim: i32, start_pos: i64, stream: hs_stream_t) -> c_int;
    pub fn hs_cache_get_dense(c: *mut hs_cache, keys_out: *mut c_void, values_out: *mut c_void, dtype: c_int, stream: hs_stream_t) -> c_int;
    pub fn hs_cache_get_view(c: *mut hs_cache, k_codes: *mut *mut c_void, v_codes: *mut *mut c_void, k_scales: *mut *mut f32, v_scales: *mut *mut f32, layout: *mut hs_kv_layout, batch: *mut i32, num_kv_heads: *mut i32, head_dim: *mut i32) -> c_int;
    pub fn hs_cache_seq_pos(c: *const hs_cache) -> i64;
    pub fn hs_cache_max_seq_len(c: *const hs_cache) -> i64;
    pub fn hs_cache_clear(c: *mut hs_cache);
    pub fn hs_cache_truncate_to(c: *mut hs_cache, pos: i64);
    pub fn hs_cache_is_initialized(c: *const hs_cache) -> c_int;
    pub fn hs_cache_memory_usage(c: *const hs_cache) -> i64;
    pub fn hs_cache_quant_type(c: *const hs_cache) -> c_int;
    pub fn hs_kv_quant_canonical_str(quant_type: c_int) -> *const c_char;
    pub fn hs_compat_create() -> *mut hs_compat;
    pub fn hs_compat_destroy(c: *mut hs_compat);
    pub fn hs_compat_set_uint(c: *mut hs_compat, field: *const c_char, value: u64) -> c_int;
    pub fn hs_compat_set_opt_uint(c: *mut hs_compat, field: *const c_char, has_value: c_int, value: u64) -> c_int;
    pub fn hs_compat_set_str(c: *mut hs_compat, field: *const c_char, value: *const c_char) -> c_int;
    pub fn hs_compat_add_layer_type(c: *mut hs_compat, value: *const c_char) -> c_int;
    pub fn hs_compat_set_rope_scaling(c: *mut hs_compat, rope_type: *const c_char, factor: f32) -> c_int;
    pub fn hs_compat_set_kv_quant(c: *mut hs_compat, mode: c_int) -> c_int;
    pub fn hs_compat_is_authoritatively_complete(c: *const hs_compat) -> c_int;
    pub fn hs_compat_fingerprint(c: *const hs_compat, out32: *mut u8) -> c_int;
    pub fn hs_compat_check(expected: *const hs_compat, observed: *const hs_compat, field: *mut c_char, field_cap: usize) -> c_int;
    pub fn hs_compat_decide_reuse(expected32: *const u8, stored32: *const u8, cache_is_empty: c_int) -> c_int;
    pub fn hs_kv_quant_mode_str(mode: c_int) -> *const c_char;
    pub fn hs_kv_quant_mode_of(quant_type: c_int) -> c_int;
    pub fn hs_cache_decode_attention(c: *mut hs_cache, q: *const c_void, out: *mut c_void, num_q_heads: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_cache_decode_step(c: *mut hs_cache, q: *const c_void, k_new: *const c_void, v_new: *const c_void, dtype: c_int, out: *mut c_void, num_q_heads: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_cache_prefill(c: *mut hs_cache, q: *const c_void, new_keys: *const c_void, new_values: *const c_void, out: *mut c_void, batch: i32, seq_len: i32, num_q_heads: i32, num_kv_heads: i32, head_dim: i32, start_pos: i64, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_cache_set_window(c: *mut hs_cache, window: i32, sinks: i32) -> c_int;
    pub fn hs_cache_track_weights(c: *mut hs_cache, on: c_int) -> c_int;
    pub fn hs_cache_get_weights(c: *mut hs_cache, weights_out: *mut f32, stream: hs_stream_t) -> c_int;
    pub fn hs_cache_evict(c: *mut hs_cache, budget: i32, sinks: i32, recent: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_cache_enable_prompt_scratch(c: *mut hs_cache, max_prompt_tokens: i64);
    pub fn hs_cache_drop_prompt_scratch(c: *mut hs_cache);
    pub fn hs_cache_prompt_copy_active(c: *const hs_cache) -> c_int;
    pub fn hs_pool_create(num_blocks: i64, num_kv_heads: i32, head_dim: i32) -> *mut hs_pool;
    pub fn hs_pool_create_format(num_blocks: i64, num_kv_heads: i32, head_dim: i32, quant_type: c_int) -> *mut hs_pool;
    pub fn hs_pool_quant_type(p: *const hs_pool) -> c_int;
    pub fn hs_pool_destroy(p: *mut hs_pool);
    pub fn hs_pool_last_error(p: *const hs_pool) -> *const c_char;
    pub fn hs_pool_allocate(p: *mut hs_pool, owner_kind: c_int, owner_id: u64, owner_name: *const c_char, block_id: *mut i32) -> c_int;
    pub fn hs_pool_free(p: *mut hs_pool, owner_kind: c_int, owner_id: u64, owner_name: *const c_char, block_id: i32) -> c_int;
    pub fn hs_pool_owner_of(p: *const hs_pool, block_id: i32, owner_kind: *mut c_int, owner_id: *mut u64, owner_name: *mut c_char, owner_name_cap: usize) -> c_int;
    pub fn hs_pool_used_blocks(p: *const hs_pool) -> i64;
    pub fn hs_pool_free_block_count(p: *const hs_pool) -> i64;
    pub fn hs_pool_total_blocks(p: *const hs_pool) -> i64;
    pub fn hs_pool_used_memory(p: *const hs_pool) -> i64;
    pub fn hs_paged_cache_create(max_seq_len: i64, pool: *mut hs_pool, owner_kind: c_int, owner_id: u64, owner_name: *const c_char) -> *mut hs_paged_cache;
    pub fn hs_paged_cache_destroy(c: *mut hs_paged_cache);
    pub fn hs_paged_cache_last_error(c: *const hs_paged_cache) -> *const c_char;
    pub fn hs_paged_cache_update(c: *mut hs_paged_cache, new_keys: *const c_void, new_values: *const c_void, dtype: c_int, seq_len: i32, start_pos: i64, stream: hs_stream_t) -> c_int;
    pub fn hs_paged_cache_get_dense(c: *mut hs_paged_cache, keys_out: *mut c_void, values_out: *mut c_void, dtype: c_int, stream: hs_stream_t) -> c_int;
    pub fn hs_paged_cache_decode_attention(c: *mut hs_paged_cache, q: *const c_void, out: *mut c_void, num_q_heads: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_paged_cache_prefill(c: *mut hs_paged_cache, q: *const c_void, new_keys: *const c_void, new_values: *const c_void, out: *mut c_void, seq_len: i32, num_q_heads: i32, start_pos: i64, softmax_scale: f32, stream: hs_stream_t) -> c_int;
    pub fn hs_paged_cache_clear(c: *mut hs_paged_cache);
    pub fn hs_paged_cache_truncate_to(c: *mut hs_paged_cache, pos: i64);
    pub fn hs_paged_cache_get_view(c: *mut hs_paged_cache, k_codes: *mut *mut c_void, v_codes: *mut *mut c_void, k_scales: *mut *mut f32, v_scales: *mut *mut f32, layout: *mut hs_kv_layout, stream: hs_stream_t) -> c_int;
    pub fn hs_paged_cache_evict(c: *mut hs_paged_cache, weights: *mut f32, weights_stride: i64, budget: i32, sinks: i32, recent: i32, stream: hs_stream_t) -> c_int;
    pub fn hs_paged_cache_seq_pos(c: *const hs_paged_cache) -> i64;
    pub fn hs_paged_cache_num_blocks(c: *const hs_paged_cache) -> i64;
    pub fn hs_paged_batch_decode_step(pool: *mut hs_pool, rows: *const *mut hs_paged_cache, n: i32, q: *const c_void, k_new: *const c_void, v_new: *const c_void, dtype: c_int, out: *mut c_void, num_q_heads: i32, softmax_scale: f32, stream: hs_stream_t) -> c_int;
}
