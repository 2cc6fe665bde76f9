// Generated by integration/gen_hip_sys.py from include/rai_hip.h -- do not edit by hand.
//
// Raw FFI of librai_hip.so: the C ABI that stands behind `impl Eval<Hip, ops::X>` (backend/hip.rs).
// Counterpart in the reference: the calls into candle_core in rai-core/src/backend/candle.rs.
#![allow(non_camel_case_types, dead_code, clippy::too_many_arguments)]
use std::ffi::{c_char, c_int, c_void, CStr};

pub const RAI_HIP_MAX_RANK: usize = 8;

pub const RAI_U8: i32 = 0;
pub const RAI_U32: i32 = 1;
pub const RAI_I64: i32 = 2;
pub const RAI_F16: i32 = 3;
pub const RAI_BF16: i32 = 4;
pub const RAI_F32: i32 = 5;
pub const RAI_F64: i32 = 6;
pub const RAI_OK: i32 = 0;
pub const RAI_ERR_BAD_DTYPE: i32 = -1;
pub const RAI_ERR_BAD_SHAPE: i32 = -2;
pub const RAI_ERR_BAD_STRIDE: i32 = -3;
pub const RAI_ERR_OOM: i32 = -4;
pub const RAI_ERR_HIP: i32 = -5;
pub const RAI_ERR_BAD_ARG: i32 = -6;
pub const RAI_ERR_UNSUPPORTED: i32 = -7;
pub const RAI_ERR_INDEX: i32 = -8;
pub const RAI_ERR_PARAM_NOT_FOUND: i32 = -9;
pub const RAI_ERR_IO: i32 = -10;
pub const RAI_UN_SIN: i32 = 0;
pub const RAI_UN_COS: i32 = 1;
pub const RAI_UN_NEG: i32 = 2;
pub const RAI_UN_SQUARE: i32 = 3;
pub const RAI_UN_SQRT: i32 = 4;
pub const RAI_UN_RSQRT: i32 = 5;
pub const RAI_UN_ABS: i32 = 6;
pub const RAI_UN_EXP: i32 = 7;
pub const RAI_UN_LOG: i32 = 8;
pub const RAI_UN_LOG2: i32 = 9;
pub const RAI_UN_LOG10: i32 = 10;
pub const RAI_UN_ERF: i32 = 11;
pub const RAI_UN_TANH: i32 = 12;
pub const RAI_UN_POWF: i32 = 13;
pub const RAI_UN_SIGN: i32 = 14;
pub const RAI_UN_GELU: i32 = 15;
pub const RAI_UN_NEW_GELU: i32 = 16;
pub const RAI_UN_SILU: i32 = 17;
pub const RAI_UN_RELU: i32 = 18;
pub const RAI_BIN_ADD: i32 = 0;
pub const RAI_BIN_SUB: i32 = 1;
pub const RAI_BIN_MUL: i32 = 2;
pub const RAI_BIN_DIV: i32 = 3;
pub const RAI_BIN_MAXIMUM: i32 = 4;
pub const RAI_BIN_MINIMUM: i32 = 5;
pub const RAI_BIN_EQ: i32 = 6;
pub const RAI_BIN_NE: i32 = 7;
pub const RAI_BIN_GT: i32 = 8;
pub const RAI_BIN_GE: i32 = 9;
pub const RAI_BIN_LT: i32 = 10;
pub const RAI_BIN_LE: i32 = 11;
pub const RAI_RED_SUM: i32 = 0;
pub const RAI_RED_MAX: i32 = 1;
pub const RAI_RED_MIN: i32 = 2;
pub const RAI_KV_E4M3: i32 = 0;
pub const RAI_KV_INT8: i32 = 1;
pub const RAI_ARCH_PHI2: i32 = 0;
pub const RAI_ARCH_QWEN2: i32 = 1;
pub const RAI_ARCH_GEMMA: i32 = 2;
pub const RAI_ARCH_PHI3: i32 = 3;
pub const RAI_ARCH_LELITAR: i32 = 4;
pub const RAI_ARCH_BEZADRA: i32 = 5;
pub const RAI_MLP_NONE: i32 = 0;
pub const RAI_MLP_DENSE: i32 = 1;
pub const RAI_MLP_MIXTURE: i32 = 2;
pub const RAI_MIXER_ATTENTION: i32 = 0;
pub const RAI_MIXER_CHANNEL_DELTA: i32 = 1;

/// Strided view over a device allocation (`rai_hip_tensor`).
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct RaiHipTensor {
    pub data: *mut c_void,
    pub dtype: i32,
    pub rank: i32,
    pub shape: [i64; RAI_HIP_MAX_RANK],
    pub stride: [i64; RAI_HIP_MAX_RANK],
    pub offset: i64,
}

/// `rai_hip_decoder_config`.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct RaiHipDecoderConfig {
    pub arch: i32,
    pub dtype: i32,
    pub vocab_size: i32,
    pub hidden_size: i32,
    pub intermediate_size: i32,
    pub num_hidden_layers: i32,
    pub num_attention_heads: i32,
    pub num_key_value_heads: i32,
    pub head_dim: i32,
    pub rotary_dim: i32,
    pub max_position_embeddings: i32,
    pub hidden_act: i32,
    pub tie_word_embeddings: i32,
    pub max_batch: i32,
    pub max_context: i32,
    pub rope_tables_f32: i32,
    pub qk_layernorm: i32,
    pub rope_theta: f64,
    pub norm_eps: f64,
}

/// `rai_hip_latent_layer`.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct RaiHipLatentLayer {
    pub heads: i32,
    pub qk_dim: i32,
    pub v_dim: i32,
    pub q_rank: i32,
    pub kv_rank: i32,
    pub window: i32,
    pub mlp_kind: i32,
    pub mlp_act: i32,
    pub intermediate: i32,
    pub experts: i32,
    pub top: i32,
    pub attn_scale: f64,
}

/// `rai_hip_latent_config`.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct RaiHipLatentConfig {
    pub dtype: i32,
    pub vocab_size: i32,
    pub width: i32,
    pub num_layers: i32,
    pub norm_groups: i32,
    pub max_batch: i32,
    pub max_context: i32,
    pub norm_eps: f64,
    pub residual_mult: f64,
}

/// `rai_hip_hybrid_layer`.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct RaiHipHybridLayer {
    pub mixer: i32,
    pub heads: i32,
    pub kv_heads: i32,
    pub qk_dim: i32,
    pub v_dim: i32,
    pub rot_dims: i32,
    pub conv_taps: i32,
    pub decay_rank: i32,
    pub gate_rank: i32,
    pub mlp_kind: i32,
    pub intermediate: i32,
    pub attn_scale: f64,
    pub softcap: f64,
    pub rot_base: f64,
    pub rot_factor: f64,
    pub rot_low: f64,
    pub rot_high: f64,
    pub rot_original: f64,
    pub mlp_limit: f64,
    pub mlp_alpha: f64,
}

/// `rai_hip_hybrid_config`.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct RaiHipHybridConfig {
    pub dtype: i32,
    pub vocab_size: i32,
    pub width: i32,
    pub num_layers: i32,
    pub loop_start: i32,
    pub loop_stop: i32,
    pub loop_times: i32,
    pub max_batch: i32,
    pub max_context: i32,
    pub norm_eps: f64,
    pub embed_scale: f64,
    pub logit_scale: f64,
}

/// Opaque decoder handle.
#[repr(C)]
pub struct RaiHipDecoder {
    _private: [u8; 0],
}

#[link(name = "rai_hip")]
extern "C" {
    pub fn rai_hip_last_error() -> *const c_char;
    pub fn rai_hip_device_count(count: *mut c_int) -> c_int;
    pub fn rai_hip_init(dev: c_int) -> c_int;
    pub fn rai_hip_sync(dev: c_int) -> c_int;
    pub fn rai_hip_alloc(dev: c_int, bytes: usize, out: *mut *mut c_void) -> c_int;
    pub fn rai_hip_retain(ptr: *mut c_void) -> c_int;
    pub fn rai_hip_release(ptr: *mut c_void) -> c_int;
    pub fn rai_hip_mem_stats(dev: c_int, in_use: *mut u64, pooled: *mut u64, n_device_mallocs: *mut u64) -> c_int;
    pub fn rai_hip_trim(dev: c_int) -> c_int;
    pub fn rai_hip_h2d(dev: c_int, dst_dev: *mut c_void, src_host: *const c_void, bytes: usize) -> c_int;
    pub fn rai_hip_d2h(dev: c_int, dst_host: *mut c_void, src_dev: *const c_void, bytes: usize) -> c_int;
    pub fn rai_hip_d2d(dev: c_int, dst_dev: *mut c_void, src_dev: *const c_void, bytes: usize) -> c_int;
    pub fn rai_hip_to_device(src_dev: c_int, input: *const RaiHipTensor, dst_dev: c_int, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_timer_create(dev: c_int, timer: *mut *mut c_void) -> c_int;
    pub fn rai_hip_timer_start(timer: *mut c_void) -> c_int;
    pub fn rai_hip_timer_stop(timer: *mut c_void) -> c_int;
    pub fn rai_hip_timer_elapsed_ms(timer: *mut c_void, ms: *mut f32) -> c_int;
    pub fn rai_hip_timer_destroy(timer: *mut c_void) -> c_int;
    pub fn rai_hip_fill(dev: c_int, out: *const RaiHipTensor, value: f64) -> c_int;
    pub fn rai_hip_arange(dev: c_int, out: *const RaiHipTensor, start: f64, step: f64) -> c_int;
    pub fn rai_hip_cast(dev: c_int, input: *const RaiHipTensor, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_copy(dev: c_int, input: *const RaiHipTensor, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_unary(dev: c_int, op: c_int, input: *const RaiHipTensor, out: *const RaiHipTensor, param: f64) -> c_int;
    pub fn rai_hip_binary(dev: c_int, op: c_int, lhs: *const RaiHipTensor, rhs: *const RaiHipTensor, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_where(dev: c_int, cond: *const RaiHipTensor, on_true: *const RaiHipTensor, on_false: *const RaiHipTensor, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_reduce(dev: c_int, op: c_int, input: *const RaiHipTensor, dims: *const i32, ndims: i32, keep_dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_softmax(dev: c_int, input: *const RaiHipTensor, dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_log_softmax(dev: c_int, input: *const RaiHipTensor, dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_argmax(dev: c_int, input: *const RaiHipTensor, dim: i32, keep_dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_argmin(dev: c_int, input: *const RaiHipTensor, dim: i32, keep_dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_argmax_static(dev: c_int, input: *const RaiHipTensor, dim: i32, keep_dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_index_select(dev: c_int, input: *const RaiHipTensor, index: *const RaiHipTensor, dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_gather(dev: c_int, x: *const RaiHipTensor, index: *const RaiHipTensor, dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_index_add(dev: c_int, x: *const RaiHipTensor, index: *const RaiHipTensor, source: *const RaiHipTensor, dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_scatter_add(dev: c_int, x: *const RaiHipTensor, index: *const RaiHipTensor, source: *const RaiHipTensor, dim: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_index_errors(dev: c_int, count: *mut u64) -> c_int;
    pub fn rai_hip_matmul(dev: c_int, a: *const RaiHipTensor, b: *const RaiHipTensor, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_linear(dev: c_int, x: *const RaiHipTensor, w: *const RaiHipTensor, bias: *const RaiHipTensor, act: i32, residual: *const RaiHipTensor, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_linear_packed(dev: c_int, x: *const RaiHipTensor, w: *const RaiHipTensor, bias: *const RaiHipTensor, bias2: *const RaiHipTensor, act: i32, act_from: i32, residual: *const RaiHipTensor, glu: i32, k_splits: i32, out1: *const RaiHipTensor, out2: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_layer_norm(dev: c_int, x: *const RaiHipTensor, w: *const RaiHipTensor, b: *const RaiHipTensor, eps: f64, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_rms_norm(dev: c_int, x: *const RaiHipTensor, w: *const RaiHipTensor, eps: f64, add_one: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_rope(dev: c_int, x: *const RaiHipTensor, cos: *const RaiHipTensor, sin: *const RaiHipTensor, rot_dim: i32, offset: i64, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_rope_tables(dev: c_int, theta: f64, rot_dim: i32, f64_powf: i32, cos: *const RaiHipTensor, sin: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_attention(dev: c_int, q: *const RaiHipTensor, k: *const RaiHipTensor, v: *const RaiHipTensor, scale: f64, causal: i32, f32_scores: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_kv_plan(dev: c_int, lens: *const RaiHipTensor, add: *const RaiHipTensor, free_pages: *const RaiHipTensor, taken: *const RaiHipTensor, tables: *const RaiHipTensor, page: i32, out_tables: *const RaiHipTensor, out_lens: *const RaiHipTensor, out_taken: *const RaiHipTensor, starts: *const RaiHipTensor, positions: *const RaiHipTensor, runs: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_rope_frequencies(dev: c_int, base: f64, factor: f64, low: f64, high: f64, original: f64, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_rope_positions(dev: c_int, x: *const RaiHipTensor, positions: *const RaiHipTensor, frequencies: *const RaiHipTensor, interleaved: i32, inverse: i32, magnitude: f64, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_kv_append(dev: c_int, new_k: *const RaiHipTensor, new_v: *const RaiHipTensor, runs: *const RaiHipTensor, format: i32, k: *const RaiHipTensor, v: *const RaiHipTensor, k_scale: *const RaiHipTensor, v_scale: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_kv_attention(dev: c_int, q: *const RaiHipTensor, tables: *const RaiHipTensor, starts: *const RaiHipTensor, lens: *const RaiHipTensor, format: i32, k: *const RaiHipTensor, v: *const RaiHipTensor, k_scale: *const RaiHipTensor, v_scale: *const RaiHipTensor, scale: f64, window: i32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_decoder_create(dev: c_int, cfg: *const RaiHipDecoderConfig, out: *mut *mut RaiHipDecoder) -> c_int;
    pub fn rai_hip_decoder_destroy(dec: *mut RaiHipDecoder) -> c_int;
    pub fn rai_hip_decoder_create_latent(dev: c_int, cfg: *const RaiHipLatentConfig, layers: *const RaiHipLatentLayer, out: *mut *mut RaiHipDecoder) -> c_int;
    pub fn rai_hip_decoder_create_hybrid(dev: c_int, cfg: *const RaiHipHybridConfig, layers: *const RaiHipHybridLayer, out: *mut *mut RaiHipDecoder) -> c_int;
    pub fn rai_hip_decoder_load_param(dec: *mut RaiHipDecoder, name: *const c_char, host_data: *const c_void, bytes: usize) -> c_int;
    pub fn rai_hip_decoder_load_safetensors(dec: *mut RaiHipDecoder, paths: *const *const c_char, n_paths: i32) -> c_int;
    pub fn rai_hip_safetensors_index_files(index_json_path: *const c_char, buf: *mut c_char, buflen: usize, n_files: *mut i32) -> c_int;
    pub fn rai_hip_decoder_dtype(dec: *mut RaiHipDecoder, dtype: *mut i32) -> c_int;
    pub fn rai_hip_decoder_param_count(dec: *mut RaiHipDecoder, count: *mut i32) -> c_int;
    pub fn rai_hip_decoder_param_name(dec: *mut RaiHipDecoder, i: i32, buf: *mut c_char, buflen: usize, numel: *mut i64) -> c_int;
    pub fn rai_hip_decoder_param_shape(dec: *mut RaiHipDecoder, i: i32, rows: *mut i64, cols: *mut i64) -> c_int;
    pub fn rai_hip_decoder_forward(dec: *mut RaiHipDecoder, ids_host: *const u32, batch: i32, seq: i32, logits_host: *mut f32, tokens_host: *mut u32) -> c_int;
    pub fn rai_hip_decoder_forward_hidden(dec: *mut RaiHipDecoder, ids_host: *const u32, hidden_in_host: *const c_void, batch: i32, seq: i32, hidden_out_host: *mut f32, logits_host: *mut f32, tokens_host: *mut u32) -> c_int;
    pub fn rai_hip_decoder_forward_rows(dec: *mut RaiHipDecoder, ids_host: *const u32, batch: i32, seq: i32, rows_host: *const i32, n_rows: i32, logits_host: *mut f32) -> c_int;
    pub fn rai_hip_decoder_generate(dec: *mut RaiHipDecoder, prompt_host: *const u32, batch: i32, prompt_len: i32, n_new: i32, tokens_host: *mut u32, prefill_ms: *mut f32, decode_ms: *mut f32) -> c_int;
    pub fn rai_hip_decoder_generate_sampled(dec: *mut RaiHipDecoder, prompt_host: *const u32, batch: i32, prompt_len: i32, n_new: i32, repeat_penalty: f32, repeat_last_n: i32, eos_token: i64, tokens_host: *mut u32, n_generated: *mut i32, prefill_ms: *mut f32, decode_ms: *mut f32) -> c_int;
    pub fn rai_hip_sample_argmax(dev: c_int, logits: *const RaiHipTensor, context: *const RaiHipTensor, repeat_penalty: f32, out: *const RaiHipTensor) -> c_int;
    pub fn rai_hip_decoder_clear_kv_cache(dec: *mut RaiHipDecoder) -> c_int;
    pub fn rai_hip_decoder_context_len(dec: *mut RaiHipDecoder, len: *mut i32) -> c_int;
    pub fn rai_hip_decoder_time_decode_step(dec: *mut RaiHipDecoder, sweeps: i32, us_per_launch: *mut f32, bytes_per_launch: *mut f64) -> c_int;
    pub fn rai_hip_decoder_time_decode_linear(dec: *mut RaiHipDecoder, sweeps: i32, us_per_launch: *mut f32, bytes_per_launch: *mut f64) -> c_int;
}

/// The candle backend `unwrap()`s every backend error (backend/candle.rs throughout); a non-zero status
/// panics with the library's message so the `Hip` device keeps that contract.
#[inline]
#[track_caller]
pub fn check(status: c_int) {
    if status != RAI_OK {
        let msg = unsafe { CStr::from_ptr(rai_hip_last_error()) }.to_string_lossy().into_owned();
        panic!("rai_hip status {status}: {msg}");
    }
}
