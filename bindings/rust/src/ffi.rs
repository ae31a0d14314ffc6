// GENERATED by bindings/rust/gen_ffi.py from include/paged_infer_cuda.h - do not edit.
#![allow(non_camel_case_types, dead_code)]

pub const PI_OK: i32 = 0;
pub const PI_ERR_INVALID_ARG: i32 = -1;
pub const PI_ERR_OOM: i32 = -2;
pub const PI_ERR_CUDA: i32 = -3;
pub const PI_ERR_NCCL: i32 = -4;
pub const PI_ERR_TIMEOUT: i32 = -5;
pub const PI_ERR_UNSUPPORTED: i32 = -6;
pub const PI_PROF_GEMV: i32 = 0;
pub const PI_PROF_GEMM_TC: i32 = 1;
pub const PI_PROF_ATTENTION: i32 = 2;
pub const PI_PROF_ROPE_KV: i32 = 3;
pub const PI_PROF_OTHER: i32 = 4;
pub const PI_PROF_COLLECTIVE: i32 = 5;
pub const PI_PROF_RECURRENCE: i32 = 6;
pub const PI_PROF_CLASSES: i32 = 7;
pub const PI_OPT_TENSOR_GEMM: i32 = 1;
pub const PI_OPT_CUDA_GRAPH: i32 = 2;
pub const PI_OPT_PDL: i32 = 3;
pub const PI_OPT_GEMV_MAX_M: i32 = 4;
pub const PI_OPT_ATTN_TMA: i32 = 5;
pub const PI_OPT_FUSE_PLANES: i32 = 6;
pub const PI_OPT_ATTN_SHARED: i32 = 7;
pub const PI_OPT_PEER_SPIN_LIMIT: i32 = 8;
pub const PI_OPT_TP_PUSH: i32 = 9;
pub const PI_OPT_ATTN_FLAT: i32 = 10;
pub const PI_OPT_KV8_WAIT_LIMIT: i32 = 11;
pub const PI_SPLIT_NONE: i32 = 0;
pub const PI_SPLIT_COLUMN: i32 = 1;
pub const PI_SPLIT_ROW: i32 = 2;
pub const PI_F32: i32 = 0;
pub const PI_INT8: i32 = 1;
pub const PI_BF16: i32 = 2;
pub const PI_F16: i32 = 3;
pub const PI_E4M3: i32 = 4;
pub const PI_MIXER_ATTENTION: i32 = 0;
pub const PI_MIXER_GLA: i32 = 1;
pub const PI_MIXER_MLSTM: i32 = 2;
pub const PI_MIXER_LATENT: i32 = 3;
pub const PI_MIXER_SSD: i32 = 4;
pub const PI_MIXER_LIGHTNING: i32 = 5;
pub const PI_MIXER_MINGRU: i32 = 6;
pub const PI_FF_GELU: i32 = 0;
pub const PI_FF_SILU: i32 = 1;
pub const PI_FF_EXPERTS: i32 = 2;
pub const PI_UNIT_CLAMPED: i32 = 0;
pub const PI_UNIT_SILU: i32 = 1;
pub const PI_UNIT_RELU2: i32 = 2;
pub const PI_SCORE_SIGMOID: i32 = 0;
pub const PI_SCORE_SOFTMAX: i32 = 1;
pub const PI_SCORE_CHOSEN: i32 = 2;
pub const PI_NORM_DYT: i32 = 0;
pub const PI_NORM_LAYER: i32 = 1;
pub const PI_NORM_RMS: i32 = 2;
pub const PI_NORM_SUM: i32 = 3;
pub const PI_TP_PEER_HANDLE_BYTES: i32 = 64;

#[repr(C)] pub struct PiCtx { _private: [u8; 0] }
#[repr(C)] pub struct PiLinear { _private: [u8; 0] }
#[repr(C)] pub struct PiKvPool { _private: [u8; 0] }
#[repr(C)] pub struct PiModel { _private: [u8; 0] }
#[repr(C)] pub struct PiStatePool { _private: [u8; 0] }
#[repr(C)] pub struct PiKv8Pool { _private: [u8; 0] }

#[repr(C)]
#[derive(Clone, Copy)]
pub struct PiKvLayout {
    pub num_layers: i32,
    pub num_blocks: i32,
    pub block_size: i32,
    pub num_kv_heads: i32,
    pub head_dim: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct PiModelConfig {
    pub hidden_size: i32,
    pub num_hidden_layers: i32,
    pub num_attention_heads: i32,
    pub num_key_value_heads: i32,
    pub intermediate_size: i32,
    pub vocab_size: i32,
    pub rms_norm_eps: f32,
    pub rope_theta: f32,
    pub attention_window: i32,
    pub rope_style: i32,
    pub max_batch: i32,
    pub max_positions: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct PiTensor {
    pub kind: i32,
    pub quantize_on_load: i32,
    pub rows: i64,
    pub cols: i64,
    pub data: *const std::ffi::c_void,
    pub scales: *const f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct PiModelWeights {
    pub token_embeddings_bf16: *const u16,
    pub final_norm: *const f32,
    pub attention_norm: *mut *const f32,
    pub ffn_norm: *mut *const f32,
    pub projections: *const PiTensor,
    pub lm_head: PiTensor,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct PiLayerConfig {
    pub mixer: i32,
    pub heads: i32,
    pub kv_heads: i32,
    pub dim: i32,
    pub vdim: i32,
    pub maps: i32,
    pub window: i32,
    pub rot_dims: i32,
    pub rot_base: f32,
    pub scale: f32,
    pub diff: f32,
    pub tau: f32,
    pub gate_cap: f32,
    pub ff: i32,
    pub ff_kind: i32,
    pub rank: i32,
    pub rot_factor: f64,
    pub rot_original: f64,
    pub rot_fast: f64,
    pub rot_slow: f64,
    pub groups: i32,
    pub norm_groups: i32,
    pub conv: i32,
    pub experts: i32,
    pub top: i32,
    pub expert_groups: i32,
    pub keep_groups: i32,
    pub shared_ff: i32,
    pub limit: f32,
    pub shared_limit: f32,
    pub biases: i32,
    pub unit_qk: i32,
    pub distance_bias: i32,
    pub sink: i32,
    pub head_gate: i32,
    pub v_mix: i32,
    pub q_temp_coef: f64,
    pub q_temp_every: f64,
    pub decay: *const f64,
    pub unit: i32,
    pub score: i32,
    pub group_best: i32,
    pub renorm: i32,
    pub shared_gate: i32,
    pub route_scale: f32,
    pub router_bias: i32,
    pub rot_banded: i32,
    pub norm_qk: i32,
    pub sigmoid_weights: i32,
    pub kv_from: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct PiLayeredConfig {
    pub width: i32,
    pub vocab_size: i32,
    pub num_layers: i32,
    pub norm_eps: f32,
    pub compute: i32,
    pub max_rows: i32,
    pub norm: i32,
    pub tied: i32,
    pub logit_scale: f32,
    pub embed_scale: f32,
    pub residual_mult: f32,
    pub side_dim: i32,
    pub residual_keep: f32,
    pub sublayer_gate: i32,
    pub pair_buckets: i32,
    pub pair_prev: i32,
    pub pair_cur: i32,
    pub layers: *const PiLayerConfig,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct PiNamedTensor {
    pub name: *const std::ffi::c_char,
    pub kind: i32,
    pub rows: i64,
    pub cols: i64,
    pub data: *const std::ffi::c_void,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct PiStepBatch {
    pub n_seqs: i32,
    pub tokens: *const u32,
    pub n_tokens: *const i32,
    pub start_pos: *const i32,
    pub block_tables: *const i32,
    pub max_blocks: i32,
    pub table_lens: *const i32,
    pub state_slots: *const i32,
    pub n_out: i32,
    pub out_rows: *const i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct PiStepArrays {
    pub block_size: i32,
    pub max_seqs: i32,
    pub max_blocks: i32,
    pub max_rows: i32,
    pub tables: *mut i32,
    pub lens: *mut i32,
    pub cu_rows: *mut i32,
    pub row_seq: *mut i32,
    pub row_pos: *mut i32,
    pub slots: *mut i64,
    pub counts: *mut i32,
}

extern "C" {
    pub fn pi_version() -> *const std::ffi::c_char;
    pub fn pi_last_error(ctx: *const PiCtx) -> *const std::ffi::c_char;
    pub fn pi_ctx_create(device: i32, stream: *mut std::ffi::c_void, out: *mut *mut PiCtx) -> i32;
    pub fn pi_nccl_unique_id(out_128_bytes: *mut std::ffi::c_void) -> i32;
    pub fn pi_ctx_create_tp(device: i32, stream: *mut std::ffi::c_void, rank: i32, tp: i32, nccl_unique_id: *const std::ffi::c_void, out: *mut *mut PiCtx) -> i32;
    pub fn pi_tp_peer_export(ctx: *mut PiCtx, max_floats: usize, handle_out_64_bytes: *mut std::ffi::c_void) -> i32;
    pub fn pi_tp_peer_import(ctx: *mut PiCtx, handles_tp_times_64_bytes: *const std::ffi::c_void) -> i32;
    pub fn pi_tp_peer_base(ctx: *const PiCtx) -> *mut std::ffi::c_void;
    pub fn pi_tp_peer_import_pointers(ctx: *mut PiCtx, bases_tp: *mut *const std::ffi::c_void) -> i32;
    pub fn pi_tp_exchange_add(ctx: *mut PiCtx, partial_dev: *const f32, x_dev: *mut f32, rows: i32, cols: i32) -> i32;
    pub fn pi_ctx_destroy(ctx: *mut PiCtx);
    pub fn pi_ctx_synchronize(ctx: *mut PiCtx) -> i32;
    pub fn pi_ctx_kernel_launches(ctx: *const PiCtx) -> u64;
    pub fn pi_ctx_reset_kernel_launches(ctx: *mut PiCtx);
    pub fn pi_ctx_profile_begin(ctx: *mut PiCtx) -> i32;
    pub fn pi_ctx_profile_end(ctx: *mut PiCtx, ms_out: *mut f64, launches_out: *mut u64) -> i32;
    pub fn pi_ctx_set_option(ctx: *mut PiCtx, option: i32, value: i32) -> i32;
    pub fn pi_quantize_rows_i8(ctx: *mut PiCtx, w_host: *const f32, rows: usize, cols: usize, q_host_out: *mut i8, scales_host_out: *mut f32) -> i32;
    pub fn pi_quantize_rows_i8_dev(ctx: *mut PiCtx, w_dev: *const f32, rows: usize, cols: usize, q_dev_out: *mut i8, scales_dev_out: *mut f32) -> i32;
    pub fn pi_linear_create_i8(ctx: *mut PiCtx, rows: usize, cols: usize, q_host: *const i8, scales_host: *const f32, split: i32, out: *mut *mut PiLinear) -> i32;
    pub fn pi_linear_create_quantized(ctx: *mut PiCtx, rows: usize, cols: usize, w_host: *const f32, split: i32, out: *mut *mut PiLinear) -> i32;
    pub fn pi_linear_create_bf16(ctx: *mut PiCtx, rows: usize, cols: usize, w_bf16_host: *const u16, split: i32, out: *mut *mut PiLinear) -> i32;
    pub fn pi_linear_create_f32(ctx: *mut PiCtx, rows: usize, cols: usize, w_host: *const f32, split: i32, out: *mut *mut PiLinear) -> i32;
    pub fn pi_linear_destroy(lin: *mut PiLinear);
    pub fn pi_linear_rows(lin: *const PiLinear) -> usize;
    pub fn pi_linear_cols(lin: *const PiLinear) -> usize;
    pub fn pi_linear_weight_bytes(lin: *const PiLinear) -> usize;
    pub fn pi_linear_kind(lin: *const PiLinear) -> i32;
    pub fn pi_linear_read_i8(ctx: *mut PiCtx, lin: *const PiLinear, q_host_out: *mut i8, scales_host_out: *mut f32) -> i32;
    pub fn pi_linear_apply(ctx: *mut PiCtx, lin: *const PiLinear, x_dev: *const f32, out_dev: *mut f32, M: i32) -> i32;
    pub fn pi_linear_apply_host(ctx: *mut PiCtx, lin: *const PiLinear, x_host: *const f32, out_host: *mut f32, M: i32) -> i32;
    pub fn pi_linear_apply_noalloc(ctx: *mut PiCtx, lin: *const PiLinear, x_dev: *const f32, out_dev: *mut f32, M: i32) -> i32;
    pub fn pi_linear_apply_bf16(ctx: *mut PiCtx, lin: *const PiLinear, x_dev: *const u16, x_stride: usize, out_dev: *mut f32, M: i32) -> i32;
    pub fn pi_kv_pool_create(ctx: *mut PiCtx, layout: *const PiKvLayout, out: *mut *mut PiKvPool) -> i32;
    pub fn pi_kv_pool_destroy(pool: *mut PiKvPool);
    pub fn pi_kv_pool_bytes(pool: *const PiKvPool) -> usize;
    pub fn pi_kv_copy_block(ctx: *mut PiCtx, pool: *mut PiKvPool, src: i32, dst: i32) -> i32;
    pub fn pi_kv_upload(ctx: *mut PiCtx, pool: *mut PiKvPool, cache_host: *const f32) -> i32;
    pub fn pi_kv_download(ctx: *mut PiCtx, pool: *const PiKvPool, cache_host_out: *mut f32) -> i32;
    pub fn pi_kv_write_token(ctx: *mut PiCtx, pool: *mut PiKvPool, layer: i32, block: i32, tok: i32, k_host: *const f32, v_host: *const f32) -> i32;
    pub fn pi_kv_read_token(ctx: *mut PiCtx, pool: *const PiKvPool, layer: i32, block: i32, tok: i32, k_host_out: *mut f32, v_host_out: *mut f32) -> i32;
    pub fn pi_paged_attention(ctx: *mut PiCtx, pool: *const PiKvPool, layer: i32, num_heads: i32, q_dev: *const f32, q_stride: usize, out_dev: *mut f32, out_stride: usize, block_tables_host: *const i32, max_blocks: i32, table_lens_host: *const i32, pos_host: *const i32, start_host: *const i32, B: i32) -> i32;
    pub fn pi_paged_attention_host(ctx: *mut PiCtx, pool: *const PiKvPool, layer: i32, num_heads: i32, q_host: *const f32, out_host: *mut f32, block_tables_host: *const i32, max_blocks: i32, table_lens_host: *const i32, pos_host: *const i32, start_host: *const i32, B: i32) -> i32;
    pub fn pi_rms_norm_host(ctx: *mut PiCtx, x_host_inout: *mut f32, weight_host: *const f32, rows: i32, n: i32, eps: f32) -> i32;
    pub fn pi_rope_host(ctx: *mut PiCtx, x_host_inout: *mut f32, pos_host: *const i32, rows: i32, heads: i32, head_dim: i32, theta: f32, style: i32) -> i32;
    pub fn pi_swiglu_host(ctx: *mut PiCtx, gate_host_inout: *mut f32, up_host: *const f32, n: usize) -> i32;
    pub fn pi_argmax_host(ctx: *mut PiCtx, logits_host: *const f32, rows: i32, n: i32, out_host: *mut u32) -> i32;
    pub fn pi_model_create(ctx: *mut PiCtx, cfg: *const PiModelConfig, weights: *const PiModelWeights, out: *mut *mut PiModel) -> i32;
    pub fn pi_model_create_synthetic(ctx: *mut PiCtx, cfg: *const PiModelConfig, seed: u64, std: f32, quant: i32, lm_head_kind: i32, out: *mut *mut PiModel) -> i32;
    pub fn pi_model_destroy(model: *mut PiModel);
    pub fn pi_model_weight_bytes(model: *const PiModel) -> usize;
    pub fn pi_model_max_batch(model: *const PiModel) -> i32;
    pub fn pi_model_decode_batch(ctx: *mut PiCtx, model: *mut PiModel, pool: *mut PiKvPool, tokens_host: *const u32, positions_host: *const i32, block_tables_host: *const i32, max_blocks: i32, table_lens_host: *const i32, B: i32, logits_host_or_null: *mut f32, argmax_host_or_null: *mut u32) -> i32;
    pub fn pi_model_decode_batch_rows(ctx: *mut PiCtx, model: *mut PiModel, pool: *mut PiKvPool, tokens_host: *const u32, positions_host: *const i32, block_tables_host: *const i32, max_blocks: i32, table_lens_host: *const i32, B: i32, logit_rows_host: *const i32, n_logit_rows: i32, logits_host: *mut f32, argmax_host: *mut u32) -> i32;
    pub fn pi_model_prefill(ctx: *mut PiCtx, model: *mut PiModel, pool: *mut PiKvPool, tokens_host: *const u32, n: i32, start_pos: i32, block_table_host: *const i32, table_len: i32, chunk: i32, last_logits_host_or_null: *mut f32, argmax_host_or_null: *mut u32) -> i32;
    pub fn pi_model_decode_multi(ctx: *mut PiCtx, model: *mut PiModel, pool: *mut PiKvPool, tokens_host: *const u32, positions_host: *const i32, block_tables_host: *const i32, max_blocks: i32, table_lens_host: *const i32, B: i32, n_steps: i32, out_tokens_host: *mut u32) -> i32;
    pub fn pi_kv_fill_normal(ctx: *mut PiCtx, pool: *mut PiKvPool, seed: u64, std: f32) -> i32;
    pub fn pi_model_create_layered(ctx: *mut PiCtx, cfg: *const PiLayeredConfig, tensors: *const PiNamedTensor, n_tensors: i32, out: *mut *mut PiModel) -> i32;
    pub fn pi_model_create_layered_synthetic(ctx: *mut PiCtx, cfg: *const PiLayeredConfig, gla_rank: i32, seed: u64, std: f32, out: *mut *mut PiModel) -> i32;
    pub fn pi_model_vocab_size(model: *const PiModel) -> i32;
    pub fn pi_model_state_bytes(model: *const PiModel) -> usize;
    pub fn pi_kv_pool_create_for_model(ctx: *mut PiCtx, model: *const PiModel, num_blocks: i32, block_size: i32, out: *mut *mut PiKvPool) -> i32;
    pub fn pi_state_pool_create(ctx: *mut PiCtx, model: *const PiModel, num_slots: i32, out: *mut *mut PiStatePool) -> i32;
    pub fn pi_state_pool_destroy(pool: *mut PiStatePool);
    pub fn pi_state_pool_bytes(pool: *const PiStatePool) -> usize;
    pub fn pi_state_copy_slot(ctx: *mut PiCtx, pool: *mut PiStatePool, src: i32, dst: i32) -> i32;
    pub fn pi_model_step(ctx: *mut PiCtx, model: *mut PiModel, pool: *mut PiKvPool, state_or_null: *mut PiStatePool, batch: *const PiStepBatch, logits_host_or_null: *mut f32, argmax_host_or_null: *mut u32) -> i32;
    pub fn pi_model_step_multi(ctx: *mut PiCtx, model: *mut PiModel, pool: *mut PiKvPool, state_or_null: *mut PiStatePool, batch: *const PiStepBatch, n_steps: i32, out_tokens_host: *mut u32) -> i32;
    pub fn pi_model_trace_layers(ctx: *mut PiCtx, model: *mut PiModel, on: i32) -> i32;
    pub fn pi_model_read_layer(ctx: *mut PiCtx, model: *const PiModel, layer: i32, rows: i32, x_host_out: *mut f32) -> i32;
    pub fn pi_step_plan(ctx: *mut PiCtx, arrays: *const PiStepArrays, start_dev: *const i32, n_tokens_dev: *const i32, n_seqs: i32, free_dev: *const i32, n_free: i32) -> i32;
    pub fn pi_kv8_pool_create(ctx: *mut PiCtx, layout: *const PiKvLayout, kind: i32, codes_dev_or_null: *mut std::ffi::c_void, scales_dev_or_null: *mut f32, out: *mut *mut PiKv8Pool) -> i32;
    pub fn pi_kv8_pool_destroy(pool: *mut PiKv8Pool);
    pub fn pi_kv8_pool_bytes(pool: *const PiKv8Pool) -> usize;
    pub fn pi_kv8_pool_pitch(pool: *const PiKv8Pool) -> i32;
    pub fn pi_kv8_copy_block(ctx: *mut PiCtx, pool: *mut PiKv8Pool, src: i32, dst: i32) -> i32;
    pub fn pi_kv8_read_token(ctx: *mut PiCtx, pool: *const PiKv8Pool, layer: i32, block: i32, tok: i32, k_host_out: *mut f32, v_host_out: *mut f32) -> i32;
    pub fn pi_kv8_write(ctx: *mut PiCtx, pool: *mut PiKv8Pool, layer: i32, dtype: i32, k_dev: *const std::ffi::c_void, k_stride: usize, v_dev: *const std::ffi::c_void, v_stride: usize, slots_dev: *const i64, n_rows: i32) -> i32;
    pub fn pi_kv8_attention(ctx: *mut PiCtx, pool: *const PiKv8Pool, layer: i32, num_heads: i32, dtype: i32, q_dev: *const std::ffi::c_void, q_stride: usize, out_dev: *mut std::ffi::c_void, out_stride: usize, arrays: *const PiStepArrays, n_seqs: i32, n_rows: i32, max_seq_rows: i32, max_context: i32, window: i32, scale: f32) -> i32;
    pub fn pi_sample(ctx: *mut PiCtx, logits_dev: *const std::ffi::c_void, dtype: i32, row_stride: usize, rows: i32, n: i32, temperature_dev: *const f32, top_k_dev: *const i32, top_p_dev: *const f32, min_p_dev: *const f32, u_dev: *const f32, ids_dev: *mut i32, probs_dev_or_null: *mut f32) -> i32;
}
