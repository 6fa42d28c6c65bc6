// GENERATED by rust/gen_ffi.py from include/tlcuda.h -- do not edit.
//
// The C ABI of libtlcuda: what takes the place of the MetalDevice / MetalBuffer /
// KernelExecutor calls of src/device/ in the TensorLogic crate.  Every function returns
// a status (0 = ok, negative = the TensorError variant named in TlcStatus below);
// tlc_last_error() gives the message of the last failure on the calling thread.
#![allow(non_camel_case_types, dead_code)]
use std::os::raw::{c_char, c_void};

#[repr(C)]
pub struct TlcBuf { _private: [u8; 0] }
#[repr(C)]
pub struct TlcComm { _private: [u8; 0] }
#[repr(C)]
pub struct TlcCtx { _private: [u8; 0] }
#[repr(C)]
pub struct TlcGguf { _private: [u8; 0] }
#[repr(C)]
pub struct TlcKvCache { _private: [u8; 0] }
#[repr(C)]
pub struct TlcKvCache8 { _private: [u8; 0] }
#[repr(C)]
pub struct TlcLlama { _private: [u8; 0] }
#[repr(C)]
pub struct TlcModel { _private: [u8; 0] }
#[repr(C)]
pub struct TlcQTensor { _private: [u8; 0] }
#[repr(C)]
pub struct TlcWeightCache { _private: [u8; 0] }

#[repr(C)]
#[derive(Clone, Copy, Debug, Default)]
pub struct TlcPoolStats {
    pub total_pooled: u64,
    pub size_classes: u64,
    pub total_memory: u64,
    pub reuse_count: u64,
    pub allocation_count: u64,
    pub eviction_count: u64,
    pub live_bytes: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug, Default)]
pub struct TlcLlamaConfig {
    pub n_layers: i32,
    pub d_model: i32,
    pub n_heads: i32,
    pub n_kv_heads: i32,
    pub head_dim: i32,
    pub ffn_dim: i32,
    pub vocab: i32,
    pub rms_eps: f32,
    pub rope_base: u32,
    pub max_seq: i32,
    pub max_batch: i32,
    pub max_prefill: i32,
    pub tp_rank: i32,
    pub tp_size: i32,
    pub logits_all_rows: i32,
    pub no_graph: i32,
}

pub const TLC_OK: i32 = 0;
pub const TLC_ERR_SHAPE_MISMATCH: i32 = -1;
pub const TLC_ERR_INVALID_OPERATION: i32 = -2;
pub const TLC_ERR_DEVICE: i32 = -3;
pub const TLC_ERR_CUDA: i32 = -4;
pub const TLC_ERR_ALLOCATION: i32 = -5;
pub const TLC_ERR_LOAD: i32 = -6;
pub const TLC_ERR_BUFFER_EXHAUSTED: i32 = -7;
pub const TLC_ERR_INDEX: i32 = -8;
pub const TLC_ERR_INVALID_DIMENSION: i32 = -9;
pub const TLC_ERR_TIMEOUT: i32 = -10;
pub const TLC_ERR_COMM: i32 = -11;
pub const TLC_SPLIT_NONE: i32 = 0;
pub const TLC_SPLIT_ROWS: i32 = 1;
pub const TLC_SPLIT_COLS: i32 = 2;

#[link(name = "tlcuda")]
extern "C" {
    pub fn tlc_last_error() -> *const c_char;
    pub fn tlc_version() -> *const c_char;
    pub fn tlc_init(ordinal: i32, out: *mut *mut TlcCtx) -> i32;
    pub fn tlc_destroy(ctx: *mut TlcCtx) -> i32;
    pub fn tlc_set_option(ctx: *mut TlcCtx, name: *const c_char, value: i64) -> i32;
    pub fn tlc_selftest_wait_timeout(ctx: *mut TlcCtx, kind: i32) -> i32;
    pub fn tlc_device_name(ctx: *mut TlcCtx, buf: *mut c_char, buflen: usize) -> i32;
    pub fn tlc_mem_info(ctx: *mut TlcCtx, free_bytes: *mut usize, total_bytes: *mut usize) -> i32;
    pub fn tlc_sm_count(ctx: *mut TlcCtx, out: *mut i32) -> i32;
    pub fn tlc_synchronize(ctx: *mut TlcCtx) -> i32;
    pub fn tlc_stream(ctx: *mut TlcCtx) -> *mut c_void;
    pub fn tlc_launch_count(ctx: *mut TlcCtx) -> u64;
    pub fn tlc_perf_report(ctx: *mut TlcCtx, buf: *mut c_char, buflen: usize, reset: i32,
                           needed_out: *mut usize) -> i32;
    pub fn tlc_alloc(ctx: *mut TlcCtx, bytes: usize, out: *mut *mut TlcBuf) -> i32;
    pub fn tlc_alloc_ptr(ctx: *mut TlcCtx, bytes: usize, out: *mut *mut c_void) -> i32;
    pub fn tlc_free(buf: *mut TlcBuf) -> i32;
    pub fn tlc_buf_ptr(buf: *mut TlcBuf) -> *mut c_void;
    pub fn tlc_buf_size(buf: *mut TlcBuf) -> usize;
    pub fn tlc_pool_stats_get(ctx: *mut TlcCtx, out: *mut TlcPoolStats) -> i32;
    pub fn tlc_pool_trim(ctx: *mut TlcCtx, max_idle_bytes: usize) -> i32;
    pub fn tlc_upload(ctx: *mut TlcCtx, dst_dev: *mut c_void, src_host: *const c_void, bytes: usize) -> i32;
    pub fn tlc_download(ctx: *mut TlcCtx, dst_host: *mut c_void, src_dev: *const c_void, bytes: usize) -> i32;
    pub fn tlc_host_alloc(bytes: usize, out: *mut *mut c_void) -> i32;
    pub fn tlc_host_free(p: *mut c_void) -> i32;
    pub fn tlc_qtensor_create(ctx: *mut TlcCtx, ty: i32, n_rows: i64, n_cols: i64, blocks: *const c_void,
                              bytes: usize, tp_rank: i32, tp_size: i32, split: i32,
                              out: *mut *mut TlcQTensor) -> i32;
    pub fn tlc_qtensor_create_synthetic(ctx: *mut TlcCtx, ty: i32, n_rows: i64, n_cols: i64, seed: u64,
                                        tensor_id: u64, scale_log2: i32, tp_rank: i32, tp_size: i32,
                                        split: i32, out: *mut *mut TlcQTensor) -> i32;
    pub fn tlc_synth_blocks_host(ty: i32, seed: u64, tensor_id: u64, scale_log2: i32, first_block: i64,
                                 n_blocks: i64, out_host: *mut c_void) -> i32;
    pub fn tlc_fill_normal_f16(ctx: *mut TlcCtx, dst_dev: *mut c_void, n: usize, seed: u64, tensor_id: u64,
                               mean: f32, std: f32) -> i32;
    pub fn tlc_qtensor_create_normal_f16(ctx: *mut TlcCtx, n_rows: i64, n_cols: i64, seed: u64,
                                         tensor_id: u64, mean: f32, std: f32, out: *mut *mut TlcQTensor) -> i32;
    pub fn tlc_qtensor_destroy(qt: *mut TlcQTensor) -> i32;
    pub fn tlc_qtensor_info(qt: *mut TlcQTensor, ty: *mut i32, n_rows: *mut i64, n_cols: *mut i64,
                            row_pitch: *mut usize, dev_ptr: *mut *const c_void) -> i32;
    pub fn tlc_qtensor_blocks(ctx: *mut TlcCtx, qt: *mut TlcQTensor, out_dev: *mut c_void) -> i32;
    pub fn tlc_tiled_bytes(ty: i32, n_rows: i64, n_cols: i64) -> usize;
    pub fn tlc_tile_blocks_host(ty: i32, n_rows: i64, n_cols: i64, blocks: *const c_void,
                                tiles_out: *mut c_void) -> i32;
    pub fn tlc_dequant(ctx: *mut TlcCtx, qt: *mut TlcQTensor, out_f16_dev: *mut c_void) -> i32;
    pub fn tlc_matmul(ctx: *mut TlcCtx, a_dev: *const c_void, b_dev: *const c_void, y_dev: *mut c_void,
                      m: i32, k: i32, k2: i32, n: i32) -> i32;
    pub fn tlc_linear(ctx: *mut TlcCtx, w: *mut TlcQTensor, x_dev: *const c_void, m: i32, x_cols: i64,
                      y_dev: *mut c_void, bias_dev: *const c_void) -> i32;
    pub fn tlc_linear_host(ctx: *mut TlcCtx, w: *mut TlcQTensor, x_host: *const c_void, m: i32,
                           x_cols: i64, y_host: *mut c_void, bias_host: *const c_void) -> i32;
    pub fn tlc_rms_norm(ctx: *mut TlcCtx, x_dev: *const c_void, w_dev: *const c_void, y_dev: *mut c_void,
                        rows: i32, d: i32, eps: f32) -> i32;
    pub fn tlc_rope(ctx: *mut TlcCtx, x_dev: *const c_void, y_dev: *mut c_void, seq: i32, heads: i32,
                    d: i32, pos_offset: i32, base: u32, positions_dev: *const i32) -> i32;
    pub fn tlc_rope_table(ctx: *mut TlcCtx, x_dev: *const c_void, cos_dev: *const c_void,
                          sin_dev: *const c_void, y_dev: *mut c_void, seq: i32, heads: i32, head_dim: i32,
                          table_rows: i32, pitch: i32) -> i32;
    pub fn tlc_sigmoid(ctx: *mut TlcCtx, x_dev: *const c_void, y_dev: *mut c_void, n: usize) -> i32;
    pub fn tlc_mul(ctx: *mut TlcCtx, a_dev: *const c_void, b_dev: *const c_void, y_dev: *mut c_void,
                   n: usize) -> i32;
    pub fn tlc_add(ctx: *mut TlcCtx, a_dev: *const c_void, b_dev: *const c_void, y_dev: *mut c_void,
                   n: usize) -> i32;
    pub fn tlc_swiglu(ctx: *mut TlcCtx, gate_dev: *const c_void, up_dev: *const c_void, y_dev: *mut c_void,
                      n: usize) -> i32;
    pub fn tlc_softmax(ctx: *mut TlcCtx, x_dev: *const c_void, y_dev: *mut c_void, rows: i32, last_dim: i32) -> i32;
    pub fn tlc_embedding(ctx: *mut TlcCtx, table_dev: *const c_void, vocab: i32, d: i32,
                         ids_host: *const i32, m: i32, y_dev: *mut c_void) -> i32;
    pub fn tlc_norm_linear_multi(ctx: *mut TlcCtx, n_weights: i32, w: *const *mut TlcQTensor,
                                 y_dev: *const *mut c_void, rope_heads: *const i32, x_dev: *const c_void,
                                 m: i32, norm_w_dev: *const c_void, eps: f32, pos_offset: i32,
                                 rope_base: u32, positions_dev: *const i32) -> i32;
    pub fn tlc_swiglu_gate_up(ctx: *mut TlcCtx, w_gate: *mut TlcQTensor, w_up: *mut TlcQTensor,
                              x_dev: *const c_void, m: i32, norm_w_dev: *const c_void, eps: f32,
                              act_dev: *mut c_void) -> i32;
    pub fn tlc_linear_residual(ctx: *mut TlcCtx, w: *mut TlcQTensor, x_dev: *const c_void, m: i32,
                               residual_dev: *const c_void, y_dev: *mut c_void) -> i32;
    pub fn tlc_kvcache_create(ctx: *mut TlcCtx, n_layers: i32, max_batch: i32, max_seq: i32,
                              n_kv_heads: i32, head_dim: i32, out: *mut *mut TlcKvCache) -> i32;
    pub fn tlc_kvcache_destroy(cache: *mut TlcKvCache) -> i32;
    pub fn tlc_kvcache_layer_ptrs(cache: *mut TlcKvCache, layer: i32, k_dev: *mut *mut c_void,
                                  v_dev: *mut *mut c_void) -> i32;
    pub fn tlc_kvcache_append(ctx: *mut TlcCtx, cache: *mut TlcKvCache, layer: i32, k_dev: *const c_void,
                              v_dev: *const c_void, m: i32, pos_offset: i32, positions_dev: *const i32) -> i32;
    pub fn tlc_attention(ctx: *mut TlcCtx, cache: *mut TlcKvCache, layer: i32, q_dev: *const c_void,
                         out_dev: *mut c_void, batch: i32, n_queries: i32, n_heads: i32, q_pos0: i32,
                         positions_dev: *const i32, max_keys: i32, scale: f32) -> i32;
    pub fn tlc_attention_decode_static(stream: *mut c_void, q_dev: *const c_void,
                                       k_cache_dev: *const c_void, v_cache_dev: *const c_void,
                                       out_dev: *mut c_void, batch: i32, n_heads: i32, n_kv_heads: i32,
                                       head_dim: i32, max_seq: i32, positions_dev: *const i32,
                                       max_keys: i32, scale: f32) -> i32;
    pub fn tlc_attention_decode_static_status(stream: *mut c_void, clamped_out: *mut i32) -> i32;
    pub fn tlc_kvcache8_create(ctx: *mut TlcCtx, n_layers: i32, max_batch: i32, max_seq: i32,
                               n_kv_heads: i32, head_dim: i32, out: *mut *mut TlcKvCache8) -> i32;
    pub fn tlc_kvcache8_destroy(cache: *mut TlcKvCache8) -> i32;
    pub fn tlc_kvcache8_append(ctx: *mut TlcCtx, cache: *mut TlcKvCache8, layer: i32, k_dev: *const c_void,
                               v_dev: *const c_void, m: i32, sequence: i32, pos_offset: i32,
                               positions_dev: *const i32) -> i32;
    pub fn tlc_kvcache8_rows(ctx: *mut TlcCtx, cache: *mut TlcKvCache8, layer: i32, sequence: i32,
                             n_sequences: i32, first: i32, n: i32, k_out_dev: *mut c_void,
                             v_out_dev: *mut c_void) -> i32;
    pub fn tlc_attention8(ctx: *mut TlcCtx, cache: *mut TlcKvCache8, layer: i32, q_dev: *const c_void,
                          out_dev: *mut c_void, batch: i32, n_queries: i32, n_heads: i32, sequence: i32,
                          q_pos0: i32, positions_dev: *const i32, max_keys: i32, scale: f32) -> i32;
    pub fn tlc_model_load_gguf(ctx: *mut TlcCtx, path: *const c_char, tp_rank: i32, tp_size: i32,
                               out: *mut *mut TlcModel) -> i32;
    pub fn tlc_weight_cache_open(ctx: *mut TlcCtx, path: *const c_char, capacity: i64,
                                 out: *mut *mut TlcWeightCache) -> i32;
    pub fn tlc_weight_cache_close(cache: *mut TlcWeightCache) -> i32;
    pub fn tlc_weight_cache_get(cache: *mut TlcWeightCache, name: *const c_char, out: *mut *mut TlcQTensor) -> i32;
    pub fn tlc_weight_cache_contains(cache: *mut TlcWeightCache, name: *const c_char) -> i32;
    pub fn tlc_weight_cache_clear(cache: *mut TlcWeightCache) -> i32;
    pub fn tlc_weight_cache_stats(cache: *mut TlcWeightCache, len: *mut i64, capacity: *mut i64,
                                  hits: *mut u64, misses: *mut u64, evictions: *mut u64) -> i32;
    pub fn tlc_gguf_open(path: *const c_char, out: *mut *mut TlcGguf) -> i32;
    pub fn tlc_gguf_close(g: *mut TlcGguf) -> i32;
    pub fn tlc_gguf_tensor_count(g: *mut TlcGguf) -> i32;
    pub fn tlc_gguf_tensor_info(g: *mut TlcGguf, index: i32, name: *mut *const c_char, ty: *mut i32,
                                rows: *mut i64, cols: *mut i64, file_offset: *mut u64, nbytes: *mut u64) -> i32;
    pub fn tlc_gguf_meta_num(g: *mut TlcGguf, key: *const c_char, out: *mut f64) -> i32;
    pub fn tlc_gguf_meta_str(g: *mut TlcGguf, key: *const c_char) -> *const c_char;
    pub fn tlc_gguf_data_start(g: *mut TlcGguf) -> u64;
    pub fn tlc_model_create(ctx: *mut TlcCtx, out: *mut *mut TlcModel) -> i32;
    pub fn tlc_model_add(m: *mut TlcModel, name: *const c_char, qt: *mut TlcQTensor) -> i32;
    pub fn tlc_model_destroy(m: *mut TlcModel) -> i32;
    pub fn tlc_model_get(m: *mut TlcModel, name: *const c_char, out: *mut *mut TlcQTensor) -> i32;
    pub fn tlc_model_tensor_count(m: *mut TlcModel) -> i32;
    pub fn tlc_model_tensor_name(m: *mut TlcModel, index: i32) -> *const c_char;
    pub fn tlc_model_meta_num(m: *mut TlcModel, key: *const c_char, out: *mut f64) -> i32;
    pub fn tlc_model_meta_str(m: *mut TlcModel, key: *const c_char) -> *const c_char;
    pub fn tlc_llama_create(ctx: *mut TlcCtx, model: *mut TlcModel, cfg: *const TlcLlamaConfig,
                            out: *mut *mut TlcLlama) -> i32;
    pub fn tlc_llama_destroy(l: *mut TlcLlama) -> i32;
    pub fn tlc_llama_prefill(l: *mut TlcLlama, ids_host: *const i32, n: i32, pos0: i32,
                             logits_host: *mut c_void, all_rows: i32, next_id_host: *mut i32) -> i32;
    pub fn tlc_llama_set_state(l: *mut TlcLlama, batch: i32, ids_host: *const i32,
                               positions_host: *const i32) -> i32;
    pub fn tlc_llama_decode_host(l: *mut TlcLlama, batch: i32, ids_host: *const i32,
                                 next_ids_host: *mut i32, logits_host: *mut c_void) -> i32;
    pub fn tlc_llama_decode_enqueue(l: *mut TlcLlama, batch: i32, steps: i32) -> i32;
    pub fn tlc_llama_read_state(l: *mut TlcLlama, batch: i32, next_ids_host: *mut i32,
                                positions_host: *mut i32) -> i32;
    pub fn tlc_llama_step_trace(l: *mut TlcLlama, steps: i32, out_ns: *mut u64, capacity: usize) -> i32;
    pub fn tlc_llama_set_sampling(l: *mut TlcLlama, temperature: f32, seed: u64) -> i32;
    pub fn tlc_sample_uniform_host(seed: u64, position: u32, sequence: u32) -> f32;
    pub fn tlc_temperature_sample(ctx: *mut TlcCtx, logits_dev: *const c_void, rows: i32, vocab: i32,
                                  temperature: f32, uniforms_host: *const f32, ids_host: *mut i32) -> i32;
    pub fn tlc_llama_decode_enqueue_parts(l: *mut TlcLlama, batch: i32, steps: i32, parts: i32) -> i32;
    pub fn tlc_token_logprobs(ctx: *mut TlcCtx, logits_dev: *const c_void, rows: i32, vocab: i32,
                              targets_dev: *const i32, top_k: i32, logprobs_dev: *mut f32,
                              entropy_dev: *mut f32, top_ids_dev: *mut i32, top_logprobs_dev: *mut f32) -> i32;
    pub fn tlc_comm_unique_id(out128: *mut c_void) -> i32;
    pub fn tlc_comm_init(ctx: *mut TlcCtx, id128: *const c_void, rank: i32, world: i32,
                         out: *mut *mut TlcComm) -> i32;
    pub fn tlc_comm_destroy(comm: *mut TlcComm) -> i32;
    pub fn tlc_comm_rank(comm: *mut TlcComm) -> i32;
    pub fn tlc_comm_size(comm: *mut TlcComm) -> i32;
    pub fn tlc_allreduce_f16(ctx: *mut TlcCtx, comm: *mut TlcComm, buf_dev: *mut c_void, count: usize) -> i32;
    pub fn tlc_allgather_f16(ctx: *mut TlcCtx, comm: *mut TlcComm, send_dev: *const c_void,
                             recv_dev: *mut c_void, count: usize) -> i32;
    pub fn tlc_comm_p2p_export(comm: *mut TlcComm, max_elems: usize, handle_out: *mut c_void) -> i32;
    pub fn tlc_comm_p2p_import(comm: *mut TlcComm, handles: *const c_void) -> i32;
    pub fn tlc_comm_p2p_ready(comm: *mut TlcComm) -> i32;
    pub fn tlc_allreduce_residual_f16(ctx: *mut TlcCtx, comm: *mut TlcComm, partial_dev: *mut c_void,
                                      residual_dev: *const c_void, out_dev: *mut c_void, count: usize) -> i32;
    pub fn tlc_llama_set_comm(l: *mut TlcLlama, comm: *mut TlcComm) -> i32;
    pub fn tlc_llama_launches_per_step(l: *mut TlcLlama, parts: i32) -> i32;
    pub fn tlc_llama_cache(l: *mut TlcLlama) -> *mut TlcKvCache;
}
