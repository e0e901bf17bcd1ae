// @generated by tools/gen_rust_ffi.py from include/shodh_hip.h -- do not edit.
#![allow(non_camel_case_types, dead_code)]
use std::os::raw::{c_char, c_int, c_void};

pub const SHODH_OK: i32 = 0;
pub const SHODH_ERR_INVALID: i32 = -1;
pub const SHODH_ERR_DIM: i32 = -2;
pub const SHODH_ERR_DEVICE: i32 = -3;
pub const SHODH_ERR_OOM: i32 = -4;
pub const SHODH_ERR_STATE: i32 = -5;
pub const SHODH_ERR_IO: i32 = -6;
pub const SHODH_ERR_NONFINITE: i32 = -7;
pub const SHODH_ERR_UNSUPPORTED: i32 = -8;
pub const SHODH_METRIC_NDP: i32 = 0;
pub const SHODH_METRIC_EUCLIDEAN: i32 = 1;
pub const SHODH_METRIC_COSINE: i32 = 2;
pub const SHODH_ORDER_SCALAR4: i32 = 0;
pub const SHODH_ORDER_AVX2: i32 = 1;
pub const SHODH_ORDER_SEQ_1M: i32 = 2;
pub const SHODH_INDEX_FLAT: i32 = 0;
pub const SHODH_INDEX_IVFPQ: i32 = 1;
pub const SHODH_SCAN_AUTO: i32 = 0;
pub const SHODH_SCAN_EXACT: i32 = 1;
pub const SHODH_SCAN_MFMA: i32 = 2;
pub const SHODH_SCAN_GRAPH: i32 = 3;
pub const SHODH_EXCHANGE_AUTO: i32 = 0;
pub const SHODH_EXCHANGE_RCCL: i32 = 1;
pub const SHODH_EXCHANGE_COPY: i32 = 2;
pub const SHODH_DTYPE_FP32: i32 = 0;
pub const SHODH_DTYPE_BF16: i32 = 1;
pub const SHODH_DTYPE_INT8: i32 = 2;
pub const SHODH_QUANT_SCOPE_BATCH: i32 = 0;
pub const SHODH_QUANT_SCOPE_PER_TEXT: i32 = 1;
pub const SHODH_WEIGHT_ABSENT: i32 = 0;
pub const SHODH_WEIGHT_F32: i32 = 1;
pub const SHODH_WEIGHT_EXPORT_Q8: i32 = 2;
pub const SHODH_WEIGHT_SELF_Q8: i32 = 3;
pub const SHODH_DTYPE_FP16: i32 = 3;
pub const SHODH_DTYPE_E4M3: i32 = 4;
pub const SHODH_REASON_COMBINED: i32 = 0;
pub const SHODH_REASON_ENTITY_MATCH: i32 = 1;
pub const SHODH_REASON_SEMANTIC_SIMILARITY: i32 = 2;
pub const SHODH_REASON_RECENT_IMPORTANT: i32 = 3;

#[repr(C)] #[derive(Clone, Copy, Debug, Default)]
pub struct shodh_index_cfg {
    pub dim: u32,
    pub metric: u32,
    pub kind: u32,
    pub order: u32,
    pub device: i32,
    pub scan_mode: u32,
    pub reserve_rows: u64,
    pub id_base: u64,
    pub nprobe: u32,
    pub reserved: u32,
    pub max_degree: u32,
    pub search_list_size: u32,
    pub alpha: f32,
    pub reserved2: u32,
}
#[repr(C)] #[derive(Clone, Copy, Debug, Default)]
pub struct shodh_sharded_cfg {
    pub dim: u32,
    pub metric: u32,
    pub kind: u32,
    pub order: u32,
    pub scan_mode: u32,
    pub nprobe: u32,
    pub block_log2: u32,
    pub exchange: u32,
    pub reserve_rows_per_shard: u64,
}
#[repr(C)] #[derive(Clone, Copy, Debug)]
pub struct shodh_embed_cfg {
    pub device: i32,
    pub dtype: u32,
    pub max_len: u32,
    pub vocab: u32,
    pub hidden: u32,
    pub layers: u32,
    pub heads: u32,
    pub intermediate: u32,
    pub max_pos: u32,
    pub type_vocab: u32,
    pub ln_eps: f32,
    pub compute_padded: u32,
    pub quant_scope: u32,
    pub weights_path: *const c_char,
}
impl Default for shodh_embed_cfg { fn default() -> Self { unsafe { std::mem::zeroed() } } }
#[repr(C)] #[derive(Clone, Copy, Debug, Default)]
pub struct shodh_rms_norm_cfg {
    pub rows: u64,
    pub x_stride: u64,
    pub residual_stride: u64,
    pub sum_stride: u64,
    pub y_stride: u64,
    pub q_stride: u64,
    pub dim: u32,
    pub dtype: u32,
    pub weight_dtype: u32,
    pub q_dtype: u32,
    pub q_group: u32,
    pub eps: f32,
}
#[repr(C)] #[derive(Clone, Copy, Debug, Default)]
pub struct shodh_attention_cfg {
    pub q_tokens: u64,
    pub kv_tokens: u64,
    pub q_stride: u64,
    pub q_head_stride: u64,
    pub k_stride: u64,
    pub k_head_stride: u64,
    pub v_stride: u64,
    pub v_head_stride: u64,
    pub out_stride: u64,
    pub out_head_stride: u64,
    pub dtype: u32,
    pub heads: u32,
    pub kv_heads: u32,
    pub head_dim: u32,
    pub seqs: u32,
    pub sinks: u32,
    pub left: i32,
    pub right: i32,
    pub scale: f32,
    pub reserved: u32,
}
#[repr(C)] #[derive(Clone, Copy, Debug, Default)]
pub struct shodh_leg_fusion_cfg {
    pub fusion_v2: u8,
    pub fusion_flat: u8,
    pub fusion_sum: u8,
    pub fusion_rrf: u8,
    pub isolate_leg: u8,
    pub flat_adaptive: u8,
    pub adapt_feature: u8,
    pub adapt_symmetric: u8,
    pub graph_w: f32,
    pub hybrid_w: f32,
    pub rrf_k: f32,
    pub flat_consensus: f32,
    pub adapt_trust_max: f32,
    pub fw_graph: f32,
    pub fw_vec: f32,
    pub fw_bm25: f32,
    pub agree_k: f32,
    pub agree_lo: f32,
    pub agree_hi: f32,
    pub peak_lo: f32,
    pub peak_hi: f32,
}
#[repr(C)] #[derive(Clone, Copy, Debug, Default)]
pub struct shodh_vama_info {
    pub num_vectors: u64,
    pub dimension: u32,
    pub max_degree: u32,
    pub medoid: u32,
    pub deleted_count: u32,
    pub incremental_inserts: u64,
    pub graph_edges: u64,
    pub distance_metric: u8,
}
#[repr(C)] #[derive(Clone, Copy, Debug, Default)]
pub struct shodh_span_info {
    pub num_vectors: u64,
    pub total_postings: u64,
    pub num_partitions: u32,
    pub dimension: u32,
    pub pq_subvectors: u32,
    pub pq_num_centroids: u32,
    pub pq_subvec_dim: u32,
    pub pq_enabled: u8,
    pub distance_metric: u8,
}
#[repr(C)] #[derive(Clone, Copy, Debug, Default)]
pub struct shodh_weights {
    pub semantic: f32,
    pub entity: f32,
    pub tag: f32,
    pub importance: f32,
    pub momentum: f32,
    pub access_count: f32,
    pub graph_strength: f32,
    pub update_count: u32,
}
#[repr(C)] #[derive(Clone, Copy, Debug, Default)]
pub struct shodh_relevance_cfg {
    pub min_importance: f32,
    pub recency_boost_hours: u64,
    pub recency_boost_multiplier: f32,
    pub graph_boost_multiplier: f32,
    pub max_results: u32,
}
#[repr(C)] pub struct shodh_index { _private: [u8; 0] }
#[repr(C)] pub struct shodh_embedder { _private: [u8; 0] }
#[repr(C)] pub struct shodh_sharded_index { _private: [u8; 0] }
#[repr(C)] pub struct shodh_weight_file { _private: [u8; 0] }
#[repr(C)] pub struct shodh_w4_weight { _private: [u8; 0] }

#[link(name = "shodh_hip")]
extern "C" {
    pub fn shodh_last_error() -> *const c_char;
    pub fn shodh_abi_version() -> c_int;
    pub fn shodh_device_count() -> c_int;
    pub fn shodh_device_info(dev: c_int, name: *mut c_char, cap: usize, hbm_bytes: *mut u64, compute_units: *mut u32) -> c_int;
    pub fn shodh_index_cfg_default(cfg: *mut shodh_index_cfg);
    pub fn shodh_index_create(cfg: *const shodh_index_cfg, out: *mut *mut shodh_index) -> c_int;
    pub fn shodh_index_destroy(idx: *mut shodh_index);
    pub fn shodh_index_add(idx: *mut shodh_index, rows: *const f32, n: u64, first_id_out: *mut u32) -> c_int;
    pub fn shodh_index_graph_overflowed(idx: *const shodh_index) -> c_int;
    pub fn shodh_index_add_device(idx: *mut shodh_index, d_rows: *const f32, n: u64, first_id_out: *mut u32) -> c_int;
    pub fn shodh_index_build(idx: *mut shodh_index, rows: *const f32, n: u64) -> c_int;
    pub fn shodh_index_build_device(idx: *mut shodh_index, d_rows: *const f32, n: u64) -> c_int;
    pub fn shodh_index_search(idx: *mut shodh_index, q: *const f32, nq: u32, k: u32, ids: *mut u32, dist: *mut f32, counts: *mut u32) -> c_int;
    pub fn shodh_index_brute_force_search(idx: *mut shodh_index, q: *const f32, nq: u32, k: u32, ids: *mut u32, dist: *mut f32, counts: *mut u32) -> c_int;
    pub fn shodh_index_search_device(idx: *mut shodh_index, d_q: *const f32, nq: u32, k: u32, d_ids: *mut u32, d_dist: *mut f32, d_counts: *mut u32, stream: *mut c_void) -> c_int;
    pub fn shodh_index_set_coalesce(idx: *mut shodh_index, enabled: c_int, linger_us: u32) -> c_int;
    pub fn shodh_index_coalesce_stats(idx: *mut shodh_index, stats6: *mut u64, reset: c_int) -> c_int;
    pub fn shodh_index_mark_deleted(idx: *mut shodh_index, id: u32, was_valid: *mut c_int) -> c_int;
    pub fn shodh_index_mark_deleted_batch(idx: *mut shodh_index, ids: *const u32, n: u64, n_marked_out: *mut u64) -> c_int;
    pub fn shodh_index_is_deleted(idx: *const shodh_index, id: u32) -> c_int;
    pub fn shodh_index_len(idx: *const shodh_index) -> u64;
    pub fn shodh_index_deleted_count(idx: *const shodh_index) -> u64;
    pub fn shodh_index_deletion_ratio(idx: *const shodh_index) -> f32;
    pub fn shodh_index_needs_compaction(idx: *const shodh_index) -> c_int;
    pub fn shodh_index_clear_deleted(idx: *mut shodh_index) -> c_int;
    pub fn shodh_index_extract_rows(idx: *const shodh_index, first: u64, n: u64, out_rows: *mut f32) -> c_int;
    pub fn shodh_index_extract_live_rows(idx: *const shodh_index, out_rows: *mut f32, ids_out: *mut u32, cap: u64, n_out: *mut u64) -> c_int;
    pub fn shodh_index_dim(idx: *const shodh_index) -> u32;
    pub fn shodh_index_stage_timings(idx: *const shodh_index, us4: *mut f32) -> c_int;
    pub fn shodh_index_kernel_timing(idx: *mut shodh_index, reset: c_int, mean_us: *mut f32, min_us: *mut f32, count: *mut u32) -> c_int;
    pub fn shodh_index_scan_stats(idx: *const shodh_index, stats8: *mut u64) -> c_int;
    pub fn shodh_index_set_graph(idx: *mut shodh_index, deg: *const u32, nbr: *const u32, stride: u32, medoid: u32) -> c_int;
    pub fn shodh_index_build_with_graph(idx: *mut shodh_index, rows: *const f32, n: u64, deg: *const u32, nbr: *const u32, stride: u32, medoid: u32) -> c_int;
    pub fn shodh_index_get_graph(idx: *const shodh_index, deg: *mut u32, nbr: *mut u32, stride: u32, medoid: *mut u32) -> c_int;
    pub fn shodh_index_vamana_build(idx: *mut shodh_index, seed: u64, init_deg: *const u32, init_nbr: *const u32, init_stride: u32) -> c_int;
    pub fn shodh_index_incremental_repair(idx: *mut shodh_index, first_node: u32, count: u32, repaired_out: *mut u32) -> c_int;
    pub fn shodh_topk_merge_device(d_in_ids: *const u32, d_in_dist: *const f32, n_lists: u32, nq: u32, k: u32, d_ids: *mut u32, d_dist: *mut f32, d_counts: *mut u32, stream: *mut c_void) -> c_int;
    pub fn shodh_topk_merge_strided_device(d_in_ids: *const u32, d_in_dist: *const f32, list_stride: u64, n_lists: u32, nq: u32, k: u32, d_ids: *mut u32, d_dist: *mut f32, d_counts: *mut u32, stream: *mut c_void) -> c_int;
    pub fn shodh_sharded_cfg_default(cfg: *mut shodh_sharded_cfg);
    pub fn shodh_sharded_index_create(cfg: *const shodh_sharded_cfg, devices: *const i32, n_devices: u32, out: *mut *mut shodh_sharded_index) -> c_int;
    pub fn shodh_sharded_index_destroy(s: *mut shodh_sharded_index);
    pub fn shodh_sharded_index_shards(s: *const shodh_sharded_index) -> u32;
    pub fn shodh_sharded_index_uses_rccl(s: *const shodh_sharded_index) -> c_int;
    pub fn shodh_sharded_index_len(s: *const shodh_sharded_index) -> u64;
    pub fn shodh_sharded_index_shard_len(s: *const shodh_sharded_index, shard: u32) -> u64;
    pub fn shodh_sharded_index_build(s: *mut shodh_sharded_index, rows: *const f32, n: u64) -> c_int;
    pub fn shodh_sharded_index_add(s: *mut shodh_sharded_index, rows: *const f32, n: u64, first_id_out: *mut u32) -> c_int;
    pub fn shodh_sharded_index_search(s: *mut shodh_sharded_index, q: *const f32, nq: u32, k: u32, ids: *mut u32, dist: *mut f32, counts: *mut u32) -> c_int;
    pub fn shodh_sharded_index_search_device(s: *mut shodh_sharded_index, d_q: *const f32, nq: u32, k: u32, d_ids: *mut u32, d_dist: *mut f32, d_counts: *mut u32, stream: *mut c_void) -> c_int;
    pub fn shodh_sharded_index_mark_deleted(s: *mut shodh_sharded_index, id: u32, was_valid: *mut c_int) -> c_int;
    pub fn shodh_sharded_index_mark_deleted_batch(s: *mut shodh_sharded_index, ids: *const u32, n: u64, n_marked_out: *mut u64) -> c_int;
    pub fn shodh_sharded_index_is_deleted(s: *mut shodh_sharded_index, id: u32) -> c_int;
    pub fn shodh_sharded_index_deleted_count(s: *mut shodh_sharded_index) -> u64;
    pub fn shodh_sharded_index_clear_deleted(s: *mut shodh_sharded_index) -> c_int;
    pub fn shodh_sharded_index_extract_rows(s: *mut shodh_sharded_index, first: u64, n: u64, out_rows: *mut f32) -> c_int;
    pub fn shodh_sharded_index_set_ivfpq(s: *mut shodh_sharded_index, centroids: *const f32, P: u32, codebook: *const f32, M: u32, ncent: u32, list_off: *const u64, ids: *const u32, codes: *const u8) -> c_int;
    pub fn shodh_sharded_index_ivfpq_insert(s: *mut shodh_sharded_index, vector_id: u32, row: *const f32) -> c_int;
    pub fn shodh_sharded_index_set_coalesce(s: *mut shodh_sharded_index, enabled: c_int, linger_us: u32) -> c_int;
    pub fn shodh_sharded_index_coalesce_stats(s: *mut shodh_sharded_index, stats6: *mut u64, reset: c_int) -> c_int;
    pub fn shodh_sharded_index_host_timings(s: *const shodh_sharded_index, us4: *mut f32) -> c_int;
    pub fn shodh_rccl_info(buf: *mut c_char, cap: usize) -> c_int;
    pub fn shodh_index_set_ivfpq(idx: *mut shodh_index, centroids: *const f32, P: u32, codebook: *const f32, M: u32, ncent: u32, list_off: *const u64, ids: *const u32, codes: *const u8) -> c_int;
    pub fn shodh_index_ivfpq_insert(idx: *mut shodh_index, vector_id: u32, row: *const f32) -> c_int;
    pub fn shodh_index_ivfpq_encode(idx: *mut shodh_index, rows: *const f32, n: u64, assign_out: *mut u32, codes_out: *mut u8) -> c_int;
    pub fn shodh_ivfpq_train(device: c_int, rows: *const f32, n: u64, dim: u32, P: u32, ivf_iters: u32, pq_iters: u32, init_perm_ivf: *const u32, init_perm_pq: *const u32, centroids_out: *mut f32, codebook_out: *mut f32) -> c_int;
    pub fn shodh_cosine_similarity_batch(device: c_int, a: *const f32, b: *const f32, n: u64, dim: u32, order: u32, out: *mut f32) -> c_int;
    pub fn shodh_top_k_similar(device: c_int, query: *const f32, query_dim: u32, cands: *const f32, n: u64, dim: u32, k: u64, order: u32, out_scores: *mut f32, out_index: *mut u32, count_out: *mut u64) -> c_int;
    pub fn shodh_embed_cfg_default(cfg: *mut shodh_embed_cfg);
    pub fn shodh_embedder_create(cfg: *const shodh_embed_cfg, out: *mut *mut shodh_embedder) -> c_int;
    pub fn shodh_embedder_destroy(e: *mut shodh_embedder);
    pub fn shodh_embedder_param_count(e: *const shodh_embedder) -> u64;
    pub fn shodh_embedder_load_weights(e: *mut shodh_embedder, blob: *const f32, n_floats: u64) -> c_int;
    pub fn shodh_embedder_load_file(e: *mut shodh_embedder, path: *const c_char) -> c_int;
    pub fn shodh_embedder_load_tensor(e: *mut shodh_embedder, name: *const c_char, data: *const f32, n: u64, transposed: u32) -> c_int;
    pub fn shodh_embedder_load_quantized(e: *mut shodh_embedder, name: *const c_char, q: *const c_void, is_signed: u32, transposed: u32, scale: *const f32, zero_point: *const c_void, n_scale: u32) -> c_int;
    pub fn shodh_embedder_finish_weights(e: *mut shodh_embedder) -> c_int;
    pub fn shodh_embedder_weight_source(e: *const shodh_embedder, name: *const c_char, source_out: *mut u32) -> c_int;
    pub fn shodh_weight_file_open(path: *const c_char, cfg: *const shodh_embed_cfg, out: *mut *mut shodh_weight_file) -> c_int;
    pub fn shodh_weight_file_close(f: *mut shodh_weight_file);
    pub fn shodh_weight_file_blob(f: *const shodh_weight_file, blob_out: *mut f32, n_floats: u64) -> c_int;
    pub fn shodh_weight_file_quantized(f: *const shodh_weight_file, name: *const c_char, q_out: *mut i8, q_len: u64, scale_out: *mut f32, zero_point_out: *mut i32, scale_cap: u32, n_scale_out: *mut u32) -> c_int;
    pub fn shodh_embedder_init_synthetic(e: *mut shodh_embedder, seed: u64, blob_out: *mut f32, n_floats: u64) -> c_int;
    pub fn shodh_embed_param_count(cfg: *const shodh_embed_cfg) -> u64;
    pub fn shodh_embedder_synthetic_weights(cfg: *const shodh_embed_cfg, seed: u64, blob_out: *mut f32, n_floats: u64) -> c_int;
    pub fn shodh_embedder_dimension(e: *const shodh_embedder) -> u32;
    pub fn shodh_embedder_encode_ids(e: *mut shodh_embedder, ids: *const i32, mask: *const u8, b: u32, out: *mut f32) -> c_int;
    pub fn shodh_embedder_encode_ids_device(e: *mut shodh_embedder, d_ids: *const i32, d_mask: *const u8, b: u32, d_out: *mut f32, stream: *mut c_void) -> c_int;
    pub fn shodh_embedder_encode_ids_scoped(e: *mut shodh_embedder, ids: *const i32, mask: *const u8, b: u32, scope: u32, out: *mut f32) -> c_int;
    pub fn shodh_embedder_encode_ids_device_scoped(e: *mut shodh_embedder, d_ids: *const i32, d_mask: *const u8, b: u32, scope: u32, d_out: *mut f32, stream: *mut c_void) -> c_int;
    pub fn shodh_embedder_set_coalesce(e: *mut shodh_embedder, enabled: c_int, linger_us: u32) -> c_int;
    pub fn shodh_embedder_coalesce_stats(e: *mut shodh_embedder, stats6: *mut u64, reset: c_int) -> c_int;
    pub fn shodh_embedder_set_quant_scope(e: *mut shodh_embedder, scope: u32) -> c_int;
    pub fn shodh_embedder_quant_scope(e: *const shodh_embedder) -> u32;
    pub fn shodh_embedder_stage_timings(e: *const shodh_embedder, us2: *mut f32) -> c_int;
    pub fn shodh_int8_dense(device: c_int, x: *const f32, w: *const f32, bias: *const f32, M: u32, N: u32, K: u32, y: *mut f32, acc_out: *mut i32, a_scale: *mut f32, a_zp: *mut i32, w_scale: *mut f32) -> c_int;
    pub fn shodh_int8_dense_quantized(device: c_int, x: *const f32, wq: *const c_void, is_signed: u32, w_scale: *const f32, w_zero_point: *const c_void, n_scale: u32, bias: *const f32, M: u32, N: u32, K: u32, y: *mut f32, acc_out: *mut i32, a_scale: *mut f32, a_zp: *mut i32) -> c_int;
    pub fn shodh_rms_norm_cfg_default(cfg: *mut shodh_rms_norm_cfg);
    pub fn shodh_rms_norm_device(device: c_int, cfg: *const shodh_rms_norm_cfg, d_x: *const c_void, d_residual: *const c_void, d_weight: *const c_void, d_sum: *mut c_void, d_y: *mut c_void, d_q: *mut c_void, d_scale: *mut f32, stream: *mut c_void) -> c_int;
    pub fn shodh_w4_weight_create(device: c_int, q: *const u8, scale: *const f32, zero: *const u8, N: u32, K: u32, group: u32, scale_dtype: u32, out: *mut *mut shodh_w4_weight) -> c_int;
    pub fn shodh_w4_weight_create_device(device: c_int, d_q: *const u8, d_scale: *const f32, d_zero: *const u8, N: u32, K: u32, group: u32, scale_dtype: u32, stream: *mut c_void, out: *mut *mut shodh_w4_weight) -> c_int;
    pub fn shodh_w4_weight_quantize(device: c_int, w: *const f32, N: u32, K: u32, group: u32, zeros: u32, scale_dtype: u32, out: *mut *mut shodh_w4_weight) -> c_int;
    pub fn shodh_w4_weight_destroy(w: *mut shodh_w4_weight);
    pub fn shodh_w4_weight_dequantize(w: *const shodh_w4_weight, out: *mut f32) -> c_int;
    pub fn shodh_w4_weight_shape(w: *const shodh_w4_weight, N: *mut u32, K: *mut u32, group: *mut u32, bytes: *mut u64) -> c_int;
    pub fn shodh_w4_dense_device(w: *const shodh_w4_weight, d_x: *const c_void, x_dtype: u32, x_stride: u64, d_x_scale: *const f32, rows: u32, d_bias: *const f32, d_y: *mut c_void, y_dtype: u32, y_stride: u64, stream: *mut c_void) -> c_int;
    pub fn shodh_attention_cfg_default(cfg: *mut shodh_attention_cfg);
    pub fn shodh_window_attention_workspace(device: c_int, cfg: *const shodh_attention_cfg, bytes: *mut u64) -> c_int;
    pub fn shodh_window_attention_device(device: c_int, cfg: *const shodh_attention_cfg, d_q: *const c_void, d_k: *const c_void, d_v: *const c_void, d_cu: *const i32, d_kv_start: *const i64, d_kv_len: *const i32, d_out: *mut c_void, d_lse: *mut f32, d_workspace: *mut c_void, workspace_bytes: u64, stream: *mut c_void) -> c_int;
    pub fn shodh_hash_embed(utf8: *const c_char, len: usize, dim: u32, out: *mut f32) -> c_int;
    pub fn shodh_finalize_pooled(pooled: *const f32, n: usize, apply_prenorm: c_int, out_dim: usize, out: *mut f32) -> usize;
    pub fn shodh_search_ids_postprocess(vec_ids: *const u32, dists: *const f32, n_res: usize, vector_to_memory: *const u8, n_vectors: usize, limit: usize, out_uuid: *mut u8, out_sim: *mut f32) -> usize;
    pub fn shodh_rrf_fuse(k: f32, weights: *const f32, n_lists: usize, uuids: *const u8, list_len: *const usize, out_uuid: *mut u8, out_score: *mut f32, out_cap: usize) -> usize;
    pub fn shodh_leg_fusion_cfg_default(c: *mut shodh_leg_fusion_cfg);
    pub fn shodh_density_weights(graph_density: f32, out3: *mut f32);
    pub fn shodh_leg_fusion_weights(has_density: c_int, graph_density: f32, graph_weight_override: f32, graph_w_floor: f32, graph_w: *mut f32, hybrid_w: *mut f32);
    pub fn shodh_fuse_legs(c: *const shodh_leg_fusion_cfg, hybrid_uuid: *const u8, hybrid_bm25: *const f32, hybrid_vec: *const f32, n_hybrid: usize, graph_uuid: *const u8, graph_activation: *const f32, n_graph: usize, query_len: usize, out_uuid: *mut u8, out_score: *mut f32, out_cap: usize, vec_trust_out: *mut f32) -> usize;
    pub fn shodh_vama_info_read(path: *const c_char, out: *mut shodh_vama_info) -> c_int;
    pub fn shodh_vama_load(path: *const c_char, vectors: *mut f32, deleted: *mut u32, degree: *mut u16, neighbors: *mut u32) -> c_int;
    pub fn shodh_vama_save(path: *const c_char, vectors: *const f32, n: u64, dim: u32, max_degree: u32, medoid: u32, metric: u8, deleted: *const u32, deleted_count: u32, incremental_inserts: u64, degree: *const u16, neighbors: *const u32) -> c_int;
    pub fn shodh_span_info_read(path: *const c_char, out: *mut shodh_span_info) -> c_int;
    pub fn shodh_span_load(path: *const c_char, centroids: *mut f32, codebook: *mut f32, list_off: *mut u64, ids: *mut u32, codes: *mut u8) -> c_int;
    pub fn shodh_span_save(path: *const c_char, num_vectors: u64, num_partitions: u32, dim: u32, pq_subvectors: u32, metric: u8, centroids: *const f32, codebook: *const f32, list_off: *const u64, ids: *const u32, codes: *const u8) -> c_int;
    pub fn shodh_weights_default(w: *mut shodh_weights);
    pub fn shodh_weights_normalize(w: *mut shodh_weights);
    pub fn shodh_weights_apply_feedback(w: *mut shodh_weights, semantic_contributed: c_int, entity_contributed: c_int, tag_contributed: c_int, helpful: c_int);
    pub fn shodh_calibrate_score(score: f32) -> f32;
    pub fn shodh_fuse_scores(w: *const shodh_weights, sem: f32, ent: f32, tag: f32, imp: f32) -> f32;
    pub fn shodh_fuse_scores_with_momentum(w: *const shodh_weights, sem: f32, ent: f32, tag: f32, imp: f32, momentum_ema: f32) -> f32;
    pub fn shodh_fuse_scores_full(w: *const shodh_weights, sem: f32, ent: f32, tag: f32, imp: f32, momentum_ema: f32, access_count: u32, graph_strength: f32) -> f32;
    pub fn shodh_fuse_scores_full_batch(device: c_int, w: *const shodh_weights, n: u64, sem: *const f32, ent: *const f32, tag: *const f32, imp: *const f32, momentum_ema: *const f32, access_count: *const u32, graph_strength: *const f32, out: *mut f32) -> c_int;
    pub fn shodh_calculate_tag_score(context_utf8: *const c_char, tags_utf8: *const *const c_char, n_tags: usize) -> f32;
    pub fn shodh_to_lowercase(utf8: *const c_char, out: *mut c_char, cap: usize) -> usize;
    pub fn shodh_apply_recency_boost(base_score: f32, age_hours: i64, boost_hours: u64, multiplier: f32) -> f32;
    pub fn shodh_relevance_cfg_default(c: *mut shodh_relevance_cfg);
    pub fn shodh_rank_surfaced(w: *const shodh_weights, cfg: *const shodh_relevance_cfg, n: usize, semantic: *const f32, entity: *const f32, tag: *const f32, importance: *const f32, momentum_ema: *const f32, access_count: *const u32, graph_strength: *const f32, age_hours: *const i64, created_at_ns: *const i64, uuid: *const u8, out_index: *mut u32, out_score: *mut f32, out_reason: *mut u8) -> usize;
    pub fn shodh_guard_mode() -> c_int;
    pub fn shodh_guard_stats(allocations: *mut u64, frees: *mut u64, live_device_bytes: *mut u64) -> c_int;
    pub fn shodh_guard_torch_alloc(bytes: i64, device: c_int, stream: *mut c_void) -> *mut c_void;
    pub fn shodh_guard_torch_free(p: *mut c_void, bytes: i64, device: c_int, stream: *mut c_void);
}
