//! Raw bindings of the C ABI in `include/nvllm_attn.h` (libnvllm_attn.so).
//! GENERATED by scripts/gen_rust_ffi.py from the header -- do not edit by hand.
//! NOT COMPILED in the build image (no Rust toolchain there); tests/test_rust_crate.py keeps
//! the symbol list and argument counts equal to the header's.
#![allow(non_camel_case_types, clippy::too_many_arguments)]
use std::ffi::{c_char, c_int, c_void};

/// hipStream_t (NULL = the default stream)
pub type Stream = *mut c_void;

/// opaque `nvllm_block_table`
#[repr(C)]
pub struct NvllmBlockTable {
    _private: [u8; 0],
}
/// opaque `nvllm_block_manager`
#[repr(C)]
pub struct NvllmBlockManager {
    _private: [u8; 0],
}
/// opaque `nvllm_batch`
#[repr(C)]
pub struct NvllmBatch {
    _private: [u8; 0],
}
/// opaque `nvllm_scheduler`
#[repr(C)]
pub struct NvllmScheduler {
    _private: [u8; 0],
}

/// `nvllm_scheduler_config` (SchedulerConfig, src/config.rs:44-57, plus the two opt-in repairs)
#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct NvllmSchedulerConfig {
    pub max_num_seqs: i64,
    pub max_prefill_tokens: i64,
    pub enable_chunked_prefill: c_int,
    pub chunk_size: i64,
    pub enable_priority: c_int,
    pub enable_preemption: c_int,
    pub reschedule_partial_prefill: c_int,
    pub enable_prefix_caching: c_int,
}

/// `nvllm_status`
pub const NVLLM_OK: c_int = 0;
pub const NVLLM_ERR_CONFIG: c_int = -1;
pub const NVLLM_ERR_UNSUPPORTED: c_int = -2;
pub const NVLLM_ERR_NULL: c_int = -3;
pub const NVLLM_ERR_HIP: c_int = -4;
pub const NVLLM_ERR_OUT_OF_BLOCKS: c_int = -5;
pub const NVLLM_ERR_BLOCK_INDEX_OOB: c_int = -6;
pub const NVLLM_ERR_TENSOR: c_int = -7;

#[link(name = "nvllm_attn")]
extern "C" {
    pub fn nvllm_flash_attn_fwd_bf16(q: *const c_void, k: *const c_void, v: *const c_void, o: *mut c_void, lse: *mut f32, batch: c_int, seq_q: c_int, seq_kv: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, softmax_scale: f32, causal: c_int, stream: Stream) -> c_int;
    pub fn nvllm_flash_attn_fwd_f32(q: *const c_void, k: *const c_void, v: *const c_void, o: *mut c_void, lse: *mut f32, batch: c_int, seq_q: c_int, seq_kv: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, softmax_scale: f32, causal: c_int, stream: Stream) -> c_int;
    pub fn nvllm_paged_attn_bf16(q: *const c_void, k_cache: *const c_void, v_cache: *const c_void, block_tables: *const i32, context_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, num_seqs: c_int, num_new_tokens: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, max_blocks_per_seq: c_int, num_cache_blocks: i64, scale: f32, stream: Stream) -> c_int;
    pub fn nvllm_paged_attn_f32(q: *const c_void, k_cache: *const c_void, v_cache: *const c_void, block_tables: *const i32, context_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, num_seqs: c_int, num_new_tokens: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, max_blocks_per_seq: c_int, num_cache_blocks: i64, scale: f32, stream: Stream) -> c_int;
    pub fn nvllm_paged_attn_bf16_noalloc(q: *const c_void, k_cache: *const c_void, v_cache: *const c_void, block_tables: *const i32, context_lens: *const i32, out: *mut c_void, num_seqs: c_int, num_new_tokens: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, max_blocks_per_seq: c_int, num_cache_blocks: i64, scale: f32, stream: Stream) -> c_int;
    pub fn nvllm_paged_attn_noalloc_max_scratch_bytes() -> usize;
    pub fn nvllm_paged_attn_workspace_bytes(num_seqs: c_int, num_new_tokens: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, max_blocks_per_seq: c_int) -> usize;
    pub fn nvllm_paged_attn_path(num_seqs: c_int, num_new_tokens: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, max_blocks_per_seq: c_int, num_cache_blocks: i64, dtype: c_int) -> c_int;
    pub fn nvllm_reshape_and_cache_bf16(key: *const c_void, value: *const c_void, k_cache: *mut c_void, v_cache: *mut c_void, slot_mapping: *const i64, num_tokens: i64, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, num_cache_blocks: i64, stream: Stream) -> c_int;
    pub fn nvllm_reshape_and_cache_f32(key: *const c_void, value: *const c_void, k_cache: *mut c_void, v_cache: *mut c_void, slot_mapping: *const i64, num_tokens: i64, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, num_cache_blocks: i64, stream: Stream) -> c_int;
    pub fn nvllm_gather_cache_blocks(cache: *const c_void, block_ids: *const i32, num_ids: i64, out: *mut c_void, num_cache_blocks: i64, block_size: c_int, num_kv_heads: c_int, head_dim: c_int, dtype: c_int, stream: Stream) -> c_int;
    pub fn nvllm_qk_norm_rope_cache_bf16(q: *const c_void, k: *const c_void, v: *const c_void, q_out: *mut c_void, k_out: *mut c_void, q_weight: *const c_void, k_weight: *const c_void, eps: f32, cos_cache: *const c_void, sin_cache: *const c_void, max_positions: i64, positions: *const i32, k_cache: *mut c_void, v_cache: *mut c_void, slot_mapping: *const i64, num_tokens: i64, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, num_cache_blocks: i64, stream: Stream) -> c_int;
    pub fn nvllm_qk_norm_rope_cache_f32(q: *const c_void, k: *const c_void, v: *const c_void, q_out: *mut c_void, k_out: *mut c_void, q_weight: *const c_void, k_weight: *const c_void, eps: f32, cos_cache: *const c_void, sin_cache: *const c_void, max_positions: i64, positions: *const i32, k_cache: *mut c_void, v_cache: *mut c_void, slot_mapping: *const i64, num_tokens: i64, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, num_cache_blocks: i64, stream: Stream) -> c_int;
    pub fn nvllm_kv8_write_workspace_bytes(num_tokens: i64, block_size: c_int, num_cache_blocks: i64) -> usize;
    pub fn nvllm_reshape_and_cache_kv8(key: *const c_void, value: *const c_void, k_cache: *mut c_void, v_cache: *mut c_void, k_scales: *mut f32, v_scales: *mut f32, slot_mapping: *const i64, workspace: *mut c_void, workspace_bytes: usize, num_tokens: i64, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, num_cache_blocks: i64, format: c_int, dtype: c_int, stream: Stream) -> c_int;
    pub fn nvllm_qk_norm_rope_cache_kv8(q: *const c_void, k: *const c_void, v: *const c_void, q_out: *mut c_void, k_out: *mut c_void, q_weight: *const c_void, k_weight: *const c_void, eps: f32, cos_cache: *const c_void, sin_cache: *const c_void, max_positions: i64, positions: *const i32, k_cache: *mut c_void, v_cache: *mut c_void, k_scales: *mut f32, v_scales: *mut f32, slot_mapping: *const i64, workspace: *mut c_void, workspace_bytes: usize, num_tokens: i64, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, num_cache_blocks: i64, format: c_int, dtype: c_int, stream: Stream) -> c_int;
    pub fn nvllm_gather_cache_blocks_kv8(k_cache: *const c_void, v_cache: *const c_void, k_scales: *const f32, v_scales: *const f32, block_ids: *const i32, num_ids: i64, k_out: *mut c_void, v_out: *mut c_void, num_cache_blocks: i64, block_size: c_int, num_kv_heads: c_int, head_dim: c_int, format: c_int, dtype: c_int, stream: Stream) -> c_int;
    pub fn nvllm_paged_attn_kv8(q: *const c_void, k_cache: *const c_void, v_cache: *const c_void, k_scales: *const f32, v_scales: *const f32, block_tables: *const i32, context_lens: *const i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, num_seqs: c_int, num_new_tokens: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, max_blocks_per_seq: c_int, num_cache_blocks: i64, scale: f32, format: c_int, dtype: c_int, stream: Stream) -> c_int;
    pub fn nvllm_paged_attn_kv8_workspace_bytes(num_seqs: c_int, num_new_tokens: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, max_blocks_per_seq: c_int, dtype: c_int) -> usize;
    pub fn nvllm_paged_attn_kv8_path(num_seqs: c_int, num_new_tokens: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int, max_blocks_per_seq: c_int, dtype: c_int) -> c_int;
    pub fn nvllm_kv_cache_kv8_layer_bytes(num_blocks: i64, block_size: i64, num_kv_heads: i64, head_dim: i64) -> i64;
    pub fn nvllm_get_last_error() -> *const c_char;
    pub fn nvllm_synchronize() -> c_int;
    pub fn nvllm_kv_cache_layer_bytes(num_blocks: i64, block_size: i64, num_kv_heads: i64, head_dim: i64, dtype: c_int) -> i64;
    pub fn nvllm_kv_cache_total_bytes(num_blocks: i64, block_size: i64, num_kv_heads: i64, head_dim: i64, num_layers: i64, dtype: c_int) -> i64;
    pub fn nvllm_debug_set_policy(name: *const c_char, value: c_int) -> c_int;
    pub fn nvllm_debug_reset_policy();
    pub fn nvllm_debug_validate_tables(block_tables: *const i32, context_lens: *const i32, num_seqs: c_int, max_blocks_per_seq: c_int, block_size: c_int, num_cache_blocks: i64, counts: *mut i32, stream: Stream) -> c_int;
    pub fn nvllm_device_count() -> c_int;
    pub fn nvllm_set_device(device: c_int) -> c_int;
    pub fn nvllm_compute_num_blocks(seq_len: i64, block_size: i64) -> i64;
    pub fn nvllm_hash_token_block(token_ids: *const u32, num_tokens: i64, has_parent: c_int, parent_hash: u64) -> u64;
    pub fn nvllm_rope_cache_f32(dim: i64, max_seq_len: i64, theta: f64, cos_out: *mut f32, sin_out: *mut f32) -> c_int;
    pub fn nvllm_slot_mapping_last_writer(slots: *const i64, n: i64, out: *mut i64) -> i64;
    pub fn nvllm_block_table_new(block_size: i64) -> *mut NvllmBlockTable;
    pub fn nvllm_block_table_free(t: *mut NvllmBlockTable);
    pub fn nvllm_block_table_block_size(t: *const NvllmBlockTable) -> i64;
    pub fn nvllm_block_table_append_block(t: *mut NvllmBlockTable, block_id: i64);
    pub fn nvllm_block_table_num_blocks(t: *const NvllmBlockTable) -> i64;
    pub fn nvllm_block_table_is_empty(t: *const NvllmBlockTable) -> c_int;
    pub fn nvllm_block_table_clear(t: *mut NvllmBlockTable);
    pub fn nvllm_block_table_get_block_id(t: *const NvllmBlockTable, logical_idx: i64, block_id_out: *mut i64) -> c_int;
    pub fn nvllm_block_table_get_physical_block_ids(t: *const NvllmBlockTable, ids_out: *mut i64, cap: i64) -> i64;
    pub fn nvllm_block_table_get_slot_mapping(t: *const NvllmBlockTable, seq_len: i64, slots_out: *mut i64, cap: i64) -> i64;
    pub fn nvllm_block_manager_new(num_blocks: i64, block_size: i64) -> *mut NvllmBlockManager;
    pub fn nvllm_block_manager_free_handle(m: *mut NvllmBlockManager);
    pub fn nvllm_block_manager_block_size(m: *const NvllmBlockManager) -> i64;
    pub fn nvllm_block_manager_num_blocks(m: *const NvllmBlockManager) -> i64;
    pub fn nvllm_block_manager_num_free_blocks(m: *const NvllmBlockManager) -> i64;
    pub fn nvllm_block_manager_num_used_blocks(m: *const NvllmBlockManager) -> i64;
    pub fn nvllm_block_manager_has_free_blocks(m: *const NvllmBlockManager) -> c_int;
    pub fn nvllm_block_manager_can_allocate(m: *const NvllmBlockManager, n: i64) -> c_int;
    pub fn nvllm_block_manager_allocate(m: *mut NvllmBlockManager, block_id_out: *mut i64) -> c_int;
    pub fn nvllm_block_manager_allocate_many(m: *mut NvllmBlockManager, n: i64, ids_out: *mut i64) -> c_int;
    pub fn nvllm_block_manager_free(m: *mut NvllmBlockManager, block_id: i64) -> c_int;
    pub fn nvllm_block_manager_free_many(m: *mut NvllmBlockManager, ids: *const i64, n: i64) -> i64;
    pub fn nvllm_block_manager_ref_count(m: *const NvllmBlockManager, block_id: i64) -> i64;
    pub fn nvllm_block_manager_prefix_hash(m: *const NvllmBlockManager, block_id: i64, hash_out: *mut u64) -> c_int;
    pub fn nvllm_block_manager_increment_ref(m: *mut NvllmBlockManager, block_id: i64) -> i64;
    pub fn nvllm_block_manager_decrement_ref(m: *mut NvllmBlockManager, block_id: i64) -> i64;
    pub fn nvllm_block_manager_get_cached_block(m: *mut NvllmBlockManager, prefix_hash: u64) -> i64;
    pub fn nvllm_block_manager_cache_block(m: *mut NvllmBlockManager, block_id: i64, prefix_hash: u64);
    pub fn nvllm_block_manager_allocate_with_prefix(m: *mut NvllmBlockManager, prefix_hash: u64, block_id_out: *mut i64, was_cached_out: *mut c_int) -> c_int;
    pub fn nvllm_block_manager_is_prefix_cached(m: *const NvllmBlockManager, prefix_hash: u64) -> c_int;
    pub fn nvllm_block_manager_num_cached_prefixes(m: *const NvllmBlockManager) -> i64;
    pub fn nvllm_block_manager_clear_prefix_cache(m: *mut NvllmBlockManager);
    pub fn nvllm_block_manager_reset(m: *mut NvllmBlockManager);
    pub fn nvllm_batch_new(max_blocks_per_seq: i64) -> *mut NvllmBatch;
    pub fn nvllm_batch_free(b: *mut NvllmBatch);
    pub fn nvllm_batch_clear(b: *mut NvllmBatch);
    pub fn nvllm_batch_add_sequence(b: *mut NvllmBatch, t: *const NvllmBlockTable, context_len: i64, num_new_tokens: i64) -> c_int;
    pub fn nvllm_batch_num_seqs(b: *const NvllmBatch) -> i64;
    pub fn nvllm_batch_num_tokens(b: *const NvllmBatch) -> i64;
    pub fn nvllm_batch_max_blocks_per_seq(b: *const NvllmBatch) -> i64;
    pub fn nvllm_batch_block_tables(b: *const NvllmBatch) -> *const i32;
    pub fn nvllm_batch_context_lens(b: *const NvllmBatch) -> *const i32;
    pub fn nvllm_batch_slot_mapping(b: *const NvllmBatch) -> *const i64;
    pub fn nvllm_batch_query_start(b: *const NvllmBatch) -> *const i32;
    pub fn nvllm_batch_positions(b: *const NvllmBatch) -> *const i32;
    pub fn nvllm_batch_upload(b: *const NvllmBatch, d_block_tables: *mut c_void, d_context_lens: *mut c_void, d_slot_mapping: *mut c_void, d_query_start: *mut c_void, d_positions: *mut c_void, stream: Stream) -> c_int;
    pub fn nvllm_scheduler_config_default(c: *mut NvllmSchedulerConfig);
    pub fn nvllm_scheduler_new(c: *const NvllmSchedulerConfig, block_size: i64, num_blocks: i64) -> *mut NvllmScheduler;
    pub fn nvllm_scheduler_free(s: *mut NvllmScheduler);
    pub fn nvllm_scheduler_add_sequence(s: *mut NvllmScheduler, seq_id: u64, prompt: *const u32, num_tokens: i64, priority: i32) -> c_int;
    pub fn nvllm_scheduler_remove_sequence(s: *mut NvllmScheduler, seq_id: u64) -> c_int;
    pub fn nvllm_scheduler_schedule(s: *mut NvllmScheduler) -> c_int;
    pub fn nvllm_scheduler_out_num_prefill(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_out_num_decode(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_out_num_preempted(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_out_prefill_ids(s: *const NvllmScheduler) -> *const u64;
    pub fn nvllm_scheduler_out_decode_ids(s: *const NvllmScheduler) -> *const u64;
    pub fn nvllm_scheduler_out_preempted_ids(s: *const NvllmScheduler) -> *const u64;
    pub fn nvllm_scheduler_out_prefill_chunk_sizes(s: *const NvllmScheduler) -> *const i64;
    pub fn nvllm_scheduler_out_num_prefill_tokens(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_out_num_decode_tokens(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_finish_sequence(s: *mut NvllmScheduler, seq_id: u64, reason: c_int);
    pub fn nvllm_scheduler_append_token(s: *mut NvllmScheduler, seq_id: u64, token: u32) -> c_int;
    pub fn nvllm_scheduler_mark_prefilled(s: *mut NvllmScheduler, seq_id: u64, num_tokens: i64) -> c_int;
    pub fn nvllm_scheduler_num_waiting(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_num_running(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_num_swapped(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_has_unfinished_sequences(s: *const NvllmScheduler) -> c_int;
    pub fn nvllm_scheduler_has_pending_requests(s: *const NvllmScheduler) -> c_int;
    pub fn nvllm_scheduler_running_sequence_ids(s: *const NvllmScheduler, out: *mut u64, cap: i64) -> i64;
    pub fn nvllm_scheduler_reset(s: *mut NvllmScheduler);
    pub fn nvllm_scheduler_seq_status(s: *const NvllmScheduler, seq_id: u64) -> c_int;
    pub fn nvllm_scheduler_seq_finish_reason(s: *const NvllmScheduler, seq_id: u64) -> c_int;
    pub fn nvllm_scheduler_seq_set_status(s: *mut NvllmScheduler, seq_id: u64, status: c_int) -> c_int;
    pub fn nvllm_scheduler_seq_info(s: *const NvllmScheduler, seq_id: u64, what: c_int) -> i64;
    pub fn nvllm_scheduler_seq_block_ids(s: *const NvllmScheduler, seq_id: u64, out: *mut i64, cap: i64) -> i64;
    pub fn nvllm_scheduler_seq_output_tokens(s: *const NvllmScheduler, seq_id: u64, out: *mut u32, cap: i64) -> i64;
    pub fn nvllm_scheduler_num_free_blocks(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_num_used_blocks(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_num_cached_prefixes(s: *const NvllmScheduler) -> i64;
    pub fn nvllm_scheduler_block_ref_count(s: *const NvllmScheduler, block_id: i64) -> i64;
    pub fn nvllm_scheduler_fill_decode_batch(s: *const NvllmScheduler, batch: *mut NvllmBatch) -> c_int;
    pub fn nvllm_scheduler_fill_prefill_batch(s: *const NvllmScheduler, num_new_tokens: i64, batch: *mut NvllmBatch, ids_out: *mut u64, cap: i64) -> i64;
    pub fn nvllm_paged_attention_seq_scratch_bytes(num_table_blocks: i64, num_new_tokens: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, block_size: c_int) -> usize;
    pub fn nvllm_paged_attention_seq(query: *const c_void, batch: c_int, num_new_tokens: c_int, k_cache: *const c_void, v_cache: *const c_void, num_cache_blocks: i64, block_table: *const NvllmBlockTable, context_len: i64, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, scale: f64, dtype: c_int, out: *mut c_void, scratch: *mut c_void, scratch_bytes: usize, stream: Stream) -> c_int;
    pub fn nvllm_write_kv_to_cache(key: *const c_void, value: *const c_void, seq_len: i64, k_cache: *mut c_void, v_cache: *mut c_void, num_cache_blocks: i64, slot_mapping: *const i64, slot_mapping_len: i64, block_size: c_int, num_kv_heads: c_int, head_dim: c_int, dtype: c_int, scratch: *mut c_void, scratch_bytes: usize, stream: Stream) -> c_int;
    pub fn nvllm_prefill_attention(q: *const c_void, k: *const c_void, v: *const c_void, out: *mut c_void, batch: c_int, seq_len: c_int, num_heads: c_int, num_kv_heads: c_int, head_dim: c_int, scale: f64, causal: c_int, dtype: c_int, stream: Stream) -> c_int;
}
