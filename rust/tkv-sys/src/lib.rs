// Raw FFI of the B200 KV handoff library (include/tkv.h).  GENERATED by gen_bindings.py: do not edit.
// Not compiled in the environment it was written in (no Rust toolchain there); tests/test_rust_shim.py checks it
// against the header mechanically: names, argument counts and types, struct field order.
#![allow(non_camel_case_types, non_upper_case_globals, dead_code)]
use std::os::raw::{c_char, c_void};

pub const TKV_OK: i32 = 0;
pub const TKV_ERR_DIMENSION_MISMATCH: i32 = 1;
pub const TKV_ERR_INVALID_CONFIG: i32 = 2;
pub const TKV_ERR_CUDA: i32 = 3;
pub const TKV_ERR_TIMEOUT: i32 = 4;
pub const TKV_ERR_POOL_EXHAUSTED: i32 = 5;
pub const TKV_DTYPE_F32: i32 = 0;
pub const TKV_DTYPE_F16: i32 = 1;
pub const TKV_DTYPE_E4M3: i32 = 2;
pub const TKV_PLAN_DEFAULT: u32 = 0;
pub const TKV_PLAN_ALLOW_SHARED_DST: u32 = 1;
pub const TKV_PLAN_FORCE_VECTOR: u32 = 2;
pub const TKV_PLAN_FORCE_BULK: u32 = 4;
pub const TKV_PLAN_INT_QUANTIZER: u32 = 8;
pub const TKV_PLAN_PEER_BULK_STORES: u32 = 16;
pub const TKV_PLAN_PULL: u32 = 32;
pub const TKV_PLAN_STAGE_HOST: u32 = 64;
pub const TKV_VARIANT_VECTOR: u32 = 1;
pub const TKV_VARIANT_BULK: u32 = 2;
pub const TKV_VARIANT_FP8_WARP: u32 = 3;
pub const TKV_VARIANT_FP8_GENERIC: u32 = 4;
pub const TKV_VARIANT_CAST_GENERIC: u32 = 5;
pub const TKV_VARIANT_FP8_STAGED: u32 = 6;
pub const TKV_VARIANT_DEQUANT: u32 = 7;
pub const TKV_VARIANT_CAST_VEC: u32 = 8;
pub const TKV_VARIANT_WIDE: u32 = 9;
pub const TKV_ATTN_DEFAULT: u32 = 0;
pub const TKV_ATTN_PER_HEAD_CTAS: u32 = 1;
pub const TKV_ATTN_MMA_SYNC: u32 = 2;
pub const TKV_PREFILL_DEFAULT: u32 = 0;
pub const TKV_PREFILL_SINGLE_TILE: u32 = 1;
pub const TKV_PREFILL_TWO_TILES: u32 = 2;
pub const TKV_REQ_QUEUED: u32 = 0;
pub const TKV_REQ_PREFILL: u32 = 1;
pub const TKV_REQ_WAITING: u32 = 2;
pub const TKV_REQ_ADMITTED: u32 = 3;
pub const TKV_REQ_TRANSFER: u32 = 4;
pub const TKV_REQ_DECODE: u32 = 5;
pub const TKV_REQ_REPREFILL: u32 = 6;
pub const TKV_RETRY_HANDOFF: u32 = 1;
pub const TKV_REPREFILL: u32 = 2;
pub const TKV_NOALLOC_MAX_BLOCK_PAIRS: u32 = 16384;
pub const TKV_NOALLOC_MAX_LAYERS: u32 = 128;
pub const TKV_NOALLOC_SCRATCH_BYTES: u32 = (4 * TKV_NOALLOC_MAX_LAYERS * 8 + 256 + TKV_NOALLOC_MAX_BLOCK_PAIRS * 16);
pub const TKV_PREFIX_NO_PAGE: u32 = 0xFFFFFFFF;

#[repr(C)]
pub struct tkv_plan {
    _private: [u8; 0],
}
#[repr(C)]
pub struct tkv_page_allocator {
    _private: [u8; 0],
}
#[repr(C)]
pub struct tkv_block_table {
    _private: [u8; 0],
}
#[repr(C)]
pub struct tkv_run_allocator {
    _private: [u8; 0],
}
#[repr(C)]
pub struct tkv_radix_tree {
    _private: [u8; 0],
}
#[repr(C)]
pub struct tkv_prefix_table {
    _private: [u8; 0],
}
#[repr(C)]
pub struct tkv_prefix_index {
    _private: [u8; 0],
}
#[repr(C)]
pub struct tkv_device_page_allocator {
    _private: [u8; 0],
}
#[repr(C)]
pub struct tkv_coordinator {
    _private: [u8; 0],
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvPool {
    pub device: i32,
    pub dtype: i32,
    pub n_layers: u32,
    pub n_kv_heads: u32,
    pub head_dim: u32,
    pub block_size: u32,
    pub total_blocks: u32,
    pub reserved: u32,
    pub k_layer_ptrs: *const u64,
    pub v_layer_ptrs: *const u64,
    pub k_scales: u64,
    pub v_scales: u64,
    pub refcounts: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvBatch {
    pub n_seqs: u32,
    pub table_stride: u32,
    pub table_layer_stride: u32,
    pub reserved: u32,
    pub seq_lens: *const u32,
    pub prefix_lens: *const u32,
    pub src_tables: *const u32,
    pub dst_tables: *const u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvShard {
    pub src_head_begin: u32,
    pub dst_head_begin: u32,
    pub n_heads: u32,
    pub src_layer_begin: u32,
    pub dst_layer_begin: u32,
    pub n_layers: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvPairing {
    pub prefill_device: i32,
    pub decode_device: i32,
    pub shard: TkvShard,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvStats {
    pub payload_bytes: u64,
    pub bytes_read: u64,
    pub bytes_written: u64,
    pub n_blocks: u64,
    pub n_chunks: u64,
    pub n_tokens: u64,
    pub n_prefix_refs: u64,
    pub worklist_bytes: u64,
    pub grid: u32,
    pub block: u32,
    pub kernel_variant: u32,
    pub peer: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvTransfer {
    pub device: i32,
    pub dtype: i32,
    pub host_memory: u32,
    pub reserved: u32,
    pub data: u64,
    pub bytes: u64,
    pub scales: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvDecodeAttn {
    pub n_seqs: u32,
    pub n_q_heads: u32,
    pub table_stride: u32,
    pub layer: u32,
    pub max_kv_len: u32,
    pub sm_scale: f32,
    pub split_tokens: u32,
    pub flags: u32,
    pub q: u64,
    pub out: u64,
    pub tables: u64,
    pub kv_lens: u64,
    pub scratch: u64,
    pub scratch_bytes: u64,
    pub total_kv_tokens: u64,
    pub status: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvPrefillAttn {
    pub n_tokens: u32,
    pub n_q_heads: u32,
    pub layer: u32,
    pub start_pos: u32,
    pub table_len: u32,
    pub sm_scale: f32,
    pub flags: u32,
    pub reserved: u32,
    pub q: u64,
    pub out: u64,
    pub table: u64,
    pub status: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvScoredAttn {
    pub n_seqs: u32,
    pub n_q_heads: u32,
    pub table_stride: u32,
    pub layer: u32,
    pub max_kv_len: u32,
    pub score_stride: u32,
    pub sm_scale: f32,
    pub decay: f32,
    pub q_dtype: i32,
    pub reserved: u32,
    pub q: u64,
    pub out: u64,
    pub tables: u64,
    pub kv_lens: u64,
    pub scores: u64,
    pub scratch: u64,
    pub scratch_bytes: u64,
    pub status: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvPrefixAttn {
    pub n_seqs: u32,
    pub n_groups: u32,
    pub n_q_heads: u32,
    pub table_stride: u32,
    pub layer: u32,
    pub max_kv_len: u32,
    pub max_prefix_len: u32,
    pub sm_scale: f32,
    pub q: u64,
    pub out: u64,
    pub tables: u64,
    pub kv_lens: u64,
    pub group_starts: u64,
    pub prefix_lens: u64,
    pub scratch: u64,
    pub scratch_bytes: u64,
    pub status: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvEvictSelect {
    pub device: i32,
    pub n_layers: u32,
    pub n_seqs: u32,
    pub n_kv_heads: u32,
    pub max_kv_len: u32,
    pub score_stride: u32,
    pub kept_stride: u32,
    pub budget: u32,
    pub recent: u32,
    pub reserved: u32,
    pub scores: u64,
    pub kv_lens: u64,
    pub protect: u64,
    pub kept: u64,
    pub new_lens: u64,
    pub status: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvEvictCompact {
    pub layer_begin: u32,
    pub n_layers: u32,
    pub n_seqs: u32,
    pub table_stride: u32,
    pub max_kv_len: u32,
    pub score_stride: u32,
    pub kept_stride: u32,
    pub reserved: u32,
    pub tables: u64,
    pub kv_lens: u64,
    pub kept: u64,
    pub new_lens: u64,
    pub scores: u64,
    pub status: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvSessionHeader {
    pub position: u64,
    pub seed: u64,
    pub seq_len: u32,
    pub n_layers: u32,
    pub n_kv_heads: u32,
    pub head_dim: u32,
    pub block_size: u32,
    pub kv_dtype: u32,
    pub block_begin: u32,
    pub n_blocks: u32,
    pub piece_index: u32,
    pub piece_count: u32,
    pub n_logits: u32,
    pub reserved: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvPrefixBatch {
    pub n_seqs: u32,
    pub stride: u32,
    pub page_stride: u32,
    pub reserved: u32,
    pub tokens: u64,
    pub lens: u64,
    pub pages: u64,
    pub page_lens: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvPrefixIndexStats {
    pub hits: u64,
    pub tokens_saved: u64,
    pub live_nodes: u64,
    pub tombstones: u64,
    pub capacity: u64,
    pub ticks: u64,
    pub group_tokens: u32,
    pub table_full: u32,
    pub key_collisions: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvPageBatch {
    pub n_seqs: u32,
    pub table_stride: u32,
    pub tables: u64,
    pub first: u64,
    pub counts: u64,
    pub seq_lens: u64,
    pub block_size: u32,
    pub reserved: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvDeviceBatch {
    pub n_seqs: u32,
    pub table_stride: u32,
    pub apply_refcounts: u32,
    pub reserved: u32,
    pub seq_lens: u64,
    pub prefix_lens: u64,
    pub src_tables: u64,
    pub dst_tables: u64,
    pub status: u64,
    pub prefix_blocks: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvCoordinatorConfig {
    pub n_prefill: u32,
    pub n_decode: u32,
    pub block_size: u32,
    pub max_inflight_per_decode: u32,
    pub max_retries: u32,
    pub headroom_blocks: u32,
    pub handoff_timeout: u64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvAdmission {
    pub request_id: u64,
    pub prefill_worker: u32,
    pub decode_worker: u32,
    pub blocks: u32,
    pub prefix_tokens: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvRequestInfo {
    pub request_id: u64,
    pub state: u32,
    pub prefill_worker: u32,
    pub decode_worker: u32,
    pub reserved_blocks: u32,
    pub prefix_tokens: u32,
    pub attempts: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct TkvCoordinatorStats {
    pub submitted: u64,
    pub admitted: u64,
    pub handoffs_completed: u64,
    pub handoffs_failed: u64,
    pub retries: u64,
    pub fallbacks: u64,
    pub finished: u64,
    pub in_system: u64,
    pub waiting: u64,
    pub reserved_blocks: u64,
}

extern "C" {
    pub fn tkv_last_error(buf: *mut c_char, len: usize);
    pub fn tkv_last_cuda_error() -> i32;
    pub fn tkv_version() -> *const c_char;
    pub fn tkv_init(devices: *const i32, n_devices: i32) -> i32;
    pub fn tkv_shutdown() -> i32;
    pub fn tkv_plan_create(src: *const TkvPool, dst: *const TkvPool, batch: *const TkvBatch, shard: *const TkvShard, flags: u32, out: *mut *mut tkv_plan) -> i32;
    pub fn tkv_plan_create_to_transfer(src: *const TkvPool, xfer: *const TkvTransfer, batch: *const TkvBatch, shard: *const TkvShard, flags: u32, out: *mut *mut tkv_plan) -> i32;
    pub fn tkv_plan_create_from_transfer(xfer: *const TkvTransfer, dst: *const TkvPool, batch: *const TkvBatch, shard: *const TkvShard, flags: u32, out: *mut *mut tkv_plan) -> i32;
    pub fn tkv_transfer_bytes(n_layers: u32, n_heads: u32, head_dim: u32, block_size: u32, dtype: i32, n_blocks: u64) -> u64;
    pub fn tkv_batch_blocks(batch: *const TkvBatch, block_size: u32) -> u64;
    pub fn tkv_plan_update(plan: *mut tkv_plan, batch: *const TkvBatch) -> i32;
    pub fn tkv_plan_destroy(plan: *mut tkv_plan) -> i32;
    pub fn tkv_plan_stats(plan: *const tkv_plan, out: *mut TkvStats) -> i32;
    pub fn tkv_handoff_enqueue(plan: *mut tkv_plan, stream: *mut c_void, done_flag: u64, flag_value: u32) -> i32;
    pub fn tkv_handoff_noalloc(src: *const TkvPool, dst: *const TkvPool, batch: *const TkvBatch, shard: *const TkvShard, stream: *mut c_void) -> i32;
    pub fn tkv_plan_tune_bulk(plan: *mut tkv_plan, stages: u32, ctas_per_sm: u32, stage_bytes: u32) -> i32;
    pub fn tkv_plan_tune_vector(plan: *mut tkv_plan, bytes_per_access: u32, unroll: u32, store_hint: u32) -> i32;
    pub fn tkv_plan_tune_small(plan: *mut tkv_plan, flag_mode: u32, inline_list: u32) -> i32;
    pub fn tkv_plan_tune_grid(plan: *mut tkv_plan, ctas_per_sm: u32) -> i32;
    pub fn tkv_plan_error(plan: *const tkv_plan, device_error: *mut u32) -> i32;
    pub fn tkv_flag_wait_host(device: i32, flag: u64, expected: u32, timeout_us: u64) -> i32;
    pub fn tkv_flag_wait_enqueue(stream: *mut c_void, flag: u64, expected: u32, max_spins: u64, status: u64) -> i32;
    pub fn tkv_refcount_apply(plan: *mut tkv_plan, delta: i32, stream: *mut c_void) -> i32;
    pub fn tkv_pairing_make(n_gpus: i32, n_layers: u32, n_kv_heads: u32, out: *mut TkvPairing, out_cap: i32, n_pairs: *mut i32) -> i32;
    pub fn tkv_cast(src: u64, src_dtype: i32, dst: u64, dst_dtype: i32, n: u64, stream: *mut c_void) -> i32;
    pub fn tkv_selfcheck_e4m3(skip_bits: u32, mismatches: *mut u64) -> i32;
    pub fn tkv_selfcheck_scaled_quant(mismatches: *mut u64) -> i32;
    pub fn tkv_memcpy_enqueue(dst: u64, src: u64, bytes: u64, stream: *mut c_void) -> i32;
    pub fn tkv_bits_checksum(data: u64, dtype: i32, n: u64, stream: *mut c_void, out: *mut u64) -> i32;
    pub fn tkv_ipc_export(devptr: u64, handle: *mut u8, offset_in_allocation: *mut u64) -> i32;
    pub fn tkv_ipc_import(handle: *const u8, offset_in_allocation: u64, devptr: *mut u64) -> i32;
    pub fn tkv_ipc_close(devptr: u64, offset_in_allocation: u64) -> i32;
    pub fn tkv_decode_attn_scratch_bytes(n_seqs: u32, n_q_heads: u32, head_dim: u32, max_kv_len: u32, split_tokens: u32) -> u64;
    pub fn tkv_decode_attn_enqueue(pool: *const TkvPool, args: *const TkvDecodeAttn, stream: *mut c_void) -> i32;
    pub fn tkv_prefill_attn_enqueue(pool: *const TkvPool, args: *const TkvPrefillAttn, stream: *mut c_void) -> i32;
    pub fn tkv_scored_attn_scratch_bytes(n_seqs: u32, n_q_heads: u32, n_kv_heads: u32, head_dim: u32, max_kv_len: u32) -> u64;
    pub fn tkv_scored_attn_enqueue(pool: *const TkvPool, args: *const TkvScoredAttn, stream: *mut c_void) -> i32;
    pub fn tkv_prefix_attn_scratch_bytes(n_seqs: u32, n_groups: u32, n_q_heads: u32, n_kv_heads: u32, head_dim: u32, max_kv_len: u32, max_prefix_len: u32) -> u64;
    pub fn tkv_prefix_attn_enqueue(pool: *const TkvPool, args: *const TkvPrefixAttn, stream: *mut c_void) -> i32;
    pub fn tkv_evict_select_enqueue(args: *const TkvEvictSelect, stream: *mut c_void) -> i32;
    pub fn tkv_evict_compact_enqueue(pool: *const TkvPool, args: *const TkvEvictCompact, stream: *mut c_void) -> i32;
    pub fn tkv_selfcheck_tensor_cores(mismatches: *mut u64) -> i32;
    pub fn tkv_session_wire_size(h: *const TkvSessionHeader) -> usize;
    pub fn tkv_session_pack(h: *const TkvSessionHeader, blocks: *const u32, logits: *const f32, out: *mut u8, cap: usize, written: *mut usize) -> i32;
    pub fn tkv_session_unpack(in_: *const u8, len: usize, h: *mut TkvSessionHeader, blocks: *mut *const u32, logits: *mut *const f32) -> i32;
    pub fn tkv_page_allocator_new(total_pages: usize) -> *mut tkv_page_allocator;
    pub fn tkv_page_allocator_delete(arg0: *mut tkv_page_allocator);
    pub fn tkv_page_allocator_allocate(arg0: *mut tkv_page_allocator, page: *mut usize) -> i32;
    pub fn tkv_page_allocator_free(arg0: *mut tkv_page_allocator, page: usize);
    pub fn tkv_page_allocator_available(arg0: *const tkv_page_allocator) -> usize;
    pub fn tkv_page_allocator_in_use(arg0: *const tkv_page_allocator) -> usize;
    pub fn tkv_page_allocator_total(arg0: *const tkv_page_allocator) -> usize;
    pub fn tkv_block_table_new(max_blocks: usize) -> *mut tkv_block_table;
    pub fn tkv_block_table_delete(arg0: *mut tkv_block_table);
    pub fn tkv_block_table_set_block(arg0: *mut tkv_block_table, logical: usize, page: usize) -> i32;
    pub fn tkv_block_table_get_block(arg0: *const tkv_block_table, logical: usize, page: *mut usize) -> i32;
    pub fn tkv_block_table_num_blocks(arg0: *const tkv_block_table) -> usize;
    pub fn tkv_block_table_max_blocks(arg0: *const tkv_block_table) -> usize;
    pub fn tkv_block_table_as_slice(arg0: *const tkv_block_table) -> *const u32;
    pub fn tkv_block_table_clear(arg0: *mut tkv_block_table, freed: *mut usize, cap: usize) -> usize;
    pub fn tkv_run_allocator_new(total_pages: usize) -> *mut tkv_run_allocator;
    pub fn tkv_run_allocator_delete(arg0: *mut tkv_run_allocator);
    pub fn tkv_run_allocator_alloc(arg0: *mut tkv_run_allocator, pages: usize, start: *mut usize) -> i32;
    pub fn tkv_run_allocator_free(arg0: *mut tkv_run_allocator, start: usize, pages: usize) -> i32;
    pub fn tkv_run_allocator_try_extend(arg0: *mut tkv_run_allocator, start: usize, pages: usize, target: usize) -> i32;
    pub fn tkv_run_allocator_free_pages(arg0: *const tkv_run_allocator) -> usize;
    pub fn tkv_run_allocator_allocated_pages(arg0: *const tkv_run_allocator) -> usize;
    pub fn tkv_run_allocator_free_runs(arg0: *const tkv_run_allocator, starts: *mut usize, pages: *mut usize, cap: usize) -> usize;
    pub fn tkv_radix_tree_new() -> *mut tkv_radix_tree;
    pub fn tkv_radix_tree_delete(arg0: *mut tkv_radix_tree);
    pub fn tkv_radix_tree_insert(arg0: *mut tkv_radix_tree, tokens: *const u32, n: usize, pages: *const usize, n_pages: usize);
    pub fn tkv_radix_tree_lookup(arg0: *mut tkv_radix_tree, tokens: *const u32, n: usize, pages_out: *mut usize, cap: usize, n_pages: *mut usize) -> usize;
    pub fn tkv_radix_tree_release(arg0: *mut tkv_radix_tree, tokens: *const u32, n: usize);
    pub fn tkv_radix_tree_evict_lru(arg0: *mut tkv_radix_tree, freed: *mut usize, cap: usize) -> usize;
    pub fn tkv_radix_tree_hit_count(arg0: *const tkv_radix_tree) -> u64;
    pub fn tkv_radix_tree_tokens_saved(arg0: *const tkv_radix_tree) -> u64;
    pub fn tkv_radix_tree_node_count(arg0: *const tkv_radix_tree) -> usize;
    pub fn tkv_prefix_table_new(max_entries: usize) -> *mut tkv_prefix_table;
    pub fn tkv_prefix_table_delete(arg0: *mut tkv_prefix_table);
    pub fn tkv_prefix_table_store(arg0: *mut tkv_prefix_table, tokens: *const u32, n: usize, salt: *const c_char, blocks: *const u32, n_blocks: usize, seq_len: usize);
    pub fn tkv_prefix_table_probe(arg0: *mut tkv_prefix_table, tokens: *const u32, n: usize, salt: *const c_char, blocks_out: *mut u32, cap: usize, n_blocks: *mut usize) -> usize;
    pub fn tkv_prefix_table_release(arg0: *mut tkv_prefix_table, tokens: *const u32, n: usize, salt: *const c_char);
    pub fn tkv_prefix_table_len(arg0: *const tkv_prefix_table) -> usize;
    pub fn tkv_prefix_table_hit_count(arg0: *const tkv_prefix_table) -> u64;
    pub fn tkv_prefix_table_tokens_saved(arg0: *const tkv_prefix_table) -> u64;
    pub fn tkv_prefix_index_create(device: i32, capacity: u64, group_tokens: u32, out: *mut *mut tkv_prefix_index) -> i32;
    pub fn tkv_prefix_index_destroy(arg0: *mut tkv_prefix_index);
    pub fn tkv_prefix_index_set_key_bits(arg0: *mut tkv_prefix_index, bits: u32) -> i32;
    pub fn tkv_prefix_index_insert(arg0: *mut tkv_prefix_index, arg1: *const TkvPrefixBatch, stream: *mut c_void) -> i32;
    pub fn tkv_prefix_index_lookup(arg0: *mut tkv_prefix_index, arg1: *const TkvPrefixBatch, out_pages: u64, out_stride: u32, out_matched: u64, stream: *mut c_void) -> i32;
    pub fn tkv_prefix_index_release(arg0: *mut tkv_prefix_index, arg1: *const TkvPrefixBatch, stream: *mut c_void) -> i32;
    pub fn tkv_prefix_index_evict_lru(arg0: *mut tkv_prefix_index, max_nodes: u32, out_pages: u64, out_cap: u32, out_count: u64, out_nodes: u64, stream: *mut c_void) -> i32;
    pub fn tkv_prefix_index_stats(arg0: *mut tkv_prefix_index, stream: *mut c_void, out: *mut TkvPrefixIndexStats) -> i32;
    pub fn tkv_device_page_allocator_create(device: i32, total_pages: u32, out: *mut *mut tkv_device_page_allocator) -> i32;
    pub fn tkv_device_page_allocator_destroy(arg0: *mut tkv_device_page_allocator);
    pub fn tkv_device_page_allocator_allocate(arg0: *mut tkv_device_page_allocator, arg1: *const TkvPageBatch, status: u64, stream: *mut c_void) -> i32;
    pub fn tkv_device_page_allocator_free(arg0: *mut tkv_device_page_allocator, arg1: *const TkvPageBatch, status: u64, stream: *mut c_void) -> i32;
    pub fn tkv_device_page_allocator_available(arg0: *mut tkv_device_page_allocator, stream: *mut c_void, out: *mut u32) -> i32;
    pub fn tkv_handoff_enqueue_device_tables(plan: *mut tkv_plan, batch: *const TkvDeviceBatch, stream: *mut c_void, done_flag: u64, flag_value: u32) -> i32;
    pub fn tkv_refcount_apply_device_tables(dst: *const TkvPool, batch: *const TkvDeviceBatch, delta: i32, stream: *mut c_void) -> i32;
    pub fn tkv_coordinator_new(arg0: *const TkvCoordinatorConfig) -> *mut tkv_coordinator;
    pub fn tkv_coordinator_delete(arg0: *mut tkv_coordinator);
    pub fn tkv_coordinator_set_headroom(arg0: *mut tkv_coordinator, decode_worker: u32, free_blocks: u64) -> i32;
    pub fn tkv_coordinator_submit(arg0: *mut tkv_coordinator, request_id: u64, n_tokens: u32, max_new_tokens: u32, priority: u32, prefill_worker: *mut u32) -> i32;
    pub fn tkv_coordinator_next_prefill(arg0: *mut tkv_coordinator, prefill_worker: u32, request_id: *mut u64) -> i32;
    pub fn tkv_coordinator_prefill_done(arg0: *mut tkv_coordinator, request_id: u64, prefix_tokens_resident: u32) -> i32;
    pub fn tkv_coordinator_admit(arg0: *mut tkv_coordinator, out: *mut TkvAdmission, cap: usize) -> usize;
    pub fn tkv_coordinator_handoff_started(arg0: *mut tkv_coordinator, request_id: u64, now: u64) -> i32;
    pub fn tkv_coordinator_handoff_complete(arg0: *mut tkv_coordinator, request_id: u64) -> i32;
    pub fn tkv_coordinator_handoff_failed(arg0: *mut tkv_coordinator, request_id: u64, action: *mut u32) -> i32;
    pub fn tkv_coordinator_timed_out(arg0: *mut tkv_coordinator, now: u64, request_ids: *mut u64, cap: usize) -> usize;
    pub fn tkv_coordinator_reprefill_done(arg0: *mut tkv_coordinator, request_id: u64) -> i32;
    pub fn tkv_coordinator_finish(arg0: *mut tkv_coordinator, request_id: u64) -> i32;
    pub fn tkv_coordinator_request(arg0: *const tkv_coordinator, request_id: u64, out: *mut TkvRequestInfo) -> i32;
    pub fn tkv_coordinator_stats(arg0: *const tkv_coordinator, out: *mut TkvCoordinatorStats) -> i32;
}
